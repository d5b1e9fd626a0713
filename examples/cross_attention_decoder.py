"""Action queries over the kept tokens of an adapted ViT block: training and
serving.

A batch of videos keeps unequal numbers of tokens. Their tokens pass the
sparse-conv adapter, then a decoder in which a set of learned queries attends to
them (``CrossAttention``: layer norms, cross attention, a residual). Training
runs under autocast(bfloat16) with float32 parameters and clips the gradients of
both as a training loop does; serving projects a video's tokens to keys and
values once and attends to them with one query at a time.

    python examples/cross_attention_decoder.py [steps]
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import eccv26_tad_amd as sv  # noqa: E402

EMBED, HEADS, KEY_HEADS, QUERIES = 384, 6, 2, 40
T, H, W, KEEP, BATCH = 8, 14, 14, 0.6, 2


class Decoder(nn.Module):
    """Learned queries, two layers of attention to the tokens, a boundary per query."""

    def __init__(self):
        super().__init__()
        self.queries = nn.Parameter(torch.randn(QUERIES, EMBED) * 0.02)
        self.layers = nn.ModuleList(sv.CrossAttention(EMBED, HEADS, kv_heads=KEY_HEADS) for _ in range(2))
        self.head = nn.Linear(EMBED, 2)

    def forward(self, tokens, lengths):
        x = self.queries.expand(tokens.shape[0], -1, -1)
        for layer in self.layers:
            x = layer(x, tokens, key_lengths=lengths)
        return self.head(x).float().sigmoid()

    @torch.no_grad()
    def serve(self, tokens):
        """One query at a time over one video's tokens ``[1, n, EMBED]``."""
        kv = [layer.project_context(tokens) for layer in self.layers]
        out = []
        for query in self.queries:
            x = query.view(1, 1, -1).to(tokens.dtype)
            for layer, pair in zip(self.layers, kv):
                x = layer(x, kv=pair)
            out.append(self.head(x).float().sigmoid())
        return torch.cat(out, 1)


def kept_tokens(dev, gen):
    """Token features, the kept positions and their neighbor table; the samples'
    own lengths (the others' tokens pad to the longest)."""
    n = int(T * H * W * KEEP)
    idx = torch.rand(BATCH, T * H * W, device=dev, generator=gen).topk(n, 1).indices.sort(1).values
    mask = torch.zeros(BATCH, T * H * W, dtype=torch.uint8, device=dev).scatter_(1, idx, 1).view(BATCH, T, H, W)
    table = sv.build_neighbor_table(mask, n=BATCH * n).view(BATCH, n, 9)
    x = torch.randn(BATCH, 1 + n, EMBED, device=dev, generator=gen)  # a CLS token before the patches
    lengths = torch.tensor([1 + n] + [1 + n // 2] * (BATCH - 1), dtype=torch.int32, device=dev)
    return x, idx, table, lengths


def main(steps=20, dev="cuda"):
    torch.manual_seed(0)
    gen = torch.Generator(device=dev).manual_seed(0)
    adapter, decoder = sv.SparseConvAdapter(EMBED).to(dev), Decoder().to(dev)
    params = [*adapter.parameters(), *decoder.parameters()]
    opt = torch.optim.AdamW(params, lr=1e-3)
    x, idx, table, lengths = kept_tokens(dev, gen)
    target = torch.rand(BATCH, QUERIES, 2, device=dev, generator=gen)
    losses, norms = [], []
    for _ in range(steps):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            boundaries = decoder(adapter(x, H, W, idx, T * H * W, table), lengths)
        loss = (boundaries - target).square().mean()
        loss.backward()
        norms.append(sv.clip_grad_norm_(params, 0.02))
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    losses, norms = torch.stack(losses).tolist(), torch.stack(norms).tolist()
    adapter, decoder = adapter.bfloat16(), decoder.bfloat16()
    with torch.no_grad():
        tokens = adapter(x.bfloat16(), H, W, idx, T * H * W, table)
        together = decoder(tokens, lengths)
        served = decoder.serve(tokens[:1])
    return losses, norms, together[:1], served


if __name__ == "__main__":
    losses, norms, together, served = main(int(sys.argv[1]) if len(sys.argv) > 1 else 20)
    print("loss %.4f -> %.4f, gradient norm %.3f -> %.3f" % (losses[0], losses[-1], norms[0], norms[-1]))
    print("served one query at a time against all together: largest difference %.2g" % float((served - together).abs().max()))
