// Helpers of the extension's source files.
#pragma once

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "../../include/svtad_sparse.h"

inline int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SVTAD_F32;
        case at::kHalf: return SVTAD_F16;
        case at::kBFloat16: return SVTAD_BF16;
        case at::kDouble: return SVTAD_F64;
        default: TORCH_CHECK(false, "opentad_sparse_ops: unsupported dtype ", t.scalar_type());
    }
    return -1;
}

inline void* stream_of(const at::Tensor& t) {
    return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void check_status(int st, const char* who) {
    TORCH_CHECK(st == SVTAD_OK, "opentad_sparse_ops.", who, ": ", svtad_last_error(), " (status ",
                st, ")");
}

inline void check_gpu(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "opentad_sparse_ops: ", name, " must be a GPU tensor");
}

// The operators of torch_ext_operators.cpp
void bind_operators(pybind11::module& m);
