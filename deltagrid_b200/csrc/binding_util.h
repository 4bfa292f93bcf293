// binding_util.h -- what the parts of the compiled module `_hsru` share: error raising,
// argument checks, the current stream and the device status words.
#pragma once

#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>
#include <unordered_map>
#include <vector>

#include "deltagrid_b200.h"

namespace py = pybind11;
using at::Tensor;

namespace dgb {

extern PyObject* g_error;      // deltagrid_b200._lib.DeltaGridError, set at import

[[noreturn]] inline void raise_status(int st, const char* what) {
    std::string msg = std::string(what) + " failed: " + dg_status_string(st);
    if (st == DG_ERR_CUDA) msg += " (cudaError " + std::to_string(dg_last_cuda_error()) + ")";
    msg += " [status " + std::to_string(st) + "]";
    const py::gil_scoped_acquire lock;         // autograd runs C++ backward nodes on threads that do not hold it
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, msg.c_str());
    throw py::error_already_set();
}
inline void check(int st, const char* what) {
    if (st != 0) raise_status(st, what);
}

// binding.cpp:18 -- TORCH_CHECK(x.is_cuda(), #x " must be a CUDA tensor")
inline void check_cuda(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
}

// AT_DISPATCH_FLOATING_TYPES_AND2(Half, BFloat16, ...) of the reference bindings
inline int dtype_code(const Tensor& t, const char* op) {
    switch (t.scalar_type()) {
    case at::kFloat: return DG_DTYPE_F32;
    case at::kDouble: return DG_DTYPE_F64;
    case at::kHalf: return DG_DTYPE_F16;
    case at::kBFloat16: return DG_DTYPE_BF16;
    default: TORCH_CHECK(false, "\"", op, "\" not implemented for '", c10::toString(t.scalar_type()), "'");
    }
    return -1;
}

// data_ptr<scalar_t>() in the reference raises when a tensor's dtype differs
inline void same_dtype(const Tensor& ref, const char* op, const char* name, const Tensor& t) {
    TORCH_CHECK(t.scalar_type() == ref.scalar_type(), op, ": expected ", name, " to have dtype ",
                c10::toString(ref.scalar_type()), ", got ", c10::toString(t.scalar_type()));
}

inline Tensor contig(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

inline void* stream_of(const Tensor& t) {
    return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// one int32 device status word per device for the kernels' self-checks; kept for
// the life of the process (never freed, so nothing runs after CUDA shuts down)
Tensor& status_word(const at::Device& dev);

inline void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// the language-model operators (binding_lm.cpp)
void bind_lm(py::module_& m);

}  // namespace dgb
