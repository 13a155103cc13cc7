// Helpers shared by the binding's sources.
#pragma once

#include <stdexcept>
#include <string>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include "mhc_proj.h"

namespace mhcp_torch {

namespace py = pybind11;

// fp32 on the tensor's own CUDA device, or on the current device for
// non-CUDA tensors (solvers_torch.cpp:52-61).
inline torch::TensorOptions target_options(const torch::Tensor& x)
{
    auto opts = torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA);
    if (x.device().is_cuda()) opts = opts.device(torch::kCUDA, x.device().index());
    return opts;
}

inline void check_status(int status, const char* what)
{
    if (status != MHC_OK)
        throw std::runtime_error(std::string(what) + " failed: " + mhc_status_string(status));
}

inline cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Storage type code of the C ABI, or -1.
inline int dtype_code(const torch::Tensor& x)
{
    switch (x.scalar_type()) {
        case torch::kFloat32: return MHC_DTYPE_F32;
        case torch::kBFloat16: return MHC_DTYPE_BF16;
        case torch::kFloat16: return MHC_DTYPE_F16;
        default: return -1;
    }
}

// The functions of torch_binding_residual.cpp.
void bind_residual_path(py::module& m);

}  // namespace mhcp_torch
