// What the sources of the PyTorch binding share.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "../../include/fa_b200.h"

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FA_OK, what, " failed (", rc, "): ", fa_last_error());
}

inline fa_stream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Scratch memory of a call; 256-byte aligned, as the caching allocator gives it
inline at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

void bind_pages(py::module_& m);  // torch_ext_pages.cpp
