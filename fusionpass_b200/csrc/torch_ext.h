// Argument helpers shared by the sources of the torch extension fusionpass_b200._fpkern.
#pragma once

#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "fpkern.h"

namespace fpk_ext {

[[noreturn]] inline void value_error(const std::string& msg) { throw pybind11::value_error(msg); }

inline void check_status(int rc, const char* what) {
  if (rc != FPK_OK)
    throw std::runtime_error(std::string(what) + ": " + fpk_status_string(rc) + " (status " + std::to_string(rc) +
                             ")");
}

inline void require_cuda(const at::Tensor& t, const char* what) {
  if (!t.defined() || !t.is_cuda())
    throw std::runtime_error(std::string(what) +
                             ": fused steps run only in libfpkern.so on a CUDA device; there is no CPU path");
}

inline void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// RMS norm, 8-bit linear and score attention (torch_block.cpp)
void bind_block(pybind11::module_& m);

}  // namespace fpk_ext
