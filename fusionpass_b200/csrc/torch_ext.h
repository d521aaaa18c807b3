// Argument helpers shared by the sources of the torch extension fusionpass_b200._fpkern.
#pragma once

#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
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

using c10::optional;

inline int32_t type_code(at::ScalarType t, const char* what) {
  if (t == at::kHalf) return FPK_F16;
  if (t == at::kBFloat16) return FPK_BF16;
  if (t == at::kFloat) return FPK_F32;
  value_error(std::string(what) + ": unsupported dtype " + c10::toString(t) + " (f16, bf16 and f32 only)");
}

// the operators have no derivative: neither backward, nor forward along a dual tensor's tangent
inline void no_derivative(const at::Tensor& t, const char* what, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    value_error(std::string(what) + ": " + name + " requires a gradient, which this operator does not have");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    value_error(std::string(what) + ": " + name + " has a tangent, which this operator has no derivative for");
}

inline void check_tensor(const at::Tensor& t, const at::Device& dev, const char* what, const char* name) {
  require_cuda(t, what);
  if (t.device() != dev) value_error(std::string(what) + ": " + name + " must be on the device of the first input");
  no_derivative(t, what, name);
}

inline bool given(const optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

// a caller's tensor has new contents: what autograd saved of it is out of date
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A result's memory is no operand's, as far as that can be told at once: of two dense tensors.
// (Views of one buffer that lie between one another are the caller's.)
inline void apart(const at::Tensor& out, const at::Tensor& in, const char* what) {
  const at::MemOverlapStatus st = at::get_overlap_status(out, in);
  if (st == at::MemOverlapStatus::Full || st == at::MemOverlapStatus::Partial)
    value_error(std::string(what) + ": out overlaps an input");
}

// a new tensor from torch's CUDA allocator, on the current stream, without the dispatcher's way there
inline at::Tensor fresh(at::IntArrayRef dims, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(dims, type, dev, c10::nullopt);
}

// [B, H, S, D] as the kernels read it: unit D stride, the others multiples of 16 bytes,
// a base on 16 bytes; copied otherwise.
inline at::Tensor aligned(const at::Tensor& t, int64_t unit, int64_t* st) {
  at::Tensor r = t;
  for (int pass = 0; pass < 2; ++pass) {
    bool ok = (r.stride(3) == 1 || r.size(3) == 1) && reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) {
      st[i] = r.size(i) == 1 ? r.size(3) : r.stride(i);  // the stride of a dim of one is never used
      ok = ok && st[i] > 0 && st[i] % unit == 0;
    }
    if (ok || r.numel() == 0) return r;
    r = r.clone(at::MemoryFormat::Contiguous);
  }
  return r;
}

// RMS norm, 8-bit linear and score attention (torch_block.cpp)
void bind_block(pybind11::module_& m);
// 8-bit cache, tree attention and the verification of drafted tokens (torch_draft.cpp)
void bind_draft(pybind11::module_& m);

}  // namespace fpk_ext
