// What the native torch operators share: the library's functions, bound at the first launch,
// and the checks that every operator makes.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "../../include/mmuon.h"

namespace mmuon_torch {

using at::Tensor;

struct Abi {
  int (*fwd)(const mmuon_butterfly_args*, void*) = nullptr;
  int (*bwd)(const mmuon_butterfly_args*, void*) = nullptr;
  size_t (*workspace)(const mmuon_butterfly_args*) = nullptr;
  int (*ce_fwd)(const mmuon_ce_args*, void*) = nullptr;
  int (*ce_fwd_bwd)(const mmuon_ce_args*, void*) = nullptr;
  size_t (*ce_workspace)(const mmuon_ce_args*, int32_t) = nullptr;
  int (*scale)(void*, int64_t, void*, int64_t, const float*, void*) = nullptr;
  int (*emb_fwd)(const mmuon_embedding_args*, void*) = nullptr;
  int (*emb_bwd)(const mmuon_embedding_args*, void*) = nullptr;
  size_t (*emb_workspace)(const mmuon_embedding_args*) = nullptr;
  const char* (*last_error)() = nullptr;
};
extern Abi abi;
extern std::atomic<bool> bound;

// Binds abi to the functions of the library that monarch_muon_amd/_abi.py loads, or raises.
void bind_library();

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", abi.last_error());
}

inline void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "libmmuon kernels need tensors on a ROCm GPU (no CPU path)");
}

// The kernels read rows of 16-B chunks.  A gradient may be a contiguous view at any element
// (one of the parts that torch.cat's backward hands out): such a one is copied.
Tensor dense_aligned(const Tensor& t);

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Whether a backward is wanted.  None of the operators has a forward-mode derivative: a tangent
// raises (dropped, it would count as zero).
inline bool any_requires_grad(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(),
                                "libmmuon operators have no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return false;
  return std::any_of(ts.begin(), ts.end(), [](const Tensor* t) { return t->requires_grad(); });
}

}  // namespace mmuon_torch
