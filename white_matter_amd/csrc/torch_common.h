// Helpers of the operators registered from C++ (torch_ops.cpp, serve_ops.cpp).
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "wmx_attn.h"

namespace wmx_torch {

using at::Tensor;

inline bool vector_ready(const Tensor& x) {
  if (x.stride(-1) != 1 && x.size(-1) != 1) return false;
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
  for (int64_t d = 0; d + 1 < x.dim(); ++d)
    if (x.size(d) > 1 && x.stride(d) % 8) return false;
  return true;
}

// bf16 with unit head_dim stride and 16-byte aligned rows; strided views
// (cache channels, capacity padding, BQHD storage) are kept without a copy
inline Tensor operand(Tensor x) {
  if (x.scalar_type() != at::kBFloat16) x = x.to(at::kBFloat16);
  if (vector_ready(x)) return x;
  x = x.contiguous();
  return vector_ready(x) ? x : x.clone();
}

// [batch, head, token] element strides of a 4-D tensor; size-1 dims give 0
inline void strides3(const Tensor& x, int64_t (&out)[3]) {
  for (int d = 0; d < 3; ++d) out[d] = x.size(d) > 1 ? x.stride(d) : 0;
}

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == WMX_OK, what, " failed (", rc, "): ", wmx_last_error());
}

inline hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline Tensor mask_bytes(const c10::optional<Tensor>& key_mask) {
  if (!key_mask) return Tensor();
  return key_mask->contiguous().view(at::kByte);
}

// Contiguous and 16-byte aligned.
inline Tensor dense16(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

}  // namespace wmx_torch
