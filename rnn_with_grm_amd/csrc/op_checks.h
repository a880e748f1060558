// What the torch ops of the additions to the reference share: checks of their arguments, strides of packed rows, streams and
// status codes of the C ABI.
#pragma once

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>

#include "grm_hip.h"

namespace grm_ops {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

inline int dtype_code(const Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GRM_HIP_F32;
    case at::kHalf: return GRM_HIP_F16;
    case at::kBFloat16: return GRM_HIP_BF16;
    default: break;
  }
  TORCH_CHECK_VALUE(false, op, ": ", name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  return -1;
}

inline bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == GRM_HIP_OK, op, " failed (", rc, "): ", grm_hip_last_error());
}

inline void check_device(const Tensor& t, const Tensor& like, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on ", like.device());
}

// Autograd's count of writes to an argument: a graph that saved it for its backward then refuses to use what it holds now.
// (No graph can save a tensor made in inference mode, and it has no count.)
inline void written(Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A contiguous optional tensor's pointer; `keep` holds what it points into.
inline void* opt_ptr(const OptTensor& t, Tensor& keep) {
  if (!has(t)) return nullptr;
  keep = t->contiguous();
  return keep.data_ptr();
}

// Rows of the last `inner` dimensions packed, any stride between tokens and sequences: a slice of a
// wider projection is read where it lies.
inline Tensor packed_rows(const Tensor& t, int64_t inner) {
  int64_t want = 1;
  for (int64_t d = t.dim() - 1; d >= t.dim() - inner; --d) {
    if (t.size(d) != 1 && t.stride(d) != want) return t.contiguous();
    want *= t.size(d);
  }
  // Rows of a sequence lie one behind the other, near enough for 32-bit offsets inside a tile of tokens.
  const int64_t d = t.dim() - inner - 1;
  if (d > 0 && t.size(d) != 1 && (t.stride(d) < want || t.stride(d) > (int64_t{1} << 21))) return t.contiguous();
  return t;
}

inline int64_t stride_of(const Tensor& t, int64_t dim, int64_t packed) { return t.size(dim) > 1 ? t.stride(dim) : packed; }

inline const int64_t* lengths_ptr(const OptTensor& lengths, int64_t B, const Tensor& like, const char* op, Tensor& keep) {
  if (!has(lengths)) return nullptr;
  check_device(*lengths, like, op, "lengths");
  TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B &&
                  (lengths->scalar_type() == at::kLong || lengths->scalar_type() == at::kInt),
              op, ": lengths must be int32 or int64 [batch]");
  keep = lengths->to(at::kLong).contiguous();
  return keep.data_ptr<int64_t>();
}

inline bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

inline Tensor f32_state(const Tensor& t) {
  Tensor m = t.contiguous();
  return aligned16(m) ? m : m.clone();
}

inline Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({std::max<int64_t>(n, 16)}, like.options().dtype(at::kByte));
}

}  // namespace grm_ops
