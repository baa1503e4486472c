// Shared by the language-model operators (embedding.hip, logprobs.hip,
// act8.hip): element types, host-side argument checks, launch status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "minispeed_ops.h"

namespace ops {

using f16 = _Float16;
using bf16 = __bf16;

constexpr int kWave = 64;

template <typename T>
__device__ __forceinline__ float widen(T x) {
  return static_cast<float>(x);
}

// One rounding to nearest even of the fp32 value.  (Left alone, the compiler
// joins a product and its narrowing to fp16 into one mixed instruction, which
// skips the rounding of the product to 32 bits.)
template <typename T>
__device__ __forceinline__ T narrow(float x) {
  if (sizeof(T) == 2) asm("" : "+v"(x));
  return static_cast<T>(x);
}

__device__ __forceinline__ float quiet_nan() { return __builtin_nanf(""); }

// Token t of a list, as a 64-bit number.
__device__ __forceinline__ int64_t token(const ms_tokens_t& ids, int64_t t) {
  const int64_t at = t < ids.inner ? t * ids.inner_stride
                                   : (t / ids.inner) * ids.outer_stride +
                                         (t % ids.inner) * ids.inner_stride;
  return ids.wide ? static_cast<const int64_t*>(ids.data)[at]
                  : static_cast<int64_t>(static_cast<const int32_t*>(ids.data)[at]);
}

// First element of row r.
__device__ __forceinline__ int64_t row_start(const ms_rows_t& m, int64_t r) {
  return r < m.inner ? r * m.inner_stride
                     : (r / m.inner) * m.outer_stride + (r % m.inner) * m.inner_stride;
}

inline bool good_dtype(int32_t d) { return d >= MS_OPS_F32 && d <= MS_OPS_BF16; }
inline int64_t dtype_bytes(int32_t d) { return d == MS_OPS_F32 ? 4 : 2; }

inline bool good_tokens(const ms_tokens_t* t) {
  return t && t->n >= 0 && t->inner >= 1 && (t->n == 0 || t->data);
}
inline bool good_rows(const ms_rows_t* m) {
  return m && m->n >= 0 && m->width >= 0 && m->inner >= 1 && good_dtype(m->dtype) &&
         (m->n == 0 || m->width == 0 || m->data);
}

// The launch's own status; errors that earlier work left are not reported here
// as ours.
inline int launched() { return static_cast<int>(hipGetLastError()); }

}  // namespace ops
