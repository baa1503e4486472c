// Shared by the language-model operators (embedding.hip, logprobs.hip,
// act8.hip): element types, host-side argument checks, launch status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

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

// Token t of a list, as a 64-bit number.  Lists hold fewer than 2^31 tokens.
__device__ __forceinline__ int64_t token(const ms_tokens_t& ids, int64_t t) {
  int64_t at;
  if (t < ids.inner) {
    at = t * ids.inner_stride;
  } else {
    const uint32_t inner = static_cast<uint32_t>(ids.inner), q = static_cast<uint32_t>(t) / inner;
    at = q * ids.outer_stride + (static_cast<uint32_t>(t) - q * inner) * ids.inner_stride;
  }
  return ids.wide ? static_cast<const int64_t*>(ids.data)[at]
                  : static_cast<int64_t>(static_cast<const int32_t*>(ids.data)[at]);
}

// First element of row r; fewer than 2^31 rows.
__device__ __forceinline__ int64_t row_start(const ms_rows_t& m, int64_t r) {
  if (r < m.inner) return r * m.inner_stride;
  const uint32_t inner = static_cast<uint32_t>(m.inner), q = static_cast<uint32_t>(r) / inner;
  return q * m.outer_stride + (static_cast<uint32_t>(r) - q * inner) * m.inner_stride;
}

// N values at any element alignment, as one load or store of up to 16 bytes:
// gfx950's global memory takes vectors at 2- and 4-byte addresses.
template <int B> struct raw_of;
template <> struct raw_of<2> { typedef uint16_t type; };
template <> struct raw_of<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct raw_of<8> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2)));
};
template <> struct raw_of<16> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};

template <typename T, int N>
struct Pack {
  T v[N];
};

template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load(const T* p) {
  typedef typename raw_of<N * sizeof(T)>::type raw;
  const raw r = *reinterpret_cast<const raw*>(p);
  Pack<T, N> x;
  static_assert(sizeof(x) == sizeof(r), "");
  __builtin_memcpy(&x, &r, sizeof(r));
  return x;
}
template <int N, typename T>
__device__ __forceinline__ void store(T* p, const Pack<T, N>& x) {
  typedef typename raw_of<N * sizeof(T)>::type raw;
  raw r;
  __builtin_memcpy(&r, &x, sizeof(r));
  *reinterpret_cast<raw*>(p) = r;
}

// N values that are read once, at any element alignment: not kept in the caches.
template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load_stream_any(const T* p) {
  typedef typename raw_of<N * sizeof(T)>::type raw;
  const raw r = __builtin_nontemporal_load(reinterpret_cast<const raw*>(p));
  Pack<T, N> x;
  __builtin_memcpy(&x, &r, sizeof(r));
  return x;
}
template <int N, typename T>
__device__ __forceinline__ void store_stream_any(T* p, const Pack<T, N>& x) {
  typedef typename raw_of<N * sizeof(T)>::type raw;
  raw r;
  __builtin_memcpy(&r, &x, sizeof(r));
  __builtin_nontemporal_store(r, reinterpret_cast<raw*>(p));
}
// 16 aligned bytes that are not read soon.
template <int N, typename T>
__device__ __forceinline__ void store_stream(T* p, const Pack<T, N>& x) {
  typedef uint32_t raw __attribute__((ext_vector_type(4)));
  static_assert(N * sizeof(T) == 16, "");
  raw r;
  __builtin_memcpy(&r, &x, 16);
  __builtin_nontemporal_store(r, reinterpret_cast<raw*>(p));
}

// A value that all lanes have, told to the compiler: branches on it leave loads
// in flight.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int read_lane(int x, int lane) {
  return __builtin_amdgcn_readlane(x, lane);
}
__device__ __forceinline__ int64_t read_lane(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

inline bool good_dtype(int32_t d) { return d >= MS_OPS_F32 && d <= MS_OPS_BF16; }
inline int64_t dtype_bytes(int32_t d) { return d == MS_OPS_F32 ? 4 : 2; }

// Whether a * b values, as many bytes and some times that, can be counted in 64 bits.
inline bool countable(int64_t a, int64_t b = 1) {
  int64_t product;
  return !__builtin_mul_overflow(a, b, &product) && product < int64_t{1} << 56;
}

inline bool good_tokens(const ms_tokens_t* t) {
  return t && t->n >= 0 && t->n <= INT32_MAX && t->inner >= 1 && (t->n == 0 || t->data);
}
inline bool good_rows(const ms_rows_t* m) {
  return m && m->n >= 0 && m->n <= INT32_MAX && m->width >= 0 && m->inner >= 1 &&
         countable(m->n, m->width) && good_dtype(m->dtype) && (m->n == 0 || m->width == 0 || m->data);
}

// A launch has fewer than 2^32 threads.
inline bool fits(int64_t blocks, int threads) { return blocks <= UINT32_MAX / threads; }

// Launches a kernel and returns the launch's own status.  (After <<<>>> only
// hipGetLastError() tells, and that is the last error of any call of the thread:
// one that earlier work left would be taken for the launch's, and taken away from those who
// look for it.)
template <typename... P, typename... A>
int launch(void (*kernel)(P...), int64_t blocks, int threads, hipStream_t s, A... a) {
  static_assert(sizeof...(P) == sizeof...(A), "");
  std::tuple<P...> values(static_cast<P>(a)...);
  return std::apply(
      [&](P&... v) {
        void* args[] = {static_cast<void*>(&v)...};
        return static_cast<int>(hipLaunchKernel(reinterpret_cast<const void*>(kernel),
                                                dim3(static_cast<unsigned>(blocks)), dim3(threads),
                                                args, 0, s));
      },
      values);
}

}  // namespace ops
