// act8.hip — activations held in 8 bits between forward and backward (gfx950).
//
// Blocks of 32 values share a power-of-two scale, so that dividing by it is
// exact and a code is one rounding of the value.
//
// All kernels stream: a lane takes units of 16 bytes of the unheld type, 8 or 4
// values, so that 4 or 8 neighbouring lanes have a block.  They are bound by
// memory, the error-function GELU of 2-byte types (29 instructions and two
// quarter-rate ones a value, forward) about as much by arithmetic.

#include "ops_common.h"

namespace {

using namespace ops;

constexpr int kBlock = MS_OPS_BLOCK;

// The exponent byte for a block whose largest magnitude has these bits: the
// magnitude rounded to 7 significant bits (half to even or up makes no
// difference: 127.5 rounds to 128 either way) is at most 127 * 2^(e - 127).
__device__ __forceinline__ uint32_t exponent_of(uint32_t magnitude) {
  if (magnitude >= 0x7F800000u) return 255u;
  const int e = static_cast<int>((magnitude + 0x10000u) >> 23) - 6;
  return e < 1 ? 1u : static_cast<uint32_t>(e);
}
// 2^(127 - e) and 2^(e - 127); NaN for e = 255.
__device__ __forceinline__ float inverse_step(uint32_t e) {
  return e == 255u ? 0.f : __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float step_of(uint32_t e) {
  return e == 255u ? quiet_nan() : __uint_as_float(e << 23);
}

struct Act {
  float f, df;
};

// Exponentials are taken 2^32 too large and the results put right by a last
// product: v_exp_f32 flushes results below 2^-126, the product does not, so
// the far tails are right down to the smallest denormal.
constexpr float kLift = 32.f, kDrop = 2.3283064e-10f;   // 2^-32

// kFine in what follows: for results of 32 bits, and in swiglu's backward pass, where it
// costs nothing (4096 x 14336 bf16 96 us either way) and its products of three come closer to
// the nearest 2-byte values.  Other 2-byte results hide it, and it costs: 8192 x 8192 fp16,
// forward and backward, gelu 77 and 83 us, 63 and 78 without; gelu_tanh 66 and 83, 56 and 78; silu
// 58 and 79, 56 and 79; swiglu forward 88 and 87, of views 109 and 102.
template <typename T, int K, bool kBackward>
constexpr bool kFineOf = sizeof(T) == 4 || (kBackward && K == MS_ACT_SWIGLU);

// 2^(32 - m L) for m = hi + lo >= 0 and L = l + l_lo.  Fine: of the exponent's
// whole and broken parts only the second goes through v_exp_f32, so that its rounding
// is that of a number below 1: relative errors of 1e-7, where that of 32 - m L,
// rounded by itself, is 4e-7 for m of some units and 1e-6 from 50 on.
template <bool kFine>
__device__ __forceinline__ float lifted_exp2(float hi, float lo, float l, float l_lo) {
  if (!kFine) return __builtin_amdgcn_exp2f(hi * -l + kLift);
  const float n = rintf(hi * -l);
  const float part = fmaf(hi, -l_lo, fmaf(lo, -l, fmaf(hi, -l, -n)));
  return ldexpf(__builtin_amdgcn_exp2f(part), static_cast<int>(n) + static_cast<int>(kLift));
}
// 1 / x; fine: to half a unit in the last place but for some (v_rcp_f32: one).
template <bool kFine>
__device__ __forceinline__ float reciprocal(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return kFine ? fmaf(fmaf(-x, r, 1.f), r, r) : r;
}

// x s(z) and its derivative s + x s (1 - s) z', s the logistic function.  With
// e = exp(-|z|), r = 1 / (1 + e): s is r or e r, 1 - s the other.
template <bool kFine>
__device__ __forceinline__ Act logistic_act(float x, float z, float dz) {
  // (200 and beyond give 0; NaN stays)
  const float m = kFine ? __builtin_elementwise_minimum(fabsf(z), 200.f) : fabsf(z);
  const float e = lifted_exp2<kFine>(m, 0.f, 1.44269502f, 1.92596303e-8f);    // log2 e
  const float r = reciprocal<kFine>(fmaf(e, kDrop, 1.f));
  const bool low = z < 0.f;
  const float s = low ? e * r : r, drop = low ? kDrop : 1.f;
  const float rest = low ? r : (e * r) * kDrop;
  // beyond +-200 the product with `rest` or s is 0, and must not be inf * 0
  const float turn = __builtin_amdgcn_fmed3f(x, -200.f, 200.f) * rest * dz;
  Act a;
  a.f = (x * s) * drop;
  a.df = fmaf(s, turn, s) * drop;
  return a;
}

template <int K, bool kFine>
__device__ __forceinline__ Act act(float x) {
  if (K == MS_ACT_GELU) {
    // Phi(-a) = exp(-a^2 / 2) Q(a), Q = erfcx(a / sqrt 2) / 2, by weighted fits over
    // [0, 15] (least squares, reweighted towards the least largest relative error), so that
    // the tail needs no difference.  Fine: r P(a r) with r = 1 / (a + 3.75), 4e-8; near 0
    // only P's first terms count.  Else t P(t) with t = 1 / (1 + 0.37 a), 2e-7, 5e-7 as
    // evaluated, one operation fewer: 8192 x 8192 bf16 forward 57 us, 59 with the other.
    const float a = __builtin_elementwise_minimum(fabsf(x), 15.f);      // NaN stays
    float q;
    if (kFine) {
      const float r = __builtin_amdgcn_rcpf(a + 3.75f), u = a * r;
      q = 0.113523148f;
      q = fmaf(q, u, -0.388860106f);
      q = fmaf(q, u, 0.299531192f);
      q = fmaf(q, u, 0.386662275f);
      q = fmaf(q, u, -0.285418391f);
      q = fmaf(q, u, -1.70484757f);
      q = fmaf(q, u, 3.83854222f);
      q = fmaf(q, u, -3.7351315f);
      q = fmaf(q, u, 1.875f) * r;
    } else {
      const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.37f, 1.f));
      q = -0.0313271917f;
      q = fmaf(q, t, 0.135133371f);
      q = fmaf(q, t, -0.194299534f);
      q = fmaf(q, t, 0.0645160899f);
      q = fmaf(q, t, 0.0134064732f);
      q = fmaf(q, t, 0.0901831239f);
      q = fmaf(q, t, 0.127163798f);
      q = fmaf(q, t, 0.147615328f);
      q = fmaf(q, t, 0.147608608f) * t;
    }
    const float a2 = a * a;
    const float e =                                                     // log2 e / 2
        lifted_exp2<kFine>(a2, fmaf(a, a, -a2), 0.721347511f, 9.62981495e-9f);
    Act y;
    // x Phi(x) = max(x, 0) - a Phi(-a);  Phi + x phi is w below 0, 1 - w above
    y.f = fmaf(a * q * e, -kDrop, fmaxf(x, 0.f));
    const float w = fmaf(a, -0.398942280f, q) * e;
    y.df = x < 0.f ? w * kDrop : fmaf(w, -kDrop, 1.f);
    return y;
  }
  if (K == MS_ACT_GELU_TANH) {
    const float c = 2.f * 0.797884561f, x2 = x * x;
    return logistic_act<kFine>(x, c * x * fmaf(x2, 0.044715f, 1.f),
                               fmaf(fminf(x2, 4e4f), 3.f * 0.044715f * c, c));
  }
  return logistic_act<kFine>(x, x, 1.f);
}

template <typename T>
struct Units {
  static constexpr int kVec = 16 / sizeof(T), kLanes = kBlock / kVec;
  typedef Pack<T, kVec> Unit;
  typedef typename raw_of<kVec>::type Codes;         // kVec codes, 4 or 8 bytes
};
// Any byte alignment: a checkpoint may begin anywhere.
typedef uint32_t any4 __attribute__((aligned(1)));
typedef uint32_t any8 __attribute__((ext_vector_type(2), aligned(1)));

// The block's largest magnitude as fp32 bits, in each of its lanes.
__device__ __forceinline__ uint32_t lanes_max(uint32_t m, int lanes) {
#define STEP(ctrl)                                                                             \
  {                                                                                            \
    const uint32_t o = __builtin_amdgcn_update_dpp(0, m, ctrl, 0xf, 0xf, true);                \
    m = o > m ? o : m;                                                                         \
  }
  STEP(0xB1);                       // quad_perm 1 0 3 2
  STEP(0x4E);                       // quad_perm 2 3 0 1
  if (lanes == 8) STEP(0x141);      // row_half_mirror: the other four
#undef STEP
  return m;
}
// Magnitudes compare as whole numbers, 2-byte types' two at a time.
__device__ __forceinline__ uint32_t block_max(const Pack<float, 4>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(x.v[i]) & 0x7FFFFFFFu;
    m = b > m ? b : m;
  }
  return lanes_max(m, 8);
}
template <typename T>
__device__ __forceinline__ uint32_t block_max(const Pack<T, 8>& x) {
  typedef uint16_t two __attribute__((ext_vector_type(2)));
  uint32_t w[4];
  __builtin_memcpy(w, &x, 16);
  two m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    two b;
    const uint32_t magnitude = w[i] & 0x7FFF7FFFu;
    __builtin_memcpy(&b, &magnitude, 4);
    m = __builtin_elementwise_max(m, b);
  }
  const uint16_t most = static_cast<uint16_t>(lanes_max(m.x > m.y ? m.x : m.y, 4));
  T as;
  __builtin_memcpy(&as, &most, 2);
  return __float_as_uint(widen(as));
}

// Codes of N values: adding 1.5 * 2^23 rounds x / step to nearest even and
// leaves it in the low byte; an infinity or NaN (inverse step 0) leaves 0.
template <int N>
__device__ __forceinline__ void encode(const float (&x)[N], float inverse,
                                       uint32_t (&codes)[N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    uint32_t k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      k[j] = __float_as_uint(fmaf(x[4 * i + j], inverse, 12582912.f));
    const uint32_t lo = __builtin_amdgcn_perm(k[1], k[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(k[3], k[2], 0x0c0c0400u);
    codes[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
}
template <int N>
__device__ __forceinline__ void decode(const uint32_t (&codes)[N / 4], float step, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = static_cast<float>(static_cast<int8_t>(codes[i / 4] >> (8 * (i % 4)))) * step;
}

__device__ __forceinline__ void put_codes(int8_t* p, const uint32_t (&c)[1]) {
  __builtin_nontemporal_store(c[0], reinterpret_cast<any4*>(p));
}
__device__ __forceinline__ void put_codes(int8_t* p, const uint32_t (&c)[2]) {
  __builtin_nontemporal_store(any8{c[0], c[1]}, reinterpret_cast<any8*>(p));
}
__device__ __forceinline__ void get_codes(const int8_t* p, uint32_t (&c)[1]) {
  c[0] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(p));
}
__device__ __forceinline__ void get_codes(const int8_t* p, uint32_t (&c)[2]) {
  const any8 v = __builtin_nontemporal_load(reinterpret_cast<const any8*>(p));
  c[0] = v.x;
  c[1] = v.y;
}

// kWhole in what follows: all of the block's units lie within n.  It is asked
// once for the block; a branch at every load would wait for each.

// Writes the 8-bit form of the unit at `i` of n values; all lanes of its block
// take part.  Values from n on are zeros.
template <bool kWhole, typename T>
__device__ __forceinline__ void hold(const typename Units<T>::Unit& x,
                                     const float (&v)[Units<T>::kVec], int64_t i, int64_t n,
                                     int8_t* codes, uint8_t* exponents) {
  constexpr int N = Units<T>::kVec;
  const uint32_t e = exponent_of(block_max(x));
  uint32_t c[N / 4];
  encode(v, inverse_step(e), c);
  if (kWhole || i + N <= n) {
    put_codes(codes + i, c);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < n) codes[i + j] = static_cast<int8_t>(c[j / 4] >> (8 * (j % 4)));
  }
  if (i % kBlock == 0 && (kWhole || i < n)) exponents[i / kBlock] = static_cast<uint8_t>(e);
}
// The values of the unit at `i`, those from n on zeros.
template <bool kWhole, typename T>
__device__ __forceinline__ void fetch(const int8_t* codes, const uint8_t* exponents, int64_t i,
                                      int64_t n, uint32_t (&c)[Units<T>::kVec / 4], uint32_t& e) {
  constexpr int N = Units<T>::kVec;
  if (kWhole) {
    e = exponents[i / kBlock];
    get_codes(codes + i, c);
    return;
  }
  e = 1;
#pragma unroll
  for (int j = 0; j < N / 4; ++j) c[j] = 0;
  if (i < n) e = exponents[i / kBlock];
  if (i + N <= n) {
    get_codes(codes + i, c);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < n)
        c[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(codes[i + j])) << (8 * (j % 4));
  }
}
template <bool kWhole, typename T>
__device__ __forceinline__ typename Units<T>::Unit fetch(const T* x, int64_t i, int64_t n) {
  constexpr int N = Units<T>::kVec;
  if (kWhole || i + N <= n) return load_stream_any<N>(x + i);
  typename Units<T>::Unit u;
#pragma unroll
  for (int j = 0; j < N; ++j) u.v[j] = i + j < n ? x[i + j] : static_cast<T>(0.f);
  return u;
}
template <bool kWhole, bool kKeep = false, typename T>
__device__ __forceinline__ void put(T* x, int64_t i, int64_t n, const float (&v)[Units<T>::kVec]) {
  constexpr int N = Units<T>::kVec;
  typename Units<T>::Unit u;
#pragma unroll
  for (int j = 0; j < N; ++j) u.v[j] = narrow<T>(v[j]);
  if (kWhole || i + N <= n) {
    if (kKeep)
      store<N>(x + i, u);
    else
      store_stream_any<N>(x + i, u);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < n) x[i + j] = u.v[j];
  }
}

// Units to a lane, in flight together: 2 where few streams meet, 1 where many do.
// Of fp16, 8192 x 8192, with 2 and 1: forward 60 and 63 us, gated 91 and 87,
// gated backward 114 both (16384 rows more: 336 and 331), pack 35 and 37, unpack
// 36 and 32 (2048 rows: 13.2 and 8.7).  Outputs are written past the caches but
// for the ungated backward's, 72 against 78 us.
constexpr int kThreads = 256;
template <int K>
constexpr int kEachOf = K == MS_ACT_SWIGLU ? 1 : 2;

template <typename T, int kEach>
__device__ __forceinline__ bool block_within(int64_t n) {
  return (static_cast<int64_t>(blockIdx.x) + 1) * (kEach * kThreads * Units<T>::kVec) <= n;
}
// Where unit k of this lane begins.
template <typename T, int kEach>
__device__ __forceinline__ int64_t unit_at(int k) {
  return ((static_cast<int64_t>(blockIdx.x) * kEach + k) * kThreads + threadIdx.x) *
         Units<T>::kVec;
}

template <bool kWhole, typename T>
__device__ __forceinline__ void pack_block(const T* x, int64_t n, int8_t* codes,
                                           uint8_t* exponents) {
  constexpr int kEach = 2;
  constexpr int N = Units<T>::kVec;
  typename Units<T>::Unit u[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) u[k] = fetch<kWhole>(x, unit_at<T, kEach>(k), n);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = widen(u[k].v[j]);
    hold<kWhole, T>(u[k], v, unit_at<T, kEach>(k), n, codes, exponents);
  }
}
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_pack(const T* x, int64_t n, int8_t* codes, uint8_t* exponents) {
  if (block_within<T, 2>(n))
    pack_block<true, T>(x, n, codes, exponents);
  else
    pack_block<false, T>(x, n, codes, exponents);
}

template <bool kWhole, typename T>
__device__ __forceinline__ void unpack_block(const int8_t* codes, const uint8_t* exponents,
                                             int64_t n, T* out) {
  constexpr int kEach = 1;
  constexpr int N = Units<T>::kVec;
  uint32_t c[kEach][N / 4], e[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    fetch<kWhole, T>(codes, exponents, unit_at<T, kEach>(k), n, c[k], e[k]);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    float v[N];
    decode(c[k], step_of(e[k]), v);
    put<kWhole>(out, unit_at<T, kEach>(k), n, v);
  }
}
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_unpack(const int8_t* codes, const uint8_t* exponents, int64_t n, T* out) {
  if (block_within<T, 1>(n))
    unpack_block<true, T>(codes, exponents, n, out);
  else
    unpack_block<false, T>(codes, exponents, n, out);
}

// Rows that are not one after the other: units within a row (kRows 1), or any of
// which may lie across rows (2).
template <bool kWhole, typename T, int kRows>
__device__ __forceinline__ typename Units<T>::Unit fetch_rows(const ms_rows_t& m, int64_t i,
                                                              int64_t n) {
  constexpr int N = Units<T>::kVec;
  const T* x = static_cast<const T*>(m.data);
  if (kRows == 0) return fetch<kWhole>(x, i, n);
  typename Units<T>::Unit u;
  if (kRows == 1) {
    const int64_t at = kWhole || i < n ? i : 0, r = at / m.width;
    u = load_stream_any<N>(x + row_start(m, r) + (at - r * m.width));
    if (!kWhole && i >= n)
#pragma unroll
      for (int j = 0; j < N; ++j) u.v[j] = static_cast<T>(0.f);
    return u;
  }
  const int64_t at = kWhole || i < n ? i : 0;
  int64_t r = at / m.width, c = at - r * m.width;
  if (c + N <= m.width && (kWhole || i + N <= n))
    return load_stream_any<N>(x + row_start(m, r) + c);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    u.v[j] = i + j < n ? x[row_start(m, r) + c] : static_cast<T>(0.f);
    if (++c == m.width && i + j + 1 < n) c = 0, ++r;
  }
  return u;
}

template <bool kWhole, typename T, int K, int kRows>
__device__ __forceinline__ void act8_block(ms_rows_t h, ms_rows_t up, T* a, int8_t* codes,
                                           uint8_t* exponents, int8_t* up_codes,
                                           uint8_t* up_exponents) {
  constexpr int kEach = kEachOf<K>;
  constexpr int N = Units<T>::kVec;
  constexpr bool kGated = K == MS_ACT_SWIGLU;
  const int64_t n = h.n * h.width;
  typename Units<T>::Unit x[kEach], u[kGated ? kEach : 1];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    x[k] = fetch_rows<kWhole, T, kRows>(h, unit_at<T, kEach>(k), n);
    if constexpr (kGated) u[k] = fetch_rows<kWhole, T, kRows>(up, unit_at<T, kEach>(k), n);
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = unit_at<T, kEach>(k);
    float v[N], f[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = widen(x[k].v[j]);
    hold<kWhole, T>(x[k], v, i, n, codes, exponents);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = act<K, kFineOf<T, K, false>>(v[j]).f;
    if constexpr (kGated) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = widen(u[k].v[j]);
      hold<kWhole, T>(u[k], v, i, n, up_codes, up_exponents);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= v[j];
    }
    put<kWhole>(a, i, n, f);
  }
}
template <typename T, int K, int kRows>
__global__ void __launch_bounds__(kThreads)
    k_act8(ms_rows_t h, ms_rows_t up, T* a, int8_t* codes, uint8_t* exponents, int8_t* up_codes,
           uint8_t* up_exponents) {
  const int64_t n = h.n * h.width;
  if (block_within<T, kEachOf<K>>(n))
    act8_block<true, T, K, kRows>(h, up, a, codes, exponents, up_codes, up_exponents);
  else
    act8_block<false, T, K, kRows>(h, up, a, codes, exponents, up_codes, up_exponents);
}

template <bool kWhole, typename T, int K, bool kAgain>
__device__ __forceinline__ void act8_grad_block(const int8_t* codes, const uint8_t* exponents,
                                                const int8_t* up_codes,
                                                const uint8_t* up_exponents, const T* grad,
                                                int64_t n, T* dh, T* dup, T* a) {
  constexpr int kEach = kEachOf<K>;
  constexpr int N = Units<T>::kVec;
  constexpr bool kGated = K == MS_ACT_SWIGLU;
  uint32_t c[kEach][N / 4], e[kEach], uc[kGated ? kEach : 1][N / 4], ue[kGated ? kEach : 1];
  typename Units<T>::Unit g[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = unit_at<T, kEach>(k);
    fetch<kWhole, T>(codes, exponents, i, n, c[k], e[k]);
    if constexpr (kGated) fetch<kWhole, T>(up_codes, up_exponents, i, n, uc[k], ue[k]);
    g[k] = fetch<kWhole>(grad, i, n);
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = unit_at<T, kEach>(k);
    float x[N], u[N], d[N], du[N], f[N];
    decode(c[k], step_of(e[k]), x);
    if constexpr (kGated) decode(uc[k], step_of(ue[k]), u);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const Act y = act<K, kFineOf<T, K, true>>(x[j]);
      const float gj = widen(g[k].v[j]);
      if constexpr (kGated) {
        d[j] = gj * u[j] * y.df;
        du[j] = gj * y.f;
        f[j] = y.f * u[j];
      } else {
        d[j] = gj * y.df;
        f[j] = y.f;
      }
    }
    put<kWhole, !kGated>(dh, i, n, d);
    if constexpr (kGated) put<kWhole>(dup, i, n, du);
    if constexpr (kAgain) put<kWhole, !kGated>(a, i, n, f);
  }
}
template <typename T, int K, bool kAgain>
__global__ void __launch_bounds__(kThreads)
    k_act8_grad(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                const uint8_t* up_exponents, const T* grad, int64_t n, T* dh, T* dup, T* a) {
  if (block_within<T, kEachOf<K>>(n))
    act8_grad_block<true, T, K, kAgain>(codes, exponents, up_codes, up_exponents, grad, n, dh, dup,
                                        a);
  else
    act8_grad_block<false, T, K, kAgain>(codes, exponents, up_codes, up_exponents, grad, n, dh, dup,
                                         a);
}

// Blocks for n values; 0: too many.
template <typename T, int kEach>
unsigned blocks_for(int64_t n) {
  constexpr int64_t kValues = kThreads * kEach * Units<T>::kVec;
  const int64_t blocks = (n + kValues - 1) / kValues;
  return fits(blocks, kThreads) ? static_cast<unsigned>(blocks) : 0;
}

template <typename T, int K>
int act8_kind(const ms_rows_t& h, const ms_rows_t& up, void* a, int8_t* codes, uint8_t* exponents,
              int8_t* up_codes, uint8_t* up_exponents, hipStream_t s) {
  const unsigned blocks = blocks_for<T, kEachOf<K>>(h.n * h.width);
  if (!blocks) return MS_OPS_EINVAL;
  T* out = static_cast<T*>(a);
  auto dense = [](const ms_rows_t& m) {
    return m.n <= 1 || (m.inner >= m.n && m.inner_stride == m.width);
  };
  const bool gated = K == MS_ACT_SWIGLU;
  return launch(dense(h) && (!gated || dense(up))  ? k_act8<T, K, 0>
                : h.width % Units<T>::kVec == 0 ? k_act8<T, K, 1>
                                                : k_act8<T, K, 2>,
                blocks, kThreads, s, h, up, out, codes, exponents, up_codes, up_exponents);
}

template <typename T>
int act8_as(const ms_rows_t& h, const ms_rows_t& up, int kind, void* a, int8_t* codes,
            uint8_t* exponents, int8_t* up_codes, uint8_t* up_exponents, hipStream_t s) {
  switch (kind) {
    case MS_ACT_GELU:
      return act8_kind<T, MS_ACT_GELU>(h, up, a, codes, exponents, up_codes, up_exponents, s);
    case MS_ACT_GELU_TANH:
      return act8_kind<T, MS_ACT_GELU_TANH>(h, up, a, codes, exponents, up_codes, up_exponents, s);
    case MS_ACT_SILU:
      return act8_kind<T, MS_ACT_SILU>(h, up, a, codes, exponents, up_codes, up_exponents, s);
    default:
      return act8_kind<T, MS_ACT_SWIGLU>(h, up, a, codes, exponents, up_codes, up_exponents, s);
  }
}

template <typename T, int K>
int grad_kind(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
              const uint8_t* up_exponents, const void* grad, int64_t n, void* dh, void* dup,
              void* a, hipStream_t s) {
  const unsigned blocks = blocks_for<T, kEachOf<K>>(n);
  if (!blocks) return MS_OPS_EINVAL;
  const T* g = static_cast<const T*>(grad);
  T *d = static_cast<T*>(dh), *du = static_cast<T*>(dup), *out = static_cast<T*>(a);
  return launch(out ? k_act8_grad<T, K, true> : k_act8_grad<T, K, false>, blocks, kThreads, s, codes,
                exponents, up_codes, up_exponents, g, n, d, du, out);
}

template <typename T>
int act8_grad_as(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                 const uint8_t* up_exponents, const void* grad, int kind, int64_t n, void* dh,
                 void* dup, void* a, hipStream_t s) {
  switch (kind) {
    case MS_ACT_GELU:
      return grad_kind<T, MS_ACT_GELU>(codes, exponents, up_codes, up_exponents, grad, n, dh, dup,
                                       a, s);
    case MS_ACT_GELU_TANH:
      return grad_kind<T, MS_ACT_GELU_TANH>(codes, exponents, up_codes, up_exponents, grad, n, dh,
                                            dup, a, s);
    case MS_ACT_SILU:
      return grad_kind<T, MS_ACT_SILU>(codes, exponents, up_codes, up_exponents, grad, n, dh, dup,
                                       a, s);
    default:
      return grad_kind<T, MS_ACT_SWIGLU>(codes, exponents, up_codes, up_exponents, grad, n, dh,
                                         dup, a, s);
  }
}

bool good_kind(int32_t k) { return k >= MS_ACT_GELU && k <= MS_ACT_SWIGLU; }

template <typename T>
int pack_as(const void* x, int64_t n, int8_t* codes, uint8_t* exponents, hipStream_t s) {
  const unsigned blocks = blocks_for<T, 2>(n);
  if (!blocks) return MS_OPS_EINVAL;
  return launch(k_pack<T>, blocks, kThreads, s, static_cast<const T*>(x), n, codes, exponents);
}
template <typename T>
int unpack_as(const int8_t* codes, const uint8_t* exponents, int64_t n, void* out,
              hipStream_t s) {
  const unsigned blocks = blocks_for<T, 1>(n);
  if (!blocks) return MS_OPS_EINVAL;
  return launch(k_unpack<T>, blocks, kThreads, s, codes, exponents, n, static_cast<T*>(out));
}

}  // namespace

extern "C" int ms_pack8(const void* x, int32_t dtype, int64_t n, int8_t* codes, uint8_t* exponents,
                        void* stream) {
  if (!good_dtype(dtype) || n < 0 || !countable(n)) return MS_OPS_EINVAL;
  if (n == 0) return MS_OPS_OK;
  if (!x || !codes || !exponents) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MS_OPS_F32: return pack_as<float>(x, n, codes, exponents, s);
    case MS_OPS_F16: return pack_as<f16>(x, n, codes, exponents, s);
    default: return pack_as<bf16>(x, n, codes, exponents, s);
  }
}

extern "C" int ms_unpack8(const int8_t* codes, const uint8_t* exponents, int64_t n, int32_t dtype,
                          void* out, void* stream) {
  if (!good_dtype(dtype) || n < 0 || !countable(n)) return MS_OPS_EINVAL;
  if (n == 0) return MS_OPS_OK;
  if (!out || !codes || !exponents) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MS_OPS_F32: return unpack_as<float>(codes, exponents, n, out, s);
    case MS_OPS_F16: return unpack_as<f16>(codes, exponents, n, out, s);
    default: return unpack_as<bf16>(codes, exponents, n, out, s);
  }
}

extern "C" int ms_act8(const ms_rows_t* h, const ms_rows_t* up, int32_t kind, void* a,
                       int8_t* codes, uint8_t* exponents, int8_t* up_codes, uint8_t* up_exponents,
                       void* stream) {
  const bool gated = kind == MS_ACT_SWIGLU;
  if (!good_kind(kind) || !good_rows(h) || gated != (up != nullptr)) return MS_OPS_EINVAL;
  if (gated && (!good_rows(up) || up->n != h->n || up->width != h->width || up->dtype != h->dtype))
    return MS_OPS_EINVAL;
  if (h->n == 0 || h->width == 0) return MS_OPS_OK;
  if (!a || !codes || !exponents || (gated && (!up_codes || !up_exponents))) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const ms_rows_t u = gated ? *up : ms_rows_t{};
  switch (h->dtype) {
    case MS_OPS_F32:
      return act8_as<float>(*h, u, kind, a, codes, exponents, up_codes, up_exponents, s);
    case MS_OPS_F16:
      return act8_as<f16>(*h, u, kind, a, codes, exponents, up_codes, up_exponents, s);
    default:
      return act8_as<bf16>(*h, u, kind, a, codes, exponents, up_codes, up_exponents, s);
  }
}

extern "C" int ms_act8_grad(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                            const uint8_t* up_exponents, const void* grad, int32_t dtype,
                            int32_t kind, int64_t n, void* dh, void* dup, void* a, void* stream) {
  const bool gated = kind == MS_ACT_SWIGLU;
  if (!good_kind(kind) || !good_dtype(dtype) || n < 0 || !countable(n)) return MS_OPS_EINVAL;
  if (n == 0) return MS_OPS_OK;
  if (!codes || !exponents || !grad || !dh) return MS_OPS_EINVAL;
  if (gated != (up_codes != nullptr) || gated != (up_exponents != nullptr) ||
      gated != (dup != nullptr))
    return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MS_OPS_F32:
      return act8_grad_as<float>(codes, exponents, up_codes, up_exponents, grad, kind, n, dh, dup,
                                 a, s);
    case MS_OPS_F16:
      return act8_grad_as<f16>(codes, exponents, up_codes, up_exponents, grad, kind, n, dh, dup, a,
                               s);
    default:
      return act8_grad_as<bf16>(codes, exponents, up_codes, up_exponents, grad, kind, n, dh, dup,
                                a, s);
  }
}
