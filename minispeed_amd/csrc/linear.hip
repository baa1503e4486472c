// Log probabilities of given tokens under softmax(scale * hidden * weight^T),
// and their gradients, without storing the logits.
//
//   x[t, v] = scale * hidden[t] . weight[v],  lse[t] = log sum over v of exp x[t, v]
//   logprob[t] = x[t, y] - lse[t]
//   d[t, v] = g[t] 1[v = y] + (l[t] - g[t]) p[t, v],   p = exp(x - lse),
//             g, l the gradients of logprob and lse
//   dhidden = scale * d weight,   dweight = scale * d^T hidden
//
// Forward, one product (product.h) with the vocabulary along m: its epilogue takes each
// token's maximum and sum of exponentials over the wave's rows, and a second kernel
// joins those partial sums.  Backward, the vocabulary is gone through in pieces: the
// piece's logits are computed again and left as d, in the operands' 16-bit type; then
// come the two products with d.  Four products' work in all for what needs at least
// three, and one piece of d (kPiece bytes at most) in place of the logits.
//
// Numbers.  Products of 16-bit values are exact in the fp32 sums.  d is rounded once
// to the operands' type, as the products take it: half an ulp of each term, so that bf16
// gradients are off by 0.0024 of their norm where rounding the results alone leaves 0.0017 (two
// planes of d would make six products of the four).  In fp16 a row of d is scaled by a power of two that
// brings its bound below 2^15 (p reaches down to 2^-20 over large vocabularies, and g is
// an inverse count of tokens); dhidden's rows are scaled back, and dweight takes its
// scales from a copy of hidden multiplied by them, lifted as far as fp16 goes: exactly but for
// underflow below 2^-40 of the largest row's gradient times its largest value, which is
// where the results themselves underflow if that row's do not overflow.
// 32-bit operands of many tokens are split into three bf16 planes of 8 bits each (x = a + b + c,
// exactly), and six products of planes are summed; what is left out is below 2^-22 of
// the terms.  The matrix units' own 32-bit products have a sixteenth of the bf16 rate, and are
// for few tokens and small products.
//
// exp and log are taken in units of log 2.
//
// Measured: 8192 x 2048 x 50257 fp16 forward 1.51-1.57 ms, 1080-1120 TFLOP/s (the product alone, by the
// library, 1.56 ms).  4 x 4096 x 128256 bf16 187 us, 5.6 TB/s, reading the
// weight.  Backward 16384 x 768 x 50257 bf16 3.9-4.0 ms (four pieces: d 390 us, 820 TFLOP/s
// as its 12 steps of k do not hide the exponentials and stores; both products 595 us, 1080
// TFLOP/s), 2048 x 4096 x 128256 5.7 ms (1130 TFLOP/s over all).
#include "product.h"

#include <algorithm>

namespace ops {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int64_t kMaxWidth = 1 << 20;
constexpr int64_t kMaxRows = INT32_MAX - 1024;     // a tile behind the last row stays in 32 bits
constexpr int64_t kPiece = int64_t{512} << 20;     // bytes of d at a time

// What a token's row of d is made of, by k_rows.
struct __attribute__((aligned(16))) row_t {
  float lse2;       // lse in units of log 2
  float soft;       // (l - g) * up: the factor of p
  float given;      // g * up: what the token's own column has more
  float down;       // 1 / up, a power of two
};

__device__ __forceinline__ float swap_halves(float x) { return __shfl_xor(x, 32); }

// ---------------------------------------------------------------------------
// Epilogues.  acc[i][j][r] is C[m0 + 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4,
// n0 + 32 j + lane % 32].

// Per token: maximum and sum over the wave's rows of the vocabulary.
struct sum_epilogue {
  float2* parts;       // [part][tokens]: maximum in units of log 2, sum relative to it
  float* picked;       // [tokens]: the given token's logit
  ms_tokens_t targets;
  float scale;

  template <int MI, int NI>
  __device__ void store(const f32x16 (&acc)[MI][NI], int m0, int n0, int part, int, int lane, int m,
                        int n) const {
    const int half = 4 * (lane >> 5), left = m - m0;
    const float unit = scale * kLog2e;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = n0 + j * 32 + (lane & 31);
      const int64_t y = t < n ? token(targets, t) - m0 : -1;
      if (y >= 0 && y < MI * 32 && (static_cast<int>(y) & 4) == half) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (i * 32 + 8 * (r / 4) + half + r % 4 == y) x = acc[i][j][r];
        picked[t] = x * scale;
      }
      // the scale can be negative, so the largest product need not be the largest logit
      float most = -__builtin_inff(), sum = 0.0f;
      if (left >= MI * 32) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, acc[i][j][r] * unit);
        most = fmaxf(most, swap_halves(most));
        const float base = most == -__builtin_inff() ? 0.0f : most;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], unit, -base));
      } else {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (i * 32 + 8 * (r / 4) + half + r % 4 < left) most = fmaxf(most, acc[i][j][r] * unit);
        most = fmaxf(most, swap_halves(most));
        const float base = most == -__builtin_inff() ? 0.0f : most;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (i * 32 + 8 * (r / 4) + half + r % 4 < left)
              sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], unit, -base));
      }
      sum += swap_halves(sum);
      if (lane < 32 && t < n) parts[static_cast<int64_t>(part) * n + t] = make_float2(most, sum);
    }
  }
};

// Four values of a type as two words.
template <typename T>
struct Quad {
  uint32_t w[2];
  __device__ explicit Quad(const T (&v)[4]) { __builtin_memcpy(w, v, sizeof(w)); }
};

// A piece's columns of d: d[t, m], dense rows of ld elements; planes of bf16 for fp32.  Two lanes
// that have one token change places with half of their values, so that each stores 16 bytes.
template <typename T, int Planes>
struct soft_epilogue {
  T* d;
  int64_t ld, plane;
  const row_t* rows;
  ms_tokens_t targets;
  float scale;
  int32_t first;         // the piece's first token of the vocabulary

  template <int MI, int NI>
  __device__ void store(const f32x16 (&acc)[MI][NI], int m0, int n0, int, int, int lane, int m,
                        int n) const {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = n0 + j * 32 + (lane & 31);
      const row_t row = rows[min(t, n - 1)];
      const int64_t y = token(targets, min(t, n - 1)) - first - m0;
      // The given token, and what is behind the vocabulary's end, are few tiles' concern.
      if (__any(y >= 0 && y < MI * 32) || m - m0 < MI * 32)
        put<MI, true>(&acc[0][j], NI, m0, t, lane, m, n, row, y);
      else
        put<MI, false>(&acc[0][j], NI, m0, t, lane, m, n, row, y);
    }
  }

  template <int MI, bool Special>
  __device__ __forceinline__ void put(const f32x16* acc, int step, int m0, int t, int lane, int m, int n,
                                      const row_t& row, int64_t y) const {
    const int half = 4 * (lane >> 5);
    const float unit = scale * kLog2e;
    const int where = y >= 0 && y < MI * 32 ? static_cast<int>(y) : -1, left = m - m0;
    // rows without a gradient are zeros, whatever their logits are
    const uint32_t keep = row.soft == 0.0f && row.given == 0.0f ? 0u : ~0u;
    if constexpr (sizeof(T) == 4) {
      if (t >= n) return;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          Pack<T, 4> o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = i * 32 + q * 8 + e + half;
            float v = __builtin_amdgcn_exp2f(fmaf(acc[i * step][q * 4 + e], unit, -row.lse2)) * row.soft;
            if (Special && at == where) v += row.given;
            o.v[e] = (Special && at >= left) || !keep ? 0.0f : v;
          }
          ops::store<4>(d + t * ld + m0 + i * 32 + q * 8 + half, o);
        }
      return;
    }
    T* out = d + t * ld + m0 + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        uint32_t words[2][Planes][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[4];
          T o[Planes][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = i * 32 + (q + h) * 8 + e + half;
            v[e] = __builtin_amdgcn_exp2f(fmaf(acc[i * step][(q + h) * 4 + e], unit, -row.lse2)) * row.soft;
            if (Special) {
              if (at == where) v[e] += row.given;
              if (at >= left) v[e] = 0.0f;
            }
#pragma unroll
            for (int s = 0; s < Planes; ++s) {
              o[s][e] = narrow<T>(v[e]);
              if (s + 1 < Planes) v[e] -= widen(o[s][e]);
            }
          }
#pragma unroll
          for (int s = 0; s < Planes; ++s) {
            const Quad<T> x(o[s]);
            words[h][s][0] = x.w[0] & keep;
            words[h][s][1] = x.w[1] & keep;
          }
        }
#pragma unroll
        for (int s = 0; s < Planes; ++s) {
          u32x4 r;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const auto swapped =
                __builtin_amdgcn_permlane32_swap(words[0][s][k], words[1][s][k], false, false);
            r[k] = swapped[0];
            r[2 + k] = swapped[1];
          }
          if (t < n) *reinterpret_cast<u32x4*>(out + s * plane + i * 32 + q * 8) = r;
        }
        __builtin_amdgcn_sched_barrier(0);      // (all at once they would not fit in the registers)
      }
  }
};

// out[n, m]: final values of type T, or fp32 partial sums, one buffer for each split.
template <typename T>
struct out_epilogue {
  T* out;                // final where `parts` is null
  float* parts;          // [split][n][m]
  const row_t* rows;     // final: each n's factor, or null
  const float* factor;   // final: one factor, or null
  float scale;
  int32_t add;           // parts: to what is there

  template <int MI, int NI>
  __device__ void store(const f32x16 (&acc)[MI][NI], int m0, int n0, int, int split, int lane, int m,
                        int n) const {
    const float all = factor ? *factor * scale : scale;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = n0 + j * 32 + (lane & 31);
      const float by = rows ? rows[min(t, n - 1)].down * all : all;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          if (parts) {
            put_sums(acc[i][j], q, m0 + i * 32, t, split, lane, m, n);
            put_sums(acc[i][j], q + 1, m0 + i * 32, t, split, lane, m, n);
          } else {
            put(acc[i][j], q, m0 + i * 32, t, lane, m, n, by);
          }
        }
    }
  }

  __device__ __forceinline__ void put_sums(const f32x16& acc, int q, int m0, int t, int split, int lane,
                                           int m, int n) const {
    const int at = m0 + q * 8 + 4 * (lane >> 5);
    if (t >= n || at >= m) return;
    float* p = parts + (static_cast<int64_t>(split) * n + t) * m + at;
    if (at + 4 <= m) {
      Pack<float, 4> x;
      if (add) x = load<4>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v[e] = (add ? x.v[e] : 0.0f) + acc[q * 4 + e];
      ops::store<4>(p, x);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at + e < m) p[e] = (add ? p[e] : 0.0f) + acc[q * 4 + e];
    }
  }

  // Rows 8 q to 8 q + 15 of a square.  2-byte values: two lanes of one n change places with half of
  // them, so that each stores 16 bytes.
  __device__ __forceinline__ void put(const f32x16& acc, int q, int m0, int t, int lane, int m, int n,
                                      float by) const {
    constexpr int V = 16 / sizeof(T);
    T x[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] = narrow<T>(acc[(q + h) * 4 + e] * by);
#pragma unroll
    for (int h = 0; h < 8 / V; ++h) {
      Pack<T, V> o;
      int at;
      if constexpr (V == 8) {
        const Quad<T> a(x[0]), b(x[1]);
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const auto swapped = __builtin_amdgcn_permlane32_swap(a.w[k], b.w[k], false, false);
          r[k] = swapped[0];
          r[2 + k] = swapped[1];
        }
        __builtin_memcpy(&o, r, 16);
        at = m0 + 8 * (q + (lane >> 5));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = x[h][e];
        at = m0 + (q + h) * 8 + 4 * (lane >> 5);
      }
      if (t >= n) continue;
      T* p = out + static_cast<int64_t>(t) * m + at;
      if (at + V <= m) {
        ops::store<V>(p, o);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (at + e < m) p[e] = o.v[e];
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Around the products.

// Joins a token's partial sums.  `lanes` threads (a power of two up to 256) to a token.
__global__ __launch_bounds__(256) void k_join(const float2* parts, const float* picked, int64_t count,
                                              int64_t n, int lanes, ms_tokens_t targets, int64_t vocab,
                                              int64_t ignore_index, float* logprob, float* lse) {
  __shared__ float2 held[256];
  const int each = 256 / lanes, which = threadIdx.x % each, lane = threadIdx.x / each;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * each + which;
  float most = -__builtin_inff(), sum = 0.0f;
  if (t < n) {
#pragma unroll 8
    for (int64_t k = lane; k < count; k += lanes) {
      const float2 x = parts[k * n + t];
      const float top = fmaxf(most, x.x), base = top == -__builtin_inff() ? 0.0f : top;
      sum = sum * __builtin_amdgcn_exp2f(most - base) + x.y * __builtin_amdgcn_exp2f(x.x - base);
      most = top;
    }
  }
  held[threadIdx.x] = make_float2(most, sum);
  for (int step = lanes / 2; step; step /= 2) {
    __syncthreads();
    if (lane < step) {
      const float2 x = held[threadIdx.x + step * each];
      const float top = fmaxf(most, x.x), base = top == -__builtin_inff() ? 0.0f : top;
      sum = sum * __builtin_amdgcn_exp2f(most - base) + x.y * __builtin_amdgcn_exp2f(x.x - base);
      most = top;
      held[threadIdx.x] = make_float2(most, sum);
    }
  }
  if (lane == 0 && t < n) {
    const float base = most == -__builtin_inff() ? 0.0f : most;
    const float l = (base + __builtin_amdgcn_logf(sum)) * kLn2;
    const int64_t y = token(targets, t);
    float p;
    if (y == ignore_index) {
      p = 0.0f;
    } else if (y < 0 || y >= vocab) {
      p = quiet_nan();
    } else {
      p = l == -__builtin_inff() ? l : picked[t] - l;
    }
    logprob[t] = p;
    lse[t] = l;
  }
}

// Whether a row's d is made of finite numbers that are not all zeros.
__device__ __forceinline__ bool lifts(float bound) { return bound > 0.0f && bound < __builtin_inff(); }

// The power of two that brings a row's d below 2^15, given the larger one of the two terms that
// meet in it; 0 for rows of zeros, infinities and NaN.  (Numbers below 2^-87, the subnormal ones
// among them, stay as far below 2^14.)
__device__ __forceinline__ int lift(float bound) {
  const int e = static_cast<int>(__float_as_uint(bound) >> 23 & 255);
  return lifts(bound) ? min(13 + 127 - e, 100) : 0;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((e + 127) << 23); }

// What the row numbers follow from.
struct rows_args {
  const float *lse, *grad_logprob, *grad_lse;
  ms_tokens_t targets;
  int64_t vocab, ignore_index;
  int32_t lifted;          // fp16
};

// A token's numbers; `up`, the power of two in them, is kNoLift where the row's scale does not matter.
constexpr int kNoLift = INT32_MAX;
__device__ __forceinline__ row_t row_numbers(const rows_args& a, int64_t t, int& up) {
  // (all loads at once: none waits for the token)
  const float given = a.grad_logprob ? a.grad_logprob[t] : 0.0f, of = a.lse[t];
  float l = a.grad_lse ? a.grad_lse[t] : 0.0f;
  const int64_t y = token(a.targets, t);
  float g = y != a.ignore_index ? given : 0.0f;
  if (y != a.ignore_index && (y < 0 || y >= a.vocab) && a.grad_logprob) g = quiet_nan();
  if (of == -__builtin_inff()) g = l = 0.0f;
  const float soft = l - g, bound = fmaxf(fabsf(soft), fabsf(g));
  const int by = a.lifted ? lift(bound) : 0;
  up = lifts(bound) ? by : kNoLift;
  return {of == -__builtin_inff() ? 0.0f : of * kLog2e, soft * pow2(by), g * pow2(by), pow2(-by)};
}

// Row numbers for the backward pass.
__global__ __launch_bounds__(256) void k_rows(rows_args a, row_t* rows) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  int up;
  if (t < a.targets.n) rows[t] = row_numbers(a, t, up);
}

// The same for an fp16 dweight.  Its sums over the tokens have one scale, so what d's row is lifted
// by, hidden's gives way for: hidden[t] 2^(low - up[t]).  `low` is the largest power of two for
// which no such row passes fp16's largest number: the least of up[t] + 30 - e, e the exponent bits of
// the row's largest value, so that all of fp16's 40 powers of two are there for rows whose
// gradients are smaller than others'.  16 lanes to a token; each block's least goes to
// least[block].  (3.7 us of 28.9 for 1024 x 256 x 512, where one block without a look at hidden took
// 2.5; 16384 x 768 x 50257 is as fast as by that.)
constexpr int kScaleBlocks = 512, kScaleThreads = 1024, kScaleRows = kScaleThreads / 16, kMostLow = 126;

// The least of the numbers of a block of W waves, in every thread.
template <int W>
__device__ __forceinline__ int block_least(int low, int (&held)[W]) {
#pragma unroll
  for (int s = 32; s; s /= 2) low = min(low, __shfl_xor(low, s));
  if ((threadIdx.x & 63) == 0) held[threadIdx.x >> 6] = low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) low = min(low, held[w]);
  return low;
}

// Chunk c .. c + V - 1 of a row, zeros behind its end.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_chunk(const ms_rows_t& from, int64_t r, int64_t c) {
  const T* p = static_cast<const T*>(from.data) + row_start(from, r) + c;
  Pack<T, V> x;
  if (c + V <= from.width) {
    x = load<V>(p);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = c + e < from.width ? p[e] : static_cast<T>(0.0f);
  }
  return x;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__global__ __launch_bounds__(kScaleThreads) void k_scaled_rows(rows_args a, ms_rows_t hidden, row_t* rows,
                                                               int* least) {
  __shared__ int held[kScaleThreads / 64];
  const int lane = threadIdx.x & 15;
  const int64_t n = a.targets.n;
  int low = kMostLow;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kScaleRows + threadIdx.x / 16; t < n;
       t += static_cast<int64_t>(gridDim.x) * kScaleRows) {
    const uint16_t* p = static_cast<const uint16_t*>(hidden.data) + row_start(hidden, t);
    const int width = static_cast<int>(hidden.width);
    // By pairs of 2-byte numbers: adding 2^10 to one and dropping its sign puts its size in order
    // behind the infinities and NaN, which have no say.
    u16x2 most = {0x400, 0x400};
    auto take = [&](u16x2 x) {
      most = __builtin_elementwise_max(most, (x + u16x2{0x400, 0x400}) & u16x2{0x7fff, 0x7fff});
    };
    if (width >= 8) {
      // (what would pass the row's end is its last 8 values again)
      for (int c = lane * 8; c < width; c += 4 * 128) {
        Pack<u16x2, 4> x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = load<4>(reinterpret_cast<const u16x2*>(p + min(c + k * 128, width - 8)));
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) take(x[k].v[e]);
      }
    } else if (lane < width) {
      take(u16x2{p[lane], p[lane]});
    }
    int up, size = max(most[0], most[1]) - 0x400;
    const row_t row = row_numbers(a, t, up);
    if (lane == 0) rows[t] = row;
#pragma unroll
    for (int s = 8; s; s /= 2) size = max(size, __shfl_xor(size, s));
    if (size && up != kNoLift) low = min(low, up + 30 - (size >> 10));
  }
  low = block_least(low, held);
  if (threadIdx.x == 0) least[blockIdx.x] = low;
}

// A matrix as the products take it: rows at `ld`, zeros behind `width`.
template <typename T>
__global__ __launch_bounds__(256) void k_layout(ms_rows_t from, int64_t ld, T* to) {
  constexpr int V = 16 / sizeof(T);
  const int64_t chunks = ld / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= from.n * chunks) return;
  const int64_t r = i / chunks, c = (i - r * chunks) * V;
  ops::store<V>(to + r * ld + c, load_chunk<T, V>(from, r, c));
}

// hidden with its rows' scales, and the factor 2^-low that dweight takes back.
__global__ __launch_bounds__(256) void k_scaled_layout(ms_rows_t from, int64_t ld, const row_t* rows,
                                                       const int* least, int count, f16* to,
                                                       float* factor) {
  __shared__ int held[4];
  const int64_t chunks = ld / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const bool there = i < from.n * chunks;
  const int64_t r = there ? i / chunks : 0, c = there ? (i - r * chunks) * 8 : 0;
  Pack<f16, 8> x = load_chunk<f16, 8>(from, r, c);
  const row_t row = rows[r];
  int low = kMostLow;
#pragma unroll
  for (int k = 0; k < kScaleBlocks / 256; ++k)
    low = min(low, least[min(static_cast<int>(threadIdx.x) + k * 256, count - 1)]);
  low = block_least(low, held);
  if (i == 0) *factor = pow2(-low);
  if (!there) return;
  // (a row without a gradient or with one that is not finite was lifted by nothing)
  const float by = lifts(fmaxf(fabsf(row.soft), fabsf(row.given))) ? row.down * pow2(low) : 1.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) x.v[e] = narrow<f16>(widen(x.v[e]) * by);
  ops::store<8>(to + r * ld + c, x);
}

// Three planes of bf16: the leading 8 bits of each value, the next 8, the rest.  Cut off
// instead of rounded, so that nothing overflows and the rest is exact.
__global__ __launch_bounds__(256) void k_planes(ms_rows_t from, int64_t ld, int64_t plane,
                                                uint16_t* to) {
  const int64_t chunks = ld / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= from.n * chunks) return;
  const int64_t r = i / chunks, c = (i - r * chunks) * 8;
  const float* p = static_cast<const float*>(from.data) + row_start(from, r) + c;
  Pack<uint16_t, 8> out[3];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = c + e < from.width ? p[e] : 0.0f;
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const uint32_t cut = __float_as_uint(x) & 0xffff0000u;
      out[s].v[e] = static_cast<uint16_t>(cut >> 16);
      // (an infinity or NaN has nothing behind it)
      x = (cut & 0x7f800000u) == 0x7f800000u ? 0.0f : x - __uint_as_float(cut);
    }
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) ops::store<8>(to + s * plane + r * ld + c, out[s]);
}

// Sums of `count` partial buffers, scaled and rounded.
template <typename T>
__global__ __launch_bounds__(256) void k_fold(const float* parts, int count, int64_t n, int64_t width,
                                              const row_t* rows, const float* factor, float scale,
                                              T* out) {
  const int64_t all = n * width;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= all) return;
  const float by = factor ? *factor * scale : scale;
  if (i + 4 <= all) {
    Pack<float, 4> sum = load<4>(parts + i);
    for (int s = 1; s < count; ++s) {
      const Pack<float, 4> x = load<4>(parts + s * all + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum.v[e] += x.v[e];
    }
    Pack<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o.v[e] = narrow<T>(sum.v[e] * (rows ? rows[(i + e) / width].down * by : by));
    ops::store<4>(out + i, o);
  } else {
    for (int64_t j = i; j < all; ++j) {
      float sum = parts[j];
      for (int s = 1; s < count; ++s) sum += parts[s * all + j];
      out[j] = narrow<T>(sum * (rows ? rows[j / width].down * by : by));
    }
  }
}

// No tokens: a gradient of zeros.
__global__ __launch_bounds__(256) void k_zero(uint16_t* to, int64_t n) {
  int64_t i = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
  for (int e = 0; e < 4; ++e, i += 256)
    if (i < n) to[i] = 0;
}

// ---------------------------------------------------------------------------
// Host.

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }

// How the products' tiles are cut.  Large ones, one block to a CU, have the highest rate (1230
// TFLOP/s at 16384 x 2048 x 4096, medium ones 1130), but leave more of the chip idle at
// the end and beside a small product.
enum Cut { kLarge, kMedium, kFew };
typedef Tiles<256, 256, 2, 4> Large;
typedef Tiles<128, 128, 2, 2> Medium;
typedef Tiles<128, 32, 4, 1> Few;

struct Shape {
  int m, n, wm, threads, slots;    // slots: blocks that the chip runs at a time
  double step, alone, rest;        // us of a block for 64 k beside others and by itself, and
                                   // for what is around them
};
constexpr Shape kShapes[] = {{256, 256, 2, 512, 256, 1.75, 1.75, 4.0},
                             {128, 128, 2, 256, 512, 0.95, 0.65, 3.0},
                             {128, 32, 4, 256, 1024, 1.2, 0.45, 2.0}};

// us of a block among `blocks` for so many steps.
double block_us(const Shape& s, int64_t blocks, int64_t steps) {
  const double fill = std::min(1.0, static_cast<double>(blocks) / s.slots);
  return steps * std::max(s.alone, s.step * fill) + s.rest;
}

int64_t tiles_of(int64_t m, int64_t n, Cut c) {
  return ceil_div(m, kShapes[c].m) * ceil_div(n, kShapes[c].n);
}

// The cut of one product without parts of k: the one whose blocks are done first.  (32-bit
// products have small tiles alone, for few tokens.)
Cut cut_of(int64_t m, int64_t n, int64_t steps, bool wide) {
  Cut best = kFew;
  double least = 1e300;
  for (Cut c : {kLarge, kMedium, kFew}) {
    if (wide && c != kFew) continue;
    const Shape& s = kShapes[c];
    const int64_t tiles = tiles_of(m, n, c);
    const double us = static_cast<double>(ceil_div(tiles, s.slots)) * block_us(s, tiles, steps);
    if (us < least) least = us, best = c;
  }
  return best;
}

// A product whose k can be cut into parts (m = 0: none): its size, 64 k at a time, and whether its
// sums go through memory also if there is one part.
struct Job {
  int64_t m, n, steps;
  bool summed;
};

struct Plan {
  Cut cut;
  int splits[2];
};

// The cut and parts with which two products in one launch are done first.  One by itself takes
// whole rounds of blocks; behind another its blocks start as those end, and half a block's time
// is left over.  Each part's sums are written and read at 2.5 TB/s, and joined by a launch of
// 5 us (summed ones are joined anyhow).
Plan plan_of(const Job& p, const Job& q, bool wide = false) {
  constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 16, 32, 64};
  Plan best{kFew, {1, 1}};
  double least = 1e300;
  const auto joining = [](const Job& j, int splits) {
    double us = 0.0;
    if (splits > 1 || j.summed) us += splits * 8e-6 / 2.5 * static_cast<double>(j.m * j.n);
    return splits > 1 && !j.summed ? us + 5.0 : us;
  };
  for (Cut c : {kLarge, kMedium, kFew}) {
    if (wide && c != kFew) continue;
    // One step of k is stores with next to nothing beside them: two blocks to a CU take turns at
    // them (dweight of 4 x 4096 x 128256 bf16: the whole call 702 us, 751 by large tiles; at 12
    // steps large ones are ahead).
    if (c == kLarge && p.steps == 1 && !q.m) continue;
    const Shape& s = kShapes[c];
    const int64_t tp = tiles_of(p.m, p.n, c), tq = q.m ? tiles_of(q.m, q.n, c) : 0;
    for (int i : kSplits) {
      if (i > 1 && p.steps / i < 8) break;
      const double more1 = joining(p, i);
      for (int j : kSplits) {
        if (j > 1 && (!q.m || q.steps / j < 8)) break;
        double us;
        if (q.m) {
          const double us1 = block_us(s, tp * i + tq * j, ceil_div(p.steps, i));
          const double us2 = block_us(s, tp * i + tq * j, ceil_div(q.steps, j));
          us = std::max(std::max(us1, us2),
                        (tp * i * us1 + tq * j * us2) / s.slots + 0.5 * us2) + joining(q, j);
        } else {
          us = ceil_div(tp * i, s.slots) * block_us(s, tp * i, ceil_div(p.steps, i));
        }
        us += more1;
        if (us < least) least = us, best = {c, {i, j}};
      }
    }
  }
  return best;
}

int64_t set_tiles(product_args& p, Cut c) {
  p.tiles_m = static_cast<int32_t>(ceil_div(p.a.rows, kShapes[c].m));
  p.tiles_n = static_cast<int32_t>(ceil_div(p.b.rows, kShapes[c].n));
  return int64_t{p.tiles_m} * p.tiles_n * p.splits;
}

template <typename T, Side SA, Side SB, typename E>
int run_product(Cut c, product_args p, const E& epilogue, hipStream_t s) {
  const int64_t blocks = set_tiles(p, c);
  if (!fits(blocks, kShapes[c].threads)) return MS_OPS_EINVAL;
  if constexpr (sizeof(T) == 4)
    return launch(k_product<T, Few, SA, SB, E>, blocks, Few::kThreads, s, p, epilogue);
  else if (c == kLarge)
    return launch(k_product<T, Large, SA, SB, E>, blocks, Large::kThreads, s, p, epilogue);
  else if (c == kMedium)
    return launch(k_product<T, Medium, SA, SB, E>, blocks, Medium::kThreads, s, p, epilogue);
  else
    return launch(k_product<T, Few, SA, SB, E>, blocks, Few::kThreads, s, p, epilogue);
}

template <typename T, Side SB1, Side SB2, typename E>
int run_products(Cut c, product_args p, const E& e, product_args q, const E& f, hipStream_t s) {
  const int64_t first = set_tiles(p, c), blocks = first + set_tiles(q, c);
  if (!fits(blocks, kShapes[c].threads)) return MS_OPS_EINVAL;
  const uint32_t n = static_cast<uint32_t>(first);
  if (c == kLarge)
    return launch(k_products<T, Large, SB1, SB2, E>, blocks, Large::kThreads, s, p, e, q, f, n);
  if (c == kMedium)
    return launch(k_products<T, Medium, SB1, SB2, E>, blocks, Medium::kThreads, s, p, e, q, f, n);
  return launch(k_products<T, Few, SB1, SB2, E>, blocks, Few::kThreads, s, p, e, q, f, n);
}

// Space cut from the workspace, or only counted while `at` is null.
struct Space {
  char* at;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = at ? reinterpret_cast<T*>(at + used) : nullptr;
    used += round_up(n * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};

bool good_sizes(const ms_rows_t* hidden, const ms_rows_t* weight) {
  return good_rows(hidden) && good_rows(weight) && hidden->dtype == weight->dtype &&
         hidden->width == weight->width && hidden->width >= 1 && hidden->width <= kMaxWidth &&
         weight->n >= 1 && hidden->n <= kMaxRows && weight->n <= kMaxRows && countable(hidden->n, weight->n);
}

// Few tokens of 32 bits, and small products, are multiplied as they are, at 120 TFLOP/s where six
// products of planes have 190, but without the planes: of 1920 x 45061, 1 token forward 81 us
// (396 by planes), 256 tokens 363 (656), their gradients 1106 (1395); 256 x 256 x 2000 12.5
// (27.4).  Between 384 and 512 tokens the planes' gradients are as fast.
constexpr int64_t kAsTheyAre = 384;
constexpr double kSmallProduct = 1 << 29;
bool as_it_is(const ms_rows_t& hidden, const ms_rows_t& weight) {
  return hidden.dtype != MS_OPS_F32 || hidden.n <= kAsTheyAre ||
         static_cast<double>(hidden.n) * hidden.width * weight.n <= kSmallProduct;
}

// Whether the products can take the matrix as it lies: rows on 16 bytes.
bool lies_well(const ms_rows_t& m) {
  const int64_t v = 16 / dtype_bytes(m.dtype);
  // (one row has no stride)
  return m.width % v == 0 && reinterpret_cast<uintptr_t>(m.data) % 16 == 0 &&
         (m.n == 1 || (m.inner >= m.n && m.inner_stride % v == 0 && m.inner_stride >= m.width &&
                       m.inner_stride <= kMaxWidth));
}

template <typename T>
int lay_out(const ms_rows_t& m, int64_t ld, void* to, hipStream_t s) {
  const int64_t blocks = ceil_div(m.n * (ld * static_cast<int64_t>(sizeof(T)) / 16), 256);
  if (!fits(blocks, 256)) return MS_OPS_EINVAL;
  return launch(k_layout<T>, blocks, 256, s, m, ld, static_cast<T*>(to));
}

// The matrix as an operand, laid out in the workspace where it does not lie well, or by planes.
operand prepare(const ms_rows_t& m, bool planes, Space& space, int& rc, hipStream_t s, bool run) {
  operand o;
  o.rows = static_cast<int32_t>(m.n);
  if (!planes && lies_well(m)) {
    o.data = m.data;
    o.ld = m.n == 1 ? m.width : m.inner_stride;
    o.plane = 0;
    return o;
  }
  o.ld = round_up(m.width, 8);
  o.plane = round_up(m.n * o.ld, 128);
  const int64_t bytes = o.plane * (planes ? 6 : dtype_bytes(m.dtype));
  char* to = space.take<char>(bytes);
  o.data = to;
  if (!run || rc) return o;
  if (planes) {
    const int64_t blocks = ceil_div(m.n * (o.ld / 8), 256);
    rc = fits(blocks, 256) ? launch(k_planes, blocks, 256, s, m, o.ld, o.plane,
                                    reinterpret_cast<uint16_t*>(to))
                           : MS_OPS_EINVAL;
  } else if (m.dtype == MS_OPS_F32) {
    rc = lay_out<float>(m, o.ld, to, s);
  } else if (m.dtype == MS_OPS_F16) {
    rc = lay_out<f16>(m, o.ld, to, s);
  } else {
    rc = lay_out<bf16>(m, o.ld, to, s);
  }
  return o;
}

// Of k in one tile: 64 values, or 32 of 4 bytes.
int64_t steps_of(int64_t k, bool wide) { return ceil_div(k, wide ? 32 : 64); }

// The forward pass, or with run = false what workspace it takes.
int forward(const ms_rows_t& hidden, const ms_rows_t& weight, const ms_tokens_t* targets, float scale,
            int64_t ignore_index, float* logprob, float* lse, Space& space, hipStream_t s, bool run) {
  int rc = 0;
  const int64_t n = hidden.n, vocab = weight.n;
  product_args p{};
  const bool planes = !as_it_is(hidden, weight), wide = hidden.dtype == MS_OPS_F32 && !planes;
  p.b = prepare(hidden, planes, space, rc, s, run);
  p.a = prepare(weight, planes, space, rc, s, run);
  p.k = static_cast<int32_t>(hidden.width);
  p.pairs = planes ? 6 : 1;
  p.splits = 1;
  const Cut c = cut_of(vocab, n, steps_of(hidden.width, wide) * p.pairs, wide);
  const int64_t count = ceil_div(vocab, kShapes[c].m) * kShapes[c].wm;
  sum_epilogue e{};
  e.parts = space.take<float2>(count * n);
  e.picked = space.take<float>(n);
  if (!run || rc) return rc;
  e.targets = *targets;
  e.scale = scale;
  rc = wide                        ? run_product<float, kAlong, kAlong>(c, p, e, s)
       : hidden.dtype == MS_OPS_F16 ? run_product<f16, kAlong, kAlong>(c, p, e, s)
                                    : run_product<bf16, kAlong, kAlong>(c, p, e, s);
  if (rc) return rc;
  // few tokens: more threads to each, as one after the other they would wait for memory
  int lanes = 8;
  while (lanes < 256 && n * lanes < 262144 && lanes * 2 <= count) lanes *= 2;
  return launch(k_join, ceil_div(n, 256 / lanes), 256, s, e.parts, e.picked, count, n, lanes, *targets,
                vocab, ignore_index, logprob, lse);
}

template <typename T>
int fold(const float* parts, int count, int64_t n, int64_t width, const row_t* rows,
         const float* factor, float scale, void* out, hipStream_t s) {
  const int64_t blocks = ceil_div(ceil_div(n * width, 4), 256);
  if (!fits(blocks, 256)) return MS_OPS_EINVAL;
  return launch(k_fold<T>, blocks, 256, s, parts, count, n, width, rows, factor, scale,
                static_cast<T*>(out));
}

// T: the products' type; Out: the results'; Planes: 3 for 32 bits.
template <typename T, typename Out, int Planes>
int backward(const ms_rows_t& hidden, const ms_rows_t& weight, const ms_tokens_t* targets,
             float scale, int64_t ignore_index, const float* lse, const float* grad_logprob,
             const float* grad_lse, void* dhidden, void* dweight, Space& space, hipStream_t s,
             bool run) {
  int rc = 0;
  const int64_t n = hidden.n, vocab = weight.n, width = hidden.width;
  constexpr bool planes = Planes > 1, wide = sizeof(T) == 4;
  constexpr int pairs = planes ? 6 : 1;
  const bool lifted = hidden.dtype == MS_OPS_F16;
  const bool scaled_weight = lifted && dweight;
  row_t* rows = space.take<row_t>(n);
  float* factor = space.take<float>(1);
  int* least = scaled_weight ? space.take<int>(kScaleBlocks) : nullptr;
  const int64_t scale_blocks = std::min<int64_t>(ceil_div(n, kScaleRows), kScaleBlocks);
  if (run) {
    const rows_args a{lse, grad_logprob, grad_lse, *targets, vocab, ignore_index, lifted ? 1 : 0};
    rc = scaled_weight ? launch(k_scaled_rows, scale_blocks, kScaleThreads, s, a, hidden, rows, least)
                       : launch(k_rows, ceil_div(n, 256), 256, s, a, rows);
  }
  const operand h = prepare(hidden, planes, space, rc, s, run);
  const operand w = prepare(weight, planes, space, rc, s, run);
  operand scaled = h;
  if (scaled_weight) {
    scaled.ld = round_up(width, 8);
    f16* to = space.take<f16>(n * scaled.ld);
    scaled.data = to;
    const int64_t blocks = ceil_div(n * (scaled.ld / 8), 256);
    if (run && !rc)
      rc = fits(blocks, 256) ? launch(k_scaled_layout, blocks, 256, s, hidden, scaled.ld, rows, least,
                                      scale_blocks, to, factor)
                             : MS_OPS_EINVAL;
  }
  // Pieces of the vocabulary, all of one size: whole large tiles, and no more of them than
  // kPiece holds
  const int64_t most = std::min(std::max<int64_t>(kPiece / (n * static_cast<int64_t>(sizeof(T)) * Planes) / 256 * 256, 256), kMaxWidth);
  const int64_t pieces = ceil_div(vocab, most);
  const int64_t piece = round_up(ceil_div(vocab, pieces), 256);
  const int64_t plane = round_up(n * piece, 128);
  T* d = space.take<T>(plane * Planes);
  const int64_t columns = std::min(piece, vocab);
  const Cut cut_d = cut_of(columns, n, steps_of(width, wide) * pairs, wide);
  // dhidden sums over the pieces in fp32
  const Job job_h{width, n, steps_of(columns, wide) * pairs, pieces > 1};
  const Job job_w{width, columns, steps_of(n, wide) * pairs, false}, none{};
  // The two products in one launch, if one cut is best for both, the one of more k first
  Plan plan_h = plan_of(job_h, none, wide), plan_w = plan_of(job_w, none, wide);
  const bool both = dhidden && dweight && plan_h.cut != kFew && plan_w.cut != kFew;
  const bool w_first = job_w.steps >= job_h.steps;
  if (both) {
    const Plan plan = w_first ? plan_of(job_w, job_h) : plan_of(job_h, job_w);
    plan_h = {plan.cut, {plan.splits[w_first], 1}};
    plan_w = {plan.cut, {plan.splits[!w_first], 1}};
  }
  const int splits_h = plan_h.splits[0], splits_w = plan_w.splits[0];
  float* parts_h = dhidden && (splits_h > 1 || pieces > 1) ? space.take<float>(splits_h * n * width)
                                                           : nullptr;
  float* parts_w = dweight && splits_w > 1 ? space.take<float>(splits_w * columns * width) : nullptr;
  if (!run || rc) return rc;

  for (int64_t first = 0; first < vocab; first += piece) {
    const int64_t here = std::min(piece, vocab - first);
    operand w_here = w;
    w_here.data = static_cast<const char*>(w.data) + first * w.ld * static_cast<int64_t>(sizeof(T));
    w_here.rows = static_cast<int32_t>(here);

    product_args p{w_here, h, static_cast<int32_t>(width), pairs, 0, 0, 1};
    soft_epilogue<T, Planes> soft{d, piece, plane, rows, *targets, scale, static_cast<int32_t>(first)};
    rc = run_product<T, kAlong, kAlong>(cut_d, p, soft, s);
    if (rc) return rc;

    // dhidden: d, its tokens' rows along k, the vocabulary
    product_args ph{w_here, {d, piece, plane, static_cast<int32_t>(n)}, static_cast<int32_t>(here),
                    pairs, 0, 0, splits_h};
    ph.a.rows = static_cast<int32_t>(width);
    const out_epilogue<Out> out_h{static_cast<Out*>(dhidden), parts_h, rows, nullptr, scale, first > 0};
    // dweight: d, its tokens' rows across k, the tokens
    product_args pw{scaled, {d, piece, plane, static_cast<int32_t>(here)}, static_cast<int32_t>(n),
                    pairs, 0, 0, splits_w};
    pw.a.rows = static_cast<int32_t>(width);
    Out* to = static_cast<Out*>(dweight) + first * width;
    const float* by = lifted ? factor : nullptr;
    const out_epilogue<Out> out_w{to, parts_w, nullptr, by, scale, 0};
    if constexpr (wide) {
      if (dhidden) rc = run_product<T, kAcross, kAlong>(plan_h.cut, ph, out_h, s);
      if (!rc && dweight) rc = run_product<T, kAcross, kAcross>(plan_w.cut, pw, out_w, s);
    } else if (both) {
      rc = w_first ? run_products<T, kAcross, kAlong>(plan_h.cut, pw, out_w, ph, out_h, s)
                   : run_products<T, kAlong, kAcross>(plan_h.cut, ph, out_h, pw, out_w, s);
    } else {
      if (dhidden) rc = run_product<T, kAcross, kAlong>(plan_h.cut, ph, out_h, s);
      if (!rc && dweight) rc = run_product<T, kAcross, kAcross>(plan_w.cut, pw, out_w, s);
    }
    if (rc) return rc;
    if (parts_w) {
      rc = fold<Out>(parts_w, splits_w, here, width, nullptr, by, scale, to, s);
      if (rc) return rc;
    }
  }
  if (parts_h) return fold<Out>(parts_h, splits_h, n, width, rows, nullptr, scale, dhidden, s);
  return 0;
}

int backward_of(const ms_rows_t& hidden, const ms_rows_t& weight, const ms_tokens_t* targets,
                float scale, int64_t ignore_index, const float* lse, const float* grad_logprob,
                const float* grad_lse, void* dhidden, void* dweight, Space& space, hipStream_t s,
                bool run) {
  switch (hidden.dtype) {
    case MS_OPS_F16:
      return backward<f16, f16, 1>(hidden, weight, targets, scale, ignore_index, lse, grad_logprob,
                                   grad_lse, dhidden, dweight, space, s, run);
    case MS_OPS_BF16:
      return backward<bf16, bf16, 1>(hidden, weight, targets, scale, ignore_index, lse, grad_logprob,
                                     grad_lse, dhidden, dweight, space, s, run);
    default:
      if (as_it_is(hidden, weight))
        return backward<float, float, 1>(hidden, weight, targets, scale, ignore_index, lse,
                                         grad_logprob, grad_lse, dhidden, dweight, space, s, run);
      return backward<bf16, float, 3>(hidden, weight, targets, scale, ignore_index, lse, grad_logprob,
                                      grad_lse, dhidden, dweight, space, s, run);
  }
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace ops

extern "C" {

int64_t ms_linear_logprobs_workspace(const ms_rows_t* hidden, const ms_rows_t* weight) {
  using namespace ops;
  if (!good_sizes(hidden, weight)) return MS_OPS_EINVAL;
  if (hidden->n == 0) return 0;
  Space space{nullptr};
  forward(*hidden, *weight, nullptr, 1.0f, 0, nullptr, nullptr, space, nullptr, false);
  return space.used;
}

int ms_linear_logprobs(const ms_rows_t* hidden, const ms_rows_t* weight, const ms_tokens_t* targets,
                       float scale, int64_t ignore_index, float* logprob, float* lse, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  using namespace ops;
  if (!good_sizes(hidden, weight) || !good_tokens(targets) || targets->n != hidden->n)
    return MS_OPS_EINVAL;
  if (hidden->n == 0) return MS_OPS_OK;
  if (!logprob || !lse) return MS_OPS_EINVAL;
  if (workspace_bytes < ms_linear_logprobs_workspace(hidden, weight) || !workspace ||
      !aligned(workspace))
    return MS_OPS_EWORKSPACE;
  Space space{static_cast<char*>(workspace)};
  return forward(*hidden, *weight, targets, scale, ignore_index, logprob, lse, space,
                 static_cast<hipStream_t>(stream), true);
}

int64_t ms_linear_logprobs_grad_workspace_for(const ms_rows_t* hidden, const ms_rows_t* weight,
                                              int32_t want_hidden, int32_t want_weight) {
  using namespace ops;
  if (!good_sizes(hidden, weight)) return MS_OPS_EINVAL;
  if (hidden->n == 0 || (!want_hidden && !want_weight)) return 0;
  Space space{nullptr};
  // (any address: a gradient that is wanted)
  char some;
  backward_of(*hidden, *weight, nullptr, 1.0f, 0, nullptr, nullptr, nullptr,
              want_hidden ? &some : nullptr, want_weight ? &some : nullptr, space, nullptr, false);
  return space.used;
}

// One gradient alone has a plan of its own, which may cut k into more parts than that of both in
// one launch and then takes more (4096 x 5120 x 32000 bf16: 430 MB for dhidden, 262 for both).
int64_t ms_linear_logprobs_grad_workspace(const ms_rows_t* hidden, const ms_rows_t* weight) {
  const auto of = [&](int32_t h, int32_t w) {
    return ms_linear_logprobs_grad_workspace_for(hidden, weight, h, w);
  };
  const int64_t both = of(1, 1);
  return both < 0 ? both : std::max(both, std::max(of(1, 0), of(0, 1)));
}

int ms_linear_logprobs_grad(const ms_rows_t* hidden, const ms_rows_t* weight,
                            const ms_tokens_t* targets, float scale, int64_t ignore_index,
                            const float* lse, const float* grad_logprob, const float* grad_lse,
                            void* dhidden, void* dweight, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  using namespace ops;
  if (!good_sizes(hidden, weight) || !good_tokens(targets) || targets->n != hidden->n)
    return MS_OPS_EINVAL;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (hidden->n == 0) {
    if (!dweight) return MS_OPS_OK;
    const int64_t words = ceil_div(weight->n * weight->width * dtype_bytes(weight->dtype), 2);
    const int64_t blocks = ceil_div(words, 1024);
    if (!fits(blocks, 256)) return MS_OPS_EINVAL;
    return launch(k_zero, blocks, 256, s, static_cast<uint16_t*>(dweight), words);
  }
  if (!lse) return MS_OPS_EINVAL;
  if (!dhidden && !dweight) return MS_OPS_OK;
  // what these gradients take, by the same steps as the run itself
  const int64_t need =
      ms_linear_logprobs_grad_workspace_for(hidden, weight, dhidden != nullptr, dweight != nullptr);
  if (workspace_bytes < need || !workspace || !aligned(workspace))
    return MS_OPS_EWORKSPACE;
  Space space{static_cast<char*>(workspace)};
  return backward_of(*hidden, *weight, targets, scale, ignore_index, lse, grad_logprob, grad_lse,
                     dhidden, dweight, space, s, true);
}

}  // extern "C"
