// logprobs.hip — log probabilities of given tokens, entropy, the most likely
// alternatives, and the gradient of the logits (gfx950).
//
//   lse = log sum exp x,  logprob = x_target - lse,  entropy = lse - sum p x
//   dx  = g (1[j = target] - p) - h p (log p + entropy)
//
// One read of the logits forward, one read and one write backward: both are
// bound by memory, the forward with 4 to 6 instructions and one exponential per
// value not far from its arithmetic.

#include <algorithm>

#include "ops_common.h"

namespace {

using namespace ops;

// exp x = 2^(x L), with the same rounded L everywhere: what it is off by only
// rescales the logits by 1 + 1.3e-8.
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.69314718f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Over the wave, the result in every lane; a fixed order.  DPP moves instead of
// shuffles, which go through the LDS.
template <typename Op>
__device__ __forceinline__ float wave_reduce(float x, float none, Op op) {
#define STEP(ctrl, rows)                                                               \
  x = op(x, __uint_as_float(__builtin_amdgcn_update_dpp(                               \
                __float_as_uint(none), __float_as_uint(x), ctrl, rows, 0xf, false)))
  STEP(0x111, 0xf);      // row_shr 1, 2, 4, 8: lane 15 of each 16 has them all
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);      // row_bcast 15, 31: lane 63 has all
  STEP(0x143, 0xc);
#undef STEP
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_max(float x) {
  return wave_reduce(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
  return wave_reduce(x, 0.f, [](float a, float b) { return a + b; });
}

// Falling value, then rising index: a 64-bit key that is larger for what
// comes first, never 0.  NaN is above +inf; -0 equals +0.
typedef uint64_t Key;
constexpr uint32_t kNanKey = 0xFFFFFFF0u;
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? kNanKey : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ Key key_of(float x, int index) {
  return static_cast<Key>(order_of(x)) << 32 | ~static_cast<uint32_t>(index);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  if (k == kNanKey) return quiet_nan();
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float value_of(Key key) {
  return value_of(static_cast<uint32_t>(key >> 32));
}
__device__ __forceinline__ int index_of(Key key) {
  return static_cast<int>(~static_cast<uint32_t>(key));
}

// Over the values with y = x L - m2: s = sum 2^y, t = sum 2^y y.  m2 is a whole
// number near L max x (0 for no values or only -inf: then s is 0), so that
// lse = (m2 + log2 s) / L keeps what x L - m2 rounds.
struct Sums {
  float m2, s, t;
};

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m2 = a.s == 0.f ? b.m2 : b.s == 0.f ? a.m2 : fmaxf(a.m2, b.m2);
  const float da = a.m2 - m2, db = b.m2 - m2;
  const float ka = a.s == 0.f ? 0.f : exp2_fast(da), kb = b.s == 0.f ? 0.f : exp2_fast(db);
  Sums r;
  r.m2 = m2;
  r.s = a.s * ka + b.s * kb;
  r.t = (ka == 0.f ? 0.f : fmaf(da, a.s, a.t) * ka) + (kb == 0.f ? 0.f : fmaf(db, b.s, b.t) * kb);
  return r;
}

// What a row's sums say.
struct Row {
  float m2, ls, lse, entropy;

  __device__ __forceinline__ explicit Row(Sums a) {
    m2 = a.m2;
    ls = log2_fast(a.s);
    lse = (m2 + ls) * kLn2;
    entropy = (ls - a.t / a.s) * kLn2;
    if (a.s == 0.f) lse = -INFINITY, entropy = 0.f;      // nothing left by a mask
  }
  __device__ __forceinline__ float logprob(float x) const {
    if (lse == -INFINITY) return -INFINITY;
    if (fabsf(x) > 1e30f) return x - lse;                // x L may overflow
    return (fmaf(x, kLog2e, -m2) - ls) * kLn2;
  }
};

struct Outputs {
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_id;
  int top;
};

__device__ __forceinline__ void write_row(const Outputs& out, int64_t r, const Row& row,
                                          int64_t target, int64_t ignore, int64_t vocab,
                                          float given) {
  out.lse[r] = row.lse;
  if (out.entropy) out.entropy[r] = row.entropy;
  const bool good = target >= 0 && target < vocab;
  out.logprob[r] = target == ignore ? 0.f : good ? row.logprob(given) : quiet_nan();
}

constexpr float kMostSum = 0x1p100f;
constexpr int kMost = MS_OPS_MAX_TOP;
static_assert(kMost <= kWave, "");

// For blocks of NT threads; `list` takes C keys.
template <int NT, int C>
struct Lists {
  static constexpr int kCandidates = C;
  alignas(16) Key list[kCandidates];
  Key few[256];
  alignas(16) uint32_t high[NT];
  int at[NT];
  int looks[4 * NT];        // thread + NT * group
  int look_count, count;
};

// The largest word (its last kSkip bits 0) that at least k of the wave's 128 are
// as large as; 0 if there are fewer, none of them 0.
template <int kSkip>
__device__ __forceinline__ uint32_t kth_largest(uint32_t a, uint32_t b, int k) {
  uint32_t least = 0;
#pragma unroll
  for (int bit = 31; bit >= kSkip; --bit) {
    const uint32_t more = least | 1u << bit;
    if (__popcll(__ballot(a >= more)) + __popcll(__ballot(b >= more)) >= k) least = more;
  }
  return least;
}
__device__ __forceinline__ int count_above(uint32_t a, uint32_t b, uint32_t than) {
  return __popcll(__ballot(a > than)) + __popcll(__ballot(b > than));
}

// The k largest of the n keys in `list`, in order: put(rank, key).  Of more than
// a wave's, those that 128 sets' maxima leave are counted against each other.
template <int NT, int C, typename Put>
__device__ __forceinline__ void select_top(Lists<NT, C>& sh, int n, int k, Put put) {
  const Key* keys = sh.list;
  if (n > kWave) {
    uint32_t high[2] = {0, 0};              // the same in every wave
    for (int i = threadIdx.x & 63; i < n; i += 2 * kWave)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = i + u * kWave;
        const uint32_t h = j < n ? static_cast<uint32_t>(sh.list[j] >> 32) : 0;
        high[u] = h > high[u] ? h : high[u];
      }
    const uint32_t least = kth_largest<0>(high[0], high[1], k);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
      const Key key = sh.list[i];
      if (key && key >> 32 >= least) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < 256) sh.few[at] = key;
      }
    }
    __syncthreads();
    if (sh.count <= 256) {
      keys = sh.few;
      n = sh.count;
    }
  }
  for (int i = threadIdx.x; i < n; i += NT) {
    const Key key = keys[i];
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) above += keys[j] > key;
    if (key && above < k) put(above, key);
  }
}

// A row by itself whatever it holds: the maximum first, then the sums, then one
// pass for each alternative.  (Inlined: a call's stack alone took the whole
// kernel from 126 to 190 us for 8192 x 50257.)  For rows that the fast way gives up: NaN, +inf,
// logits beyond 2^19, or 69 above all that the first look saw.
template <int NT, typename T>
__device__ __forceinline__ void slow_row(float* value, Key* keys, const T* x, int64_t vocab,
                                         int64_t r, const Outputs& out, int64_t target,
                                         int64_t ignore) {
  constexpr int kThreads = NT, kWaves = NT / kWave;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto block = [&](float v, auto op) {
    __syncthreads();
    if (lane == 0) value[wave] = v;
    __syncthreads();
    float y = value[0];
    for (int w = 1; w < kWaves; ++w) y = op(y, value[w]);
    return y;
  };
  float most = -INFINITY;
  for (int64_t j = threadIdx.x; j < vocab; j += kThreads) most = fmaxf(most, widen(x[j]));
  most = block(wave_max(most), [](float a, float b) { return fmaxf(a, b); });
  const float base = most == -INFINITY ? 0.f : most;
  float s = 0.f, t = 0.f;
  for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
    const float y = (widen(x[j]) - base) * kLog2e, e = exp2_fast(y);
    s += e;
    t = fmaf(e, fmaxf(y, -1e30f), t);
  }
  auto add = [](float a, float b) { return a + b; };
  s = block(wave_sum(s), add);
  t = block(wave_sum(t), add);
  const bool empty = s == 0.f;
  const float ls = log2_fast(s);
  auto logprob = [&](float v) { return empty ? -INFINITY : (v - base) - ls * kLn2; };
  if (threadIdx.x == 0) {
    out.lse[r] = empty ? -INFINITY : base + ls * kLn2;
    if (out.entropy) out.entropy[r] = empty ? 0.f : (ls - t / s) * kLn2;
    const bool good = target >= 0 && target < vocab;
    out.logprob[r] = target == ignore ? 0.f : good ? logprob(widen(x[target])) : quiet_nan();
  }
  Key last = ~0ull;
  for (int k = 0; k < out.top; ++k) {
    Key mine = 0;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
      const Key key = key_of(widen(x[j]), static_cast<int>(j));
      if (key > mine && key < last) mine = key;
    }
    for (int b = 32; b; b >>= 1) {
      const Key other = __shfl_xor(static_cast<unsigned long long>(mine), b);
      if (other > mine) mine = other;
    }
    __syncthreads();
    if (lane == 0) keys[wave] = mine;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) mine = keys[w] > mine ? keys[w] : mine;
    last = mine;
    if (threadIdx.x == 0) {
      out.top_id[r * out.top + k] = index_of(mine);
      out.top_logprob[r * out.top + k] = logprob(value_of(mine));
    }
  }
}

// A wave's whole m2 for the largest logit it has seen.  A mask's lowest values, for
// which seen * L may overflow, get 0: they add nothing, which is right beside
// logits above kFarBelow / 2 and nowhere else.
constexpr float kFarBelow = -524288.f;        // -2^19
// Below this the first look may have met only masked values, -1e4 for one.
constexpr float kLow = -64.f;
__device__ __forceinline__ float reference(float seen) {
  return seen < kFarBelow ? 0.f : rintf(seen * kLog2e);
}
// ... whether leaving them out was wrong
__device__ __forceinline__ bool needed(Sums all) { return all.s == 0.f || all.m2 < kFarBelow / 2; }

// What a part of a split row leaves for k_join_parts, its keys behind it.
struct Part {
  Sums sums;
  int given_up;         // 2: values were left out
};

struct Split {
  int parts;            // of a row
  int64_t length;       // of a part
  char* work;           // [n, parts] of `stride` bytes: a Part and `top` keys
  int64_t stride;
};

// 16 bytes of logits, as words until they are used: taken apart into values
// beside a conditional load, every load is waited for before the next.
typedef uint32_t Words __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> values_of(Words w) {
  Pack<T, 16 / sizeof(T)> x;
  __builtin_memcpy(&x, &w, 16);
  return x;
}
template <typename T>
__device__ __forceinline__ Words no_values() {         // all -inf
  Pack<T, 16 / sizeof(T)> x;
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) x.v[i] = static_cast<T>(-INFINITY);
  Words w;
  __builtin_memcpy(&w, &x, 16);
  return w;
}

// The largest of the values seen, in as few instructions as the type has.
template <typename T>
struct Largest {
  float value = -INFINITY;
  template <int N>
  __device__ __forceinline__ void see(const Pack<T, N>& p) {
#pragma unroll
    for (int i = 0; i < N; ++i) value = fmaxf(value, widen(p.v[i]));
  }
  __device__ __forceinline__ float get() const { return value; }
};
template <>
struct Largest<f16> {
  typedef f16 two __attribute__((ext_vector_type(2)));
  two value = {static_cast<f16>(-INFINITY), static_cast<f16>(-INFINITY)};
  template <int N>
  __device__ __forceinline__ void see(const Pack<f16, N>& p) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      value = __builtin_elementwise_max(value, two{p.v[i], p.v[i + 1]});
  }
  __device__ __forceinline__ float get() const { return fmaxf(widen(value.x), widen(value.y)); }
};

// A block takes a row, or a part of one where there are few rows, in groups of
// kGroup rounds of an aligned 16-byte unit to every thread; the next group is
// loaded while one is worked on.  (At the rows' own alignment, 50257 values of 2
// bytes, units of which 7 of 8 lie across 16 bytes, the loads alone ran at 4.5
// TB/s instead of 6.8.)
//
// The first group gives a reference, one per wave, so that no running maximum
// is kept but for waves that may have seen only masked values.  Where later logits
// are 69 above all that the wave saw the row is done again by slow_row: s < 2^100
// keeps t, up to 100 s, in range too.
//
// For the alternatives each thread keeps the largest value of its best group and
// that of its others.  The k-th largest of the threads' values bounds the k-th
// largest of all from below; the few groups that may reach it are read again,
// their values that do listed in LDS and counted against each other.
//
// Measured, 8192 x 50257 fp16: 123 us, 6.7 TB/s read, of 7.3 that a
// kernel which only reads gets; 2048 x 128256 bf16, entropy, 8 alternatives: 95 us, 5.5.
template <typename T, int NT, bool kTop, bool kEntropy>
__global__ void __launch_bounds__(NT, kTop && NT < 256 ? 6 : 8)      // 6 fit beside their LDS
    k_logprobs(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, Outputs out, Split split) {
  constexpr int kVec = 16 / sizeof(T), kWaves = NT / kWave, kGroup = kTop ? 3 : 4;
  typedef Pack<T, kVec> Unit;
  __shared__ Sums sums[kWaves];
  __shared__ float value[kWaves];
  __shared__ int out_of[kWaves];
  __shared__ Lists<(kTop ? NT : 1), (kTop ? 1024 : kMost)> sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = blockIdx.x / split.parts, vocab = logits.width;
  const int64_t begin = (blockIdx.x - r * split.parts) * split.length;
  const int64_t target = token(targets, r);
  const T* row = static_cast<const T*>(logits.data) + row_start(logits, r);
  const T* x = row + begin;
  const int n = static_cast<int>(vocab - begin < split.length ? vocab - begin : split.length);
  const int off = static_cast<int>(-(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (kVec - 1));
  const int head = off < n ? off : n;               // values before the first whole unit
  const int units = (n - head) / kVec, rest = n - head - units * kVec;
  const int rounds = (units + NT - 1) / NT;
  const T* first = x + head;

  // the last round's threads without a unit load the last one
  auto load_group = [&](int k0, Words (&p)[kGroup]) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k)
      if (k0 + k < rounds) {
        const int u = (k0 + k) * NT + threadIdx.x;
        p[k] = __builtin_nontemporal_load(reinterpret_cast<const Words*>(
            first + static_cast<int64_t>(u < units ? u : units - 1) * kVec));
      }
  };
  // ... and drop it
  auto mask_group = [&](int k0, Words (&p)[kGroup]) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k)
      if (k0 + k >= rounds - 1 && (k0 + k) * NT + static_cast<int>(threadIdx.x) >= units)
        p[k] = no_values<T>();
  };
  Words now[kGroup], next[kGroup];
  load_group(0, now);
  // the values before and behind the units, one to a thread
  const int tid = threadIdx.x;
  const int alone = tid < head                          ? tid
                    : tid >= kVec && tid - kVec < rest ? head + units * kVec + tid - kVec
                                                       : -1;
  // loads come back in order: what waits for one waits for those before it
  const T single_raw = x[alone >= 0 ? alone : 0];
  load_group(kGroup, next);
  const bool good = target >= 0 && target < vocab;
  const T given_raw = row[good ? target : 0];
  mask_group(0, now);
  const float single = alone >= 0 ? widen(single_raw) : -INFINITY;

  Largest<T> largest;
#pragma unroll
  for (int k = 0; k < kGroup; ++k) largest.see(values_of<T>(now[k]));
  float seen = wave_max(fmaxf(single, largest.get())), s = 0.f, t = 0.f;
  float m2 = reference(seen);
  bool left_out = seen < kFarBelow && seen != -INFINITY;
  auto add = [&](float v) {
    const float y = fmaf(v, kLog2e, -m2), e = exp2_fast(y);
    s += e;
    if (kEntropy) t = fmaf(e, fmaxf(y, -1e30f), t);
  };
  add(single);
  float best = largest.get(), others = -INFINITY;
  int best_group = 0;
  for (int k0 = 0;;) {
    if (k0 && seen < kLow) {
      // a wave that may have seen nothing but what is masked looks again
      Largest<T> here;
#pragma unroll
      for (int k = 0; k < kGroup; ++k)
        if (k0 + k < rounds) here.see(values_of<T>(now[k]));
      const float high = wave_max(here.get());
      left_out |= high < kFarBelow && high != -INFINITY;
      if (high > seen) {
        const float to = reference(high);
        if (seen >= kFarBelow) {
          const float d = m2 - to, k = exp2_fast(d);
          if (kEntropy) t = fmaf(d, s, t) * k;
          s *= k;
        }
        seen = high;
        m2 = to;
      }
    }
    Largest<T> here;
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      if (k0 + k >= rounds) break;
#pragma unroll
      for (int i = 0; i < kVec; ++i) add(widen(values_of<T>(now[k]).v[i]));
      if (kTop) here.see(values_of<T>(now[k]));
    }
    if (kTop && k0) {
      const float high = here.get();
      const bool better = high > best;
      others = fmaxf(others, better ? best : high);
      best_group = better ? k0 / kGroup : best_group;
      best = better ? high : best;
    }
    k0 += kGroup;
    if (k0 >= rounds) break;
#pragma unroll
    for (int k = 0; k < kGroup; ++k) now[k] = next[k];
    load_group(k0 + kGroup, next);
    if (k0 + kGroup >= rounds) mask_group(k0, now);
  }

  s = wave_sum(s);
  if (kEntropy) t = wave_sum(t);
  if (lane == 0) sums[wave] = Sums{m2, s, t}, out_of[wave] = left_out;
  const float most = fmaxf(single, best);
  if constexpr (kTop) {
    sh.high[tid] = tid < units || alone >= 0 ? order_of(most) : 0;
    if (tid == 0) sh.count = sh.look_count = 0;
  }
  __syncthreads();
  bool give_up = false, some_out = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    give_up |= !(sums[w].s < kMostSum) || !(sums[w].m2 <= 1 << 20);
    some_out |= out_of[w];
  }
  if (!kTop && !give_up && !some_out && wave) return;
  Sums all = sums[0];
  for (int w = 1; w < kWaves; ++w) all = join(all, sums[w]);
  if (split.parts == 1) give_up |= some_out && needed(all);
  const float given = widen(given_raw);

  if constexpr (kTop) {
    if (!give_up) {
      // 128 sets of neighbouring threads, two to a lane, the same in every wave
      constexpr int kSet = NT / (2 * kWave);
      uint32_t high[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2 * kSet; ++i) {
        const uint32_t h = sh.high[lane * 2 * kSet + i];
        high[i / kSet] = h > high[i / kSet] ? h : high[i / kSet];
      }
      // (2-byte types widen to words whose last bits are all the same)
      constexpr int kSkip = sizeof(T) == 2 ? 13 : 0;
      constexpr uint32_t kRest = (1u << kSkip) - 1;
      uint32_t least = kth_largest<kSkip>(high[0], high[1], out.top);
      int last = INT32_MAX;              // of those equal to `least`, indices up to here
      constexpr int kAgain = 2;
      auto unit_of = [&](int k, int thread) {
        return load<kVec>(first + static_cast<int64_t>(k * NT + thread) * kVec);
      };
      if (least && count_above(high[0], high[1], least - 1) > out.top + 16) {
        // many equal ones: tell them by their indices
        uint32_t mine = 0;                              // the whole of that word
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if ((high[u] & ~kRest) == least) mine = high[u];
        least = read_lane(static_cast<int>(mine),
                          __ffsll(static_cast<unsigned long long>(__ballot(mine != 0))) - 1);
        int at = INT32_MAX;                             // the thread's first that equals it
        if (alone >= 0 && order_of(single) == least) at = alone;
        if (order_of(most) >= least)
          for (int k = 0; k * NT + tid < units; ++k) {
            const Unit p = unit_of(k, tid);
#pragma unroll
            for (int i = kVec - 1; i >= 0; --i) {
              const int j = head + (k * NT + tid) * kVec + i;
              if (order_of(widen(p.v[i])) == least && j < at) at = j;
            }
            if (at != INT32_MAX && at != alone) break;
          }
        sh.at[tid] = at;
        __syncthreads();
        uint32_t early[2] = {0, 0};                     // ~index: larger for what comes first
#pragma unroll
        for (int i = 0; i < 2 * kSet; ++i) {
          const int j = sh.at[lane * 2 * kSet + i];
          const uint32_t e = j == INT32_MAX ? 0 : ~static_cast<uint32_t>(j);
          early[i / kSet] = e > early[i / kSet] ? e : early[i / kSet];
        }
        // a set with a larger one counts for that
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (high[u] > least) early[u] = 0;
        last = static_cast<int>(~kth_largest<0>(
            early[0], early[1], out.top - count_above(high[0], high[1], least)));
        if (last < 0) last = INT32_MAX;
      }
      auto offer = [&](float v, int j) {
        const uint32_t o = order_of(v);
        if (o < least || (o == least && j > last)) return;
        const int at = atomicAdd(&sh.count, 1);
        if (at < sh.kCandidates) sh.list[at] = key_of(v, static_cast<int>(begin) + j);
      };
      const float least_value = least > 0x007FFFFFu ? value_of(least) : -INFINITY;
      if (alone >= 0) offer(single, alone);
      if (tid < units && order_of(best) >= least)
        for (int g = 0; g * kGroup * NT + tid < units; ++g) {
          // (of a thread whose best only equals `least`, groups behind `last` are out)
          const bool out_of_reach =
              order_of(best) == least && (g * kGroup * NT + tid) * kVec + head > last;
          if ((g == best_group || order_of(others) >= least) && !out_of_reach) {
            const int at = atomicAdd(&sh.look_count, 1);
            if (at < 4 * NT) sh.looks[at] = tid + NT * g;
          }
        }
      __syncthreads();
      if (sh.look_count <= 4 * NT) {
        const int again = sh.look_count * kGroup;
        for (int i0 = tid; i0 < again; i0 += kAgain * NT) {
          Words p[kAgain];
          int u[kAgain];
#pragma unroll
          for (int j = 0; j < kAgain; ++j) {
            const int i = i0 + j * NT < again ? i0 + j * NT : i0;
            const int look = sh.looks[i / kGroup];
            u[j] = ((look / NT) * kGroup + i % kGroup) * NT + look % NT;
            p[j] = *reinterpret_cast<const Words*>(
                first + static_cast<int64_t>(u[j] < units ? u[j] : 0) * kVec);
            if (i0 + j * NT >= again) u[j] = units;
          }
#pragma unroll
          for (int j = 0; j < kAgain; ++j)
            if (u[j] < units)
#pragma unroll
              for (int i = 0; i < kVec; ++i)
                if (widen(values_of<T>(p[j]).v[i]) >= least_value)
                  offer(widen(values_of<T>(p[j]).v[i]), head + u[j] * kVec + i);
        }
      } else {
        // more groups than the list takes (a long row, many alternatives): all again
        // (1024 x 262144 bf16, 50 alternatives, with half the list: 180 us instead of 121)
        for (int u = tid; u < units; u += NT) {
          const Unit p = unit_of(0, u);
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (widen(p.v[i]) >= least_value) offer(widen(p.v[i]), head + u * kVec + i);
        }
      }
      __syncthreads();
      give_up = sh.count > sh.kCandidates;
    }
  }

  if (split.parts == 1) {
    if (give_up) {
      slow_row<NT>(value, sh.list, row, vocab, r, out, target, ignore);
      return;
    }
    const Row done(all);
    if (tid == 0) write_row(out, r, done, target, ignore, vocab, given);
    if constexpr (kTop)
      select_top(sh, sh.count, out.top, [&](int rank, Key key) {
        out.top_id[r * out.top + rank] = index_of(key);
        out.top_logprob[r * out.top + rank] = done.logprob(value_of(key));
      });
    return;
  }
  char* left = split.work + blockIdx.x * split.stride;
  if (tid == 0) *reinterpret_cast<Part*>(left) = Part{all, give_up ? 1 : some_out ? 2 : 0};
  if constexpr (kTop) {
    if (give_up) return;
    Key* keys = reinterpret_cast<Key*>(left + sizeof(Part));
    if (n < out.top) {                               // a last part of few values
      if (tid < out.top) keys[tid] = 0;
      __syncthreads();
    }
    select_top(sh, sh.count, out.top, [&](int rank, Key key) { keys[rank] = key; });
  }
}

// Threads to a block.  With alternatives 256, of which more fit a CU beside their
// LDS and end together: 8192 x 50257 bf16 with entropy, 8 and 50 alternatives
// 149 and 181 us, 198 and 226 with 512 (and 146 and 190 with groups of 4 rounds).
// Without, 512: 126 us, 130 with 256.  Rows of up to kMidUnits units (half of that with
// alternatives) are over soon, so 128, more rows beside each other: 32768 x 4097 and
// 8192, 16384 x 16384 bf16 61, 86 and 86 us, 156, 171 and 127 with 512; 8 alternatives
// 116, 145 and 121, 134, 172 and 121 with 256.
constexpr int kThreads = 512, kTopThreads = 256, kMidThreads = 128, kMidUnits = 2048;

// A row's parts.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join_parts(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, Outputs out,
                 Split split) {
  __shared__ Lists<kThreads, kMost * kWave> sh;
  __shared__ float value[kThreads / kWave];
  const int64_t r = blockIdx.x, vocab = logits.width;
  const T* row = static_cast<const T*>(logits.data) + row_start(logits, r);
  const int64_t target = token(targets, r);
  const float given = target >= 0 && target < vocab ? widen(row[target]) : 0.f;
  const char* work = split.work + r * split.parts * split.stride;
  const int keys = split.parts * out.top;          // no more than the list takes
  for (int i = threadIdx.x; i < keys; i += kThreads) {
    const int p = i / out.top;
    sh.list[i] =
        reinterpret_cast<const Key*>(work + p * split.stride + sizeof(Part))[i - p * out.top];
  }
  // as many parts as lanes, in every wave
  const int lane = threadIdx.x & 63;
  Part mine{{0.f, 0.f, 0.f}, 0};
  if (lane < split.parts) mine = *reinterpret_cast<const Part*>(work + lane * split.stride);
  bool give_up = __any(mine.given_up == 1);
  const bool some_out = __any(mine.given_up == 2);
  Sums all = mine.sums;
  for (int k = 1; k < kWave; k <<= 1) {
    Sums other;
    other.m2 = __shfl_xor(all.m2, k);
    other.s = __shfl_xor(all.s, k);
    other.t = __shfl_xor(all.t, k);
    all = lane & k ? join(other, all) : join(all, other);
  }
  __syncthreads();
  give_up |= some_out && needed(all);
  if (give_up) {
    slow_row<kThreads>(value, sh.list, row, vocab, r, out, target, ignore);
    return;
  }
  const Row done(all);
  if (threadIdx.x == 0) write_row(out, r, done, target, ignore, vocab, given);
  if (out.top)
    select_top(sh, keys, out.top, [&](int rank, Key key) {
      out.top_id[r * out.top + rank] = index_of(key);
      out.top_logprob[r * out.top + rank] = done.logprob(value_of(key));
    });
}

// -- short rows -----------------------------------------------------------------

// Rows of up to kShortUnits units: a wave to a row, which it holds in registers, R
// units to a lane; the blocks that fit beside each other go through all rows.
// With entropy, bf16: 65536 x 512 25 us, 65536 x 4096 86 us (6.2 TB/s), with 8 alternatives 57 and
// 149.  (A block of 128 threads to a row: 65536 x 512 56 and 140 us, which is what
// starting the blocks takes.)
constexpr int kShortThreads = 256, kShortWaves = kShortThreads / kWave;
constexpr int kShortUnits = 8 * kWave;
constexpr int kShortBlocks = 2048;               // 8 to a CU
constexpr int kShortList = 256;

// Where a row's units lie, and the value before or behind them that a lane takes.
template <typename T>
struct ShortRow {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  int head, units, alone;

  // aligned_to: the address whose 16-byte units are taken
  __device__ __forceinline__ ShortRow(const T* row, const T* aligned_to, int vocab, int lane) {
    x = row;
    const int off =
        static_cast<int>(-(reinterpret_cast<uintptr_t>(aligned_to) / sizeof(T)) & (kVec - 1));
    head = off < vocab ? off : vocab;
    units = (vocab - head) / kVec;
    const int rest = vocab - head - units * kVec;
    alone = lane < head                             ? lane
            : lane >= kVec && lane - kVec < rest ? head + units * kVec + lane - kVec
                                                    : -1;
  }
  // kAny: the units lie at any address.  Lanes without a unit load the last one.
  template <bool kAny, int R>
  __device__ __forceinline__ void load(Words (&w)[R], int lane) const {
    typedef typename raw_of<16>::type AnyWords;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int u = k * kWave + lane;
      const T* at = x + head + static_cast<int64_t>(u < units ? u : units - 1) * kVec;
      if (units > 0)
        w[k] = kAny ? __builtin_nontemporal_load(reinterpret_cast<const AnyWords*>(at))
                    : __builtin_nontemporal_load(reinterpret_cast<const Words*>(at));
    }
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (k * kWave + lane >= units) w[k] = no_values<T>();
  }
  __device__ __forceinline__ float load_alone() const {
    const T raw = x[alone >= 0 ? alone : 0];
    return alone >= 0 ? widen(raw) : -INFINITY;
  }
};

// A wave's values: f(value, index) for each that it has.
template <typename T, int R, typename F>
__device__ __forceinline__ void each_value(const ShortRow<T>& row, const Words (&w)[R],
                                           float single, int lane, F f) {
  constexpr int kVec = 16 / sizeof(T);
  if (row.alone >= 0) f(single, row.alone);
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (k * kWave + lane < row.units)
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        f(widen(values_of<T>(w[k]).v[i]), row.head + (k * kWave + lane) * kVec + i);
}

__device__ __forceinline__ int wave_count(int x) {
  for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k);
  return uniform(x);
}

// The `top` first of a row in key order, into `list`, whatever it holds, and perhaps
// others, kShortList at most; how many.  Of the values that equal the last one those with
// the lowest indices.  At least `top` values are as large as `least`.  (The row is read again
// for each step: its words taken apart in registers cost every row its place.)
template <typename T>
__device__ __forceinline__ int list_exactly(const T* x, int vocab, int lane, int top,
                                            uint32_t least, Key* list) {
  auto count = [&](auto test) {
    int n = 0;
    for (int j = lane; j < vocab; j += kWave) n += test(order_of(widen(x[j])));
    return wave_count(n);
  };
  int above = count([&](uint32_t o) { return o > least; });
  // (a mask that leaves little has that little in few lanes: `least` is what is masked, and
  // what is above fits the list.  With the search for it a row took 116 us.)
  if (above > kShortList) {
    uint32_t bound = 0;                       // the largest word that `top` are as large as
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t more = bound | 1u << bit;
      if (more <= least || count([&](uint32_t o) { return o >= more; }) >= top) bound = more;
    }
    least = bound;
    above = count([&](uint32_t o) { return o > least; });
  }
  const int missing = above < top ? top - above : 0;      // of those that equal `least`
  int to = 0, equal = 0;
  const uint64_t lower = (1ull << lane) - 1;
  for (int j0 = 0; j0 < vocab; j0 += kWave) {
    const int j = j0 + lane;
    const float v = j < vocab ? widen(x[j]) : 0.f;
    const uint32_t o = j < vocab ? order_of(v) : 0;
    const uint64_t same = __ballot(j < vocab && o == least);
    const int before = equal + static_cast<int>(__popcll(same & lower));
    const bool in = j < vocab && (o > least || (o == least && before < missing));
    const uint64_t all = __ballot(in);
    if (in) list[to + __popcll(all & lower)] = key_of(v, j);
    to += __popcll(all);
    equal += __popcll(same);
  }
  return to;
}

template <typename T, int R, bool kTop, bool kEntropy>
__global__ void __launch_bounds__(kShortThreads)
    k_logprobs_short(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, Outputs out) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ Key lists[kTop ? kShortWaves : 1][kTop ? kShortList : 1];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int vocab = static_cast<int>(logits.width);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kShortWaves + wave; r < logits.n;
       r += static_cast<int64_t>(gridDim.x) * kShortWaves) {
    const int64_t target = token(targets, r);
    const T* x = static_cast<const T*>(logits.data) + row_start(logits, r);
    const ShortRow<T> row(x, x, vocab, lane);
    Words w[R];
    row.template load<false>(w, lane);
    const float single = row.load_alone();
    const bool good = target >= 0 && target < vocab;
    const float given = widen(x[good ? target : 0]);
    Largest<T> largest[2];                             // of each half of the units
#pragma unroll
    for (int k = 0; k < R; ++k) {
      Pack<T, kVec / 2> half[2];
      __builtin_memcpy(half, &w[k], 16);
      largest[0].see(half[0]);
      largest[1].see(half[1]);
    }
    const float mine = fmaxf(single, largest[0].get()), other = largest[1].get();
    const float most = wave_max(fmaxf(mine, other)), base = most == -INFINITY ? 0.f : most;
    float s = 0.f, t = 0.f;
    auto add = [&](float v) {
      const float y = (v - base) * kLog2e, e = exp2_fast(y);
      s += e;
      if (kEntropy) t = fmaf(e, fmaxf(y, -1e30f), t);
    };
    add(single);
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < kVec; ++i) add(widen(values_of<T>(w[k]).v[i]));
    s = wave_sum(s);
    if (kEntropy) t = wave_sum(t);
    const bool empty = s == 0.f;
    const float ls = log2_fast(s) * kLn2;
    auto logprob = [&](float v) { return empty ? -INFINITY : (v - base) - ls; };
    if (lane == 0) {
      out.lse[r] = empty ? -INFINITY : base + ls;
      if (kEntropy) out.entropy[r] = empty ? 0.f : ls - t / s * kLn2;
      out.logprob[r] = target == ignore ? 0.f : good ? logprob(given) : quiet_nan();
    }
    if constexpr (kTop) {
      // the k-th largest of the 128 half lanes' largest bounds the k-th largest from
      // below; what reaches it is listed and counted against each other
      constexpr int kSkip = sizeof(T) == 2 ? 13 : 0;
      Key* list = lists[wave];
      const bool unit = lane < row.units;
      uint32_t least = kth_largest<kSkip>(unit || row.alone >= 0 ? order_of(mine) : 0,
                                          unit ? order_of(other) : 0, out.top);
      // the last bits of a 2-byte type's word, which are not searched, are 1 in a negative
      // value's: without them all of a masked row's values would lie above
      if (least && !(least >> 31)) least |= (1u << kSkip) - 1;
      int found = kShortList + 1;
      if (least == 0 && vocab <= kShortList) {           // fewer than that: all of them
        for (int j = lane; j < vocab; j += kWave) list[j] = key_of(widen(x[j]), j);
        found = vocab;
      } else if (s < INFINITY && least > 0x007FFFFFu) {
        const float least_value = value_of(least);
        int to = 0;
        auto offer = [&](float v, int j) {
          const uint64_t hits = __ballot(v >= least_value);
          if (!hits) return;
          const int at = to + __popcll(hits & ((1ull << lane) - 1));
          if (v >= least_value && at < kShortList) list[at] = key_of(v, j);
          to += __popcll(hits);
        };
        offer(single, row.alone);
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            offer(widen(values_of<T>(w[k]).v[i]), row.head + (k * kWave + lane) * kVec + i);
        found = to;
      }
      if (found > kShortList) {
        found = list_exactly(x, vocab, lane, out.top, least, list);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int i = lane; i < found; i += kWave) {
        const Key key = list[i];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < found; ++j) above += list[j] > key;
        if (above < out.top) {
          out.top_id[r * out.top + above] = index_of(key);
          out.top_logprob[r * out.top + above] = logprob(value_of(key));
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// -- gradient -----------------------------------------------------------------

// Beyond this an fp32 lse no longer tells logits from each other (a row masked
// with the type's lowest value: lse - max is lost), and the row's maximum and
// sum are found again.
constexpr float kFarLse = 256.f;

constexpr int kGradThreads = 256, kGradWaves = kGradThreads / kWave;
constexpr int kFarUnits = 4;              // units to a thread in flight, rows beyond kFarLse
constexpr int kGradGroup = 1;             // 16-byte units to a thread; 1, 2, 4: 263, 280, 290 us

// A block takes kGradGroup rounds of aligned 16-byte units of the gradient's row
// (the logits' row may lie otherwise).  With c a whole number near lse L and
// p' = 2^(x L - c): dx = p' (a + b x), where a and b hold what c rounded off; the
// target's g is added to the one value.  8192 x 50257 fp16: 263 us, 6.3 TB/s, what
// a copy of as many bytes gets.
// A value's gradient but for the target's g; lse within kFarLse.
template <bool kEntropy>
struct RowGrad {
  float c, a, b;

  __device__ __forceinline__ RowGrad(float lse, float entropy, float g, float h) {
    c = rintf(lse * kLog2e);
    const float k = exp2_fast(-fmaf(lse, kLog2e, -c));
    b = -h * k;
    a = -(g + h * (entropy - lse)) * k;
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float p = exp2_fast(fmaf(v, kLog2e, -c));
    if (!kEntropy) return p * a;
    return p * fmaf(b, fmaxf(v, -1e6f), a);        // -inf: p is 0, and 0 * inf must not be
  }
};

template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kGradThreads)
    k_logprobs_grad(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, const float* lse,
                    const float* entropy, const float* grad_logprob, const float* grad_entropy,
                    int blocks_per_row, T* __restrict__ out) {
  constexpr int kVec = 16 / sizeof(T), kEach = kGradGroup * kGradThreads;
  __shared__ float slot[kGradWaves];
  const int64_t r = blockIdx.x / static_cast<unsigned>(blocks_per_row);
  const int part = static_cast<int>(blockIdx.x - r * blocks_per_row);
  const int vocab = static_cast<int>(logits.width), tid = threadIdx.x;
  const T* x = static_cast<const T*>(logits.data) + row_start(logits, r);
  T* d = out + r * vocab;
  const int off = static_cast<int>(-(reinterpret_cast<uintptr_t>(d) / sizeof(T)) & (kVec - 1));
  const int head = off < vocab ? off : vocab;
  const int units = (vocab - head) / kVec, rest = vocab - head - units * kVec;

  typedef typename raw_of<16>::type AnyWords;          // the logits may lie otherwise
  Words in[kGradGroup];
  if (units > 0)
#pragma unroll
    for (int i = 0; i < kGradGroup; ++i) {
      const int u = part * kEach + i * kGradThreads + tid;
      in[i] = __builtin_nontemporal_load(reinterpret_cast<const AnyWords*>(
          x + head + static_cast<int64_t>(u < units ? u : units - 1) * kVec));
    }
  const int64_t target = token(targets, r);
  const bool counts = grad_logprob && target != ignore;
  float g = counts ? grad_logprob[r] : 0.f;
  if (counts && (target < 0 || target >= vocab)) g = quiet_nan();
  const int hit = target >= 0 && target < vocab ? static_cast<int>(target) : -1;
  const float h = kEntropy ? grad_entropy[r] : 0.f, big_h = kEntropy ? entropy[r] : 0.f;
  const float l = lse[r];

  if (l == -INFINITY) {
    // the first block takes the head too, the last one what is behind the units; with
    // the head before them the last block but one may already reach the row's end
    const int begin = part ? head + part * kEach * kVec : 0;
    const int behind = head + (part + 1) * kEach * kVec;
    const int end = part == blocks_per_row - 1 || behind > vocab ? vocab : behind;
    for (int j = begin + tid; j < end; j += kGradThreads) {
      const float v = widen(x[j]);
      d[j] = narrow<T>(v != v ? v : 0.f);              // a NaN says so whatever lse is
    }
    return;
  }
  // the value of this thread before or behind the units, if `head` and `rest` are the block's
  const int alone_head = tid < head ? tid : -1;
  const int alone_rest = tid >= kVec && tid - kVec < rest ? head + units * kVec + tid - kVec : -1;
  if (fabsf(l) > kFarLse) {
    // One block for the whole row: the maximum and the sum first, then the gradient.
    // 8192 x 50257 fp16, all rows so 496 us, one of them 317, none 266; where every block
    // of a row went through all of it 13250 us and 340.
    if (part) return;
    const int alone = alone_head >= 0 ? alone_head : alone_rest;
    const float single = alone >= 0 ? widen(x[alone]) : -INFINITY;
    auto load_far = [&](int u0, Words (&w)[kFarUnits]) {
#pragma unroll
      for (int i = 0; i < kFarUnits; ++i) {
        const int u = u0 + i * kGradThreads + tid;
        w[i] = *reinterpret_cast<const AnyWords*>(
            x + head + static_cast<int64_t>(u < units ? u : units - 1) * kVec);
      }
#pragma unroll
      for (int i = 0; i < kFarUnits; ++i)
        if (u0 + i * kGradThreads + tid >= units) w[i] = no_values<T>();
    };
    float most = single, s = single == -INFINITY ? 0.f : 1.f;
    if (single != single || single == INFINITY) s = quiet_nan();
    for (int u0 = 0; u0 < units; u0 += kFarUnits * kGradThreads) {
      Words w[kFarUnits];
      load_far(u0, w);
      Largest<T> largest;
#pragma unroll
      for (int i = 0; i < kFarUnits; ++i) largest.see(values_of<T>(w[i]));
      const float to = fmaxf(most, largest.get());
      if (to > most) s *= exp2_fast((most - to) * kLog2e);
      most = to;
      const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
      for (int i = 0; i < kFarUnits; ++i)
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          s += exp2_fast((widen(values_of<T>(w[i]).v[j]) - base) * kLog2e);
    }
    auto block = [&](float v, auto op) {
      __syncthreads();
      if ((tid & 63) == 0) slot[tid >> 6] = v;
      __syncthreads();
      float y = slot[0];
      for (int w = 1; w < kGradWaves; ++w) y = op(y, slot[w]);
      return y;
    };
    const float mine = most;
    most = block(wave_max(most), [](float a, float b) { return fmaxf(a, b); });
    s *= exp2_fast((mine - most) * kLog2e);
    const float ls =
        log2_fast(block(wave_sum(s), [](float a, float b) { return a + b; })) * kLn2;
    auto one = [&](float v, int j) {
      const float logp = (v - most) - ls, p = exp2_fast(logp * kLog2e);
      float dj = j == hit ? g - g * p : -g * p;
      if (kEntropy && p != 0.f) dj -= h * p * (logp + big_h);
      return narrow<T>(dj);
    };
    if (alone >= 0) d[alone] = one(single, alone);
    for (int u0 = 0; u0 < units; u0 += kFarUnits * kGradThreads) {
      Words w[kFarUnits];
      load_far(u0, w);
#pragma unroll
      for (int i = 0; i < kFarUnits; ++i) {
        const int u = u0 + i * kGradThreads + tid, j0 = head + u * kVec;
        if (u >= units) continue;
        Pack<T, kVec> z;
#pragma unroll
        for (int j = 0; j < kVec; ++j) z.v[j] = one(widen(values_of<T>(w[i]).v[j]), j0 + j);
        store_stream<kVec>(d + j0, z);
      }
    }
    return;
  }

  const RowGrad<kEntropy> one(l, big_h, g, h);
#pragma unroll
  for (int i = 0; i < kGradGroup; ++i) {
    const int u = part * kEach + i * kGradThreads + tid;
    if (u < units) {
      float y[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = one(widen(values_of<T>(in[i]).v[j]));
      const unsigned at = static_cast<unsigned>(hit - head - u * kVec);
      if (at < kVec && hit >= 0)
#pragma unroll
        for (int j = 0; j < kVec; ++j) y[j] += at == j ? g : 0.f;
      Pack<T, kVec> z;
#pragma unroll
      for (int j = 0; j < kVec; ++j) z.v[j] = narrow<T>(y[j]);
      store_stream<kVec>(d + head + static_cast<int64_t>(u) * kVec, z);
    }
  }
  const int alone = part == 0 && alone_head >= 0           ? alone_head
                    : part == blocks_per_row - 1 ? alone_rest
                                                 : -1;
  if (alone >= 0) d[alone] = narrow<T>(one(widen(x[alone])) + (alone == hit ? g : 0.f));
}

// Short rows: a wave to each, as forward, by the units of the gradient's row.  65536 x
// 512 and 4096 bf16 29 and 190 us (4.6 and 5.6 TB/s), 55 us for the first with a
// block to each.
template <typename T, int R, bool kEntropy>
__global__ void __launch_bounds__(kShortThreads)
    k_logprobs_grad_short(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, const float* lse,
                          const float* entropy, const float* grad_logprob,
                          const float* grad_entropy, T* __restrict__ out) {
  constexpr int kVec = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int vocab = static_cast<int>(logits.width);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kShortWaves + wave; r < logits.n;
       r += static_cast<int64_t>(gridDim.x) * kShortWaves) {
    const int64_t target = token(targets, r);
    const T* x = static_cast<const T*>(logits.data) + row_start(logits, r);
    T* d = out + r * vocab;
    const ShortRow<T> row(x, d, vocab, lane);
    Words w[R];
    row.template load<true>(w, lane);
    const float single = row.load_alone();
    const bool counts = grad_logprob && target != ignore;
    float g = counts ? grad_logprob[r] : 0.f;
    if (counts && (target < 0 || target >= vocab)) g = quiet_nan();
    const int hit = target >= 0 && target < vocab ? static_cast<int>(target) : -1;
    const float h = kEntropy ? grad_entropy[r] : 0.f, big_h = kEntropy ? entropy[r] : 0.f;
    const float l = lse[r];
    auto write = [&](auto one) {
      if (row.alone >= 0) d[row.alone] = narrow<T>(one(single) + (row.alone == hit ? g : 0.f));
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int j0 = row.head + (k * kWave + lane) * kVec;
        if (k * kWave + lane >= row.units) continue;
        Pack<T, kVec> z;
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          z.v[i] = narrow<T>(one(widen(values_of<T>(w[k]).v[i])) + (j0 + i == hit ? g : 0.f));
        store_stream<kVec>(d + j0, z);
      }
    };
    if (l == -INFINITY) {
      g = 0.f;
      write([](float v) { return v != v ? v : 0.f; });
    } else if (fabsf(l) > kFarLse) {
      float most = single, s = 0.f;
      each_value(row, w, single, lane, [&](float v, int) { most = fmaxf(most, v); });
      most = wave_max(most);
      each_value(row, w, single, lane,
                 [&](float v, int) { s += exp2_fast((v - most) * kLog2e); });
      const float ls = log2_fast(wave_sum(s)) * kLn2;
      write([&](float v) {
        const float logp = (v - most) - ls, p = exp2_fast(logp * kLog2e);
        float y = -g * p;
        if (kEntropy && p != 0.f) y -= h * p * (logp + big_h);
        return y;
      });
    } else {
      write(RowGrad<kEntropy>(l, big_h, g, h));
    }
  }
}

bool is_short(int64_t vocab, int32_t dtype) {
  return vocab * dtype_bytes(dtype) <= kShortUnits * 16;
}
// How a row is split: short ones not at all, others not from 512 rows on, two
// blocks to a CU; else so that there are as many blocks, each with a unit to every
// thread at least.
Split split_of(int64_t n, int64_t vocab, int32_t dtype, int32_t top) {
  const int64_t least = (top ? kTopThreads : kThreads) * (16 / dtype_bytes(dtype));
  Split s;
  const int64_t wanted = std::min<int64_t>(kWave, 512 / std::max<int64_t>(n, 1));
  s.length = vocab;
  if (wanted > 1 && vocab > least && !is_short(vocab, dtype)) {
    s.length = (vocab + wanted - 1) / wanted;
    s.length = std::max(least, (s.length + 63) / 64 * 64);
  }
  s.parts = static_cast<int>((vocab + s.length - 1) / s.length);
  s.stride = (static_cast<int64_t>(sizeof(Part)) + 8 * top + 15) & ~15ll;
  s.work = nullptr;
  return s;
}

template <typename T, int NT, bool kTop>
int launch_rows(const ms_rows_t& logits, const ms_tokens_t& targets, int64_t ignore,
                const Outputs& out, const Split& split, hipStream_t s) {
  if (!fits(logits.n * split.parts, NT)) return MS_OPS_EINVAL;
  return launch(out.entropy ? k_logprobs<T, NT, kTop, true> : k_logprobs<T, NT, kTop, false>,
                logits.n * split.parts, NT, s, logits, targets, ignore, out, split);
}

template <typename T, int R>
int launch_short(const ms_rows_t& logits, const ms_tokens_t& targets, int64_t ignore,
                  const Outputs& out, hipStream_t s) {
  const int64_t blocks =
      std::min<int64_t>(kShortBlocks, (logits.n + kShortWaves - 1) / kShortWaves);
  return launch(out.top ? out.entropy ? k_logprobs_short<T, R, true, true>
                                      : k_logprobs_short<T, R, true, false>
                : out.entropy ? k_logprobs_short<T, R, false, true>
                              : k_logprobs_short<T, R, false, false>,
                blocks, kShortThreads, s, logits, targets, ignore, out);
}

template <typename T>
int logprobs_as(const ms_rows_t& logits, const ms_tokens_t& targets, int64_t ignore,
                const Outputs& out, const Split& split, hipStream_t s) {
  const int64_t lane_units = (logits.width * static_cast<int64_t>(sizeof(T)) + 1023) / 1024;
  if (is_short(logits.width, logits.dtype)) {
    return (lane_units <= 1   ? launch_short<T, 1>
            : lane_units <= 2 ? launch_short<T, 2>
            : lane_units <= 4 ? launch_short<T, 4>
                              : launch_short<T, 8>)(logits, targets, ignore, out, s);
  }
  const bool mid = logits.width * static_cast<int64_t>(sizeof(T)) <=
                   kMidUnits * 16 / (out.top ? 2 : 1);
  const int rc =
      out.top && mid ? launch_rows<T, kMidThreads, true>(logits, targets, ignore, out, split, s)
      : mid     ? launch_rows<T, kMidThreads, false>(logits, targets, ignore, out, split, s)
      : out.top ? launch_rows<T, kTopThreads, true>(logits, targets, ignore, out, split, s)
                : launch_rows<T, kThreads, false>(logits, targets, ignore, out, split, s);
  if (rc || split.parts == 1) return rc;
  return launch(k_join_parts<T>, logits.n, kThreads, s, logits, targets, ignore, out, split);
}

template <typename T>
int grad_as(const ms_rows_t& logits, const ms_tokens_t& targets, int64_t ignore, const float* lse,
            const float* entropy, const float* grad_logprob, const float* grad_entropy,
            void* dlogits, hipStream_t s) {
  if (is_short(logits.width, logits.dtype)) {
    const int64_t lane_units = (logits.width * static_cast<int64_t>(sizeof(T)) + 1023) / 1024;
    const int64_t short_blocks =
        std::min<int64_t>(kShortBlocks, (logits.n + kShortWaves - 1) / kShortWaves);
#define SHORT(R) (grad_entropy ? k_logprobs_grad_short<T, R, true> : k_logprobs_grad_short<T, R, false>)
    return launch(lane_units <= 1   ? SHORT(1)
                  : lane_units <= 2 ? SHORT(2)
                  : lane_units <= 4 ? SHORT(4)
                                    : SHORT(8),
                  short_blocks, kShortThreads, s, logits, targets, ignore, lse, entropy,
                  grad_logprob, grad_entropy, static_cast<T*>(dlogits));
#undef SHORT
  }
  constexpr int64_t kEach = kGradGroup * kGradThreads * (16 / sizeof(T));
  const int64_t per_row = std::max<int64_t>((logits.width + kEach - 1) / kEach, 1);
  if (!fits(logits.n * per_row, kGradThreads)) return MS_OPS_EINVAL;
  return launch(grad_entropy ? k_logprobs_grad<T, true> : k_logprobs_grad<T, false>,
                logits.n * per_row, kGradThreads, s, logits, targets, ignore, lse, entropy,
                grad_logprob, grad_entropy, static_cast<int>(per_row), static_cast<T*>(dlogits));
}

}  // namespace

extern "C" int64_t ms_logprobs_workspace(int64_t n, int64_t vocab, int32_t dtype, int32_t top) {
  if (n < 0 || n > INT32_MAX || vocab < 1 || !good_dtype(dtype) || top < 0) return -1;
  const Split s = split_of(n, vocab, dtype, top);
  return s.parts > 1 ? n * s.parts * s.stride : 0;
}

extern "C" int ms_logprobs(const ms_rows_t* logits, const ms_tokens_t* targets,
                           int64_t ignore_index, int32_t top, float* logprob, float* entropy,
                           float* lse, float* top_logprob, int64_t* top_id, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  if (!good_rows(logits) || !good_tokens(targets) || targets->n != logits->n) return MS_OPS_EINVAL;
  if (logits->width < 1 || logits->width > INT32_MAX - 65536) return MS_OPS_EINVAL;
  if (top < 0 || top > MS_OPS_MAX_TOP || top > logits->width) return MS_OPS_EINVAL;
  if (logits->n == 0) return MS_OPS_OK;
  if (!logprob || !lse || (top && (!top_logprob || !top_id))) return MS_OPS_EINVAL;
  Split split = split_of(logits->n, logits->width, logits->dtype, top);
  if (split.parts > 1 &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
       workspace_bytes < ms_logprobs_workspace(logits->n, logits->width, logits->dtype, top)))
    return MS_OPS_EWORKSPACE;
  split.work = static_cast<char*>(workspace);
  const Outputs out = {logprob, entropy, lse, top_logprob, top_id, top};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (logits->dtype) {
    case MS_OPS_F32: return logprobs_as<float>(*logits, *targets, ignore_index, out, split, s);
    case MS_OPS_F16: return logprobs_as<f16>(*logits, *targets, ignore_index, out, split, s);
    default: return logprobs_as<bf16>(*logits, *targets, ignore_index, out, split, s);
  }
}

extern "C" int ms_logprobs_grad(const ms_rows_t* logits, const ms_tokens_t* targets,
                                int64_t ignore_index, const float* lse, const float* entropy,
                                const float* grad_logprob, const float* grad_entropy,
                                void* dlogits, void* stream) {
  if (!good_rows(logits) || !good_tokens(targets) || targets->n != logits->n) return MS_OPS_EINVAL;
  if (logits->width < 1 || logits->width > INT32_MAX - 65536) return MS_OPS_EINVAL;
  if (logits->n == 0) return MS_OPS_OK;
  if (!lse || !dlogits || (grad_entropy && !entropy)) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (logits->dtype) {
    case MS_OPS_F32:
      return grad_as<float>(*logits, *targets, ignore_index, lse, entropy, grad_logprob,
                            grad_entropy, dlogits, s);
    case MS_OPS_F16:
      return grad_as<f16>(*logits, *targets, ignore_index, lse, entropy, grad_logprob,
                          grad_entropy, dlogits, s);
    default:
      return grad_as<bf16>(*logits, *targets, ignore_index, lse, entropy, grad_logprob,
                           grad_entropy, dlogits, s);
  }
}
