// logprobs.hip — log probabilities of given tokens, entropy, the most likely
// alternatives, and the gradient of the logits (gfx950).

#include "ops_common.h"

namespace {

using namespace ops;

// exp x = 2^(x L); the same rounded L everywhere, and its own inverse, so
// that what L is off by only rescales the logits by 1 + 1.3e-8.
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.69314718f;

// Rows whose maximum (or lse) is beyond this are computed from x - max, and
// their gradient finds max and sum again: an fp32 lse no longer tells them
// apart from their maximum (a row masked with the type's lowest value).
constexpr float kFar = 1024.f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int k = 32; k; k >>= 1) x = fmaxf(x, __shfl_xor(x, k));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k);
  return x;
}

// Over the block, the result in every thread; `slot`: one float per wave.
template <int W, typename F>
__device__ __forceinline__ float block_join(float x, float* slot, F join) {
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = x;
  __syncthreads();
  float r = slot[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r = join(r, slot[w]);
  return r;
}

// Falling value, then rising index: a 64-bit key that is larger for what
// comes first.  NaN is above +inf; -0 equals +0.
constexpr uint32_t kNanKey = 0xFFFFFFF0u;      // with any index below all ones
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return kNanKey;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == kNanKey) return quiet_nan();
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct RowStats {
  float lse, logprob, entropy;
};

// Sums of the row over y = x L - m2 (m2 a whole number near max L, or far
// rows: y = (x - max) L): s = sum 2^y, t = sum 2^y y.
__device__ __forceinline__ RowStats finish(float most, float s, float t, float given, bool good) {
  RowStats r;
  const bool far = !(fabsf(most) <= kFar);
  const float ls = log2_fast(s);
  const bool empty = most == -INFINITY && s == 0.f;
  if (empty) {
    r.lse = -INFINITY;
    r.logprob = -INFINITY;
    r.entropy = 0.f;
  } else if (far && most != -INFINITY) {
    r.lse = most + ls * kLn2;
    r.logprob = (given - most) - ls * kLn2;
    r.entropy = (ls - t / s) * kLn2;
  } else {
    const float m2 = most == -INFINITY ? 0.f : rintf(most * kLog2e);
    r.lse = (m2 + ls) * kLn2;
    // given - max is (nearly) exact; what m2 rounded off comes back with log s
    const float base = most == -INFINITY ? 0.f : most;
    r.logprob = (given - base) + (fmaf(base, kLog2e, -m2) - ls) * kLn2;
    r.entropy = (ls - t / s) * kLn2;
  }
  if (!good) r.logprob = quiet_nan();
  return r;
}

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_logprobs(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, int top, float* logprob,
               float* entropy, float* lse, float* top_logprob, int64_t* top_id) {
  __shared__ float slot[kWaves];
  __shared__ uint64_t best[kWaves];
  for (int64_t r = blockIdx.x; r < logits.n; r += gridDim.x) {
    const T* x = static_cast<const T*>(logits.data) + row_start(logits, r);
    const int64_t v = logits.width;
    float most = -INFINITY;
    for (int64_t j = threadIdx.x; j < v; j += kThreads) most = fmaxf(most, widen(x[j]));
    most = block_join<kWaves>(wave_max(most), slot, [](float a, float b) { return fmaxf(a, b); });
    const bool far = !(fabsf(most) <= kFar) && most != -INFINITY;
    const float base = most == -INFINITY ? 0.f : most;
    const float m2 = rintf(base * kLog2e);
    float s = 0.f, t = 0.f;
    for (int64_t j = threadIdx.x; j < v; j += kThreads) {
      const float xj = widen(x[j]);
      const float y = far ? (xj - base) * kLog2e : fmaf(xj, kLog2e, -m2);
      const float e = exp2_fast(y);
      s += e;
      t += e * fmaxf(y, -1e30f);
    }
    auto add = [](float a, float b) { return a + b; };
    s = block_join<kWaves>(wave_sum(s), slot, add);
    t = block_join<kWaves>(wave_sum(t), slot, add);
    const int64_t y = token(targets, r);
    const bool good = y >= 0 && y < v;
    const RowStats st = finish(most, s, t, good ? widen(x[y]) : 0.f, good);
    if (threadIdx.x == 0) {
      lse[r] = st.lse;
      logprob[r] = y == ignore ? 0.f : st.logprob;
      if (entropy) entropy[r] = st.entropy;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t mine = 0;
      for (int64_t j = threadIdx.x; j < v; j += kThreads) {
        const uint64_t key = static_cast<uint64_t>(order_key(widen(x[j]))) << 32 |
                             static_cast<uint32_t>(~static_cast<uint32_t>(j));
        if (key > mine && key < last) mine = key;
      }
      for (int b = 32; b; b >>= 1) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(mine), b);
        if (other > mine) mine = other;
      }
      __syncthreads();
      if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
      __syncthreads();
      mine = best[0];
      for (int w = 1; w < kWaves; ++w) mine = best[w] > mine ? best[w] : mine;
      last = mine;
      if (threadIdx.x == 0) {
        const uint32_t j = ~static_cast<uint32_t>(mine);
        const float value = key_value(static_cast<uint32_t>(mine >> 32));
        top_id[r * top + k] = j;
        top_logprob[r * top + k] = finish(most, s, t, value, true).logprob;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_logprobs_grad(ms_rows_t logits, ms_tokens_t targets, int64_t ignore, const float* lse,
                    const float* entropy, const float* grad_logprob, const float* grad_entropy,
                    T* __restrict__ out) {
  __shared__ float slot[kWaves];
  for (int64_t r = blockIdx.x; r < logits.n; r += gridDim.x) {
    const T* x = static_cast<const T*>(logits.data) + row_start(logits, r);
    const int64_t v = logits.width;
    T* d = out + r * v;
    const int64_t y = token(targets, r);
    float g = grad_logprob && y != ignore ? grad_logprob[r] : 0.f;
    if (grad_logprob && y != ignore && (y < 0 || y >= v)) g = quiet_nan();
    const float h = grad_entropy ? grad_entropy[r] : 0.f;
    const float big_h = grad_entropy ? entropy[r] : 0.f;
    const float l = lse[r];
    if (l == -INFINITY) {
      for (int64_t j = threadIdx.x; j < v; j += kThreads) d[j] = narrow<T>(0.f);
      continue;
    }
    float base = l, ls = 0.f;
    if (fabsf(l) > kFar) {
      float most = -INFINITY;
      for (int64_t j = threadIdx.x; j < v; j += kThreads) most = fmaxf(most, widen(x[j]));
      most =
          block_join<kWaves>(wave_max(most), slot, [](float a, float b) { return fmaxf(a, b); });
      float s = 0.f;
      for (int64_t j = threadIdx.x; j < v; j += kThreads)
        s += exp2_fast((widen(x[j]) - most) * kLog2e);
      s = block_join<kWaves>(wave_sum(s), slot, [](float a, float b) { return a + b; });
      base = most;
      ls = log2_fast(s) * kLn2;
    }
    for (int64_t j = threadIdx.x; j < v; j += kThreads) {
      const float logp = (widen(x[j]) - base) - ls;
      const float p = exp2_fast(logp * kLog2e);
      float dj = j == y ? g - g * p : -g * p;
      if (p != 0.f) dj -= h * p * (logp + big_h);
      d[j] = narrow<T>(dj);
    }
  }
}

unsigned blocks_for(int64_t n) {
  const int64_t most = 1 << 20;
  return static_cast<unsigned>(n < most ? n : most);
}

}  // namespace

extern "C" int64_t ms_logprobs_workspace(int64_t, int64_t, int32_t, int32_t) { return 0; }

extern "C" int ms_logprobs(const ms_rows_t* logits, const ms_tokens_t* targets,
                           int64_t ignore_index, int32_t top, float* logprob, float* entropy,
                           float* lse, float* top_logprob, int64_t* top_id, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (!good_rows(logits) || !good_tokens(targets) || targets->n != logits->n) return MS_OPS_EINVAL;
  if (logits->width < 1 || logits->width > INT32_MAX) return MS_OPS_EINVAL;
  if (top < 0 || top > MS_OPS_MAX_TOP || top > logits->width) return MS_OPS_EINVAL;
  if (logits->n == 0) return MS_OPS_OK;
  if (!logprob || !lse || (top && (!top_logprob || !top_id))) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for(logits->n);
  switch (logits->dtype) {
    case MS_OPS_F32:
      k_logprobs<float><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, top, logprob,
                                                    entropy, lse, top_logprob, top_id);
      break;
    case MS_OPS_F16:
      k_logprobs<f16><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, top, logprob,
                                                  entropy, lse, top_logprob, top_id);
      break;
    default:
      k_logprobs<bf16><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, top, logprob,
                                                   entropy, lse, top_logprob, top_id);
  }
  return launched();
}

extern "C" int ms_logprobs_grad(const ms_rows_t* logits, const ms_tokens_t* targets,
                                int64_t ignore_index, const float* lse, const float* entropy,
                                const float* grad_logprob, const float* grad_entropy,
                                void* dlogits, void* stream) {
  if (!good_rows(logits) || !good_tokens(targets) || targets->n != logits->n) return MS_OPS_EINVAL;
  if (logits->width < 1 || logits->width > INT32_MAX) return MS_OPS_EINVAL;
  if (logits->n == 0) return MS_OPS_OK;
  if (!lse || !dlogits || (grad_entropy && !entropy)) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for(logits->n);
  switch (logits->dtype) {
    case MS_OPS_F32:
      k_logprobs_grad<float><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, lse,
                                                         entropy, grad_logprob, grad_entropy,
                                                         static_cast<float*>(dlogits));
      break;
    case MS_OPS_F16:
      k_logprobs_grad<f16><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, lse,
                                                       entropy, grad_logprob, grad_entropy,
                                                       static_cast<f16*>(dlogits));
      break;
    default:
      k_logprobs_grad<bf16><<<blocks, kThreads, 0, s>>>(*logits, *targets, ignore_index, lse,
                                                        entropy, grad_logprob, grad_entropy,
                                                        static_cast<bf16*>(dlogits));
  }
  return launched();
}
