// act8.hip — activations held in 8 bits between forward and backward (gfx950).
//
// Blocks of 32 values share a power-of-two scale, so that dividing by it is
// exact and a code is one rounding of the value.

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
__device__ __forceinline__ int8_t code_of(float x, uint32_t e) {
  return e == 255u ? 0 : static_cast<int8_t>(static_cast<int>(rintf(x * inverse_step(e))));
}

struct Act {
  float f, df;
};

constexpr float kLog2e = 1.44269504f;
// Exponentials are taken 2^32 too large and the results put right by a last
// product: v_exp_f32 flushes results below 2^-126, the product does not, so
// the far tails are right down to the smallest denormal.
constexpr float kLift = 32.f, kDrop = 2.3283064e-10f;   // 2^-32
__device__ __forceinline__ float lifted_exp2(float y) {
  return __builtin_amdgcn_exp2f(y + kLift);
}

// x s(z) and its derivative s + x s (1 - s) z', s the logistic function.  With
// e = exp(-|z|), r = 1 / (1 + e): s is r or e r, 1 - s the other.
__device__ __forceinline__ Act logistic_act(float x, float z, float dz) {
  const float e = lifted_exp2(fabsf(z) * -kLog2e);
  const float r = __builtin_amdgcn_rcpf(fmaf(e, kDrop, 1.f));
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

template <int K>
__device__ __forceinline__ Act act(float x) {
  if (K == MS_ACT_GELU) {
    // Phi(-a) = exp(-a^2 / 2) Q(a), Q = erfcx(a / sqrt 2) / 2 as t P(t) with
    // t = 1 / (1 + 0.37 a): P by a weighted least squares fit of the relative
    // error (2e-7; 5e-7 as evaluated), so the tail needs no difference.
    const float m = fabsf(x), a = m > 15.f ? 15.f : m;      // NaN stays
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.37f, 1.f));
    float q = -0.0313271917f;
    q = fmaf(q, t, 0.135133371f);
    q = fmaf(q, t, -0.194299534f);
    q = fmaf(q, t, 0.0645160899f);
    q = fmaf(q, t, 0.0134064732f);
    q = fmaf(q, t, 0.0901831239f);
    q = fmaf(q, t, 0.127163798f);
    q = fmaf(q, t, 0.147615328f);
    q = fmaf(q, t, 0.147608608f) * t;
    const float e = lifted_exp2(a * a * (-0.5f * kLog2e));
    Act r;
    // x Phi(x) = max(x, 0) - a Phi(-a);  Phi + x phi is w below 0, 1 - w above
    r.f = fmaf(a * q * e, -kDrop, fmaxf(x, 0.f));
    const float w = fmaf(a, -0.398942280f, q) * e;
    r.df = x < 0.f ? w * kDrop : fmaf(w, -kDrop, 1.f);
    return r;
  }
  if (K == MS_ACT_GELU_TANH) {
    const float c = 2.f * 0.797884561f, x2 = x * x;
    return logistic_act(x, c * x * fmaf(x2, 0.044715f, 1.f),
                        fmaf(fminf(x2, 4e4f), 3.f * 0.044715f * c, c));
  }
  return logistic_act(x, x, 1.f);
}

// One thread per block of 32.
template <typename T, bool kRows>
__device__ __forceinline__ uint32_t hold(const T* x, const ms_rows_t& m, int64_t i0, int64_t n,
                                         int8_t* codes, uint8_t* exponents) {
  uint32_t most = 0;
  for (int64_t i = i0; i < n && i < i0 + kBlock; ++i) {
    const float v = widen(kRows ? x[row_start(m, i / m.width) + i % m.width] : x[i]);
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    most = b > most ? b : most;
  }
  const uint32_t e = exponent_of(most);
  exponents[i0 / kBlock] = static_cast<uint8_t>(e);
  for (int64_t i = i0; i < n && i < i0 + kBlock; ++i)
    codes[i] = code_of(widen(kRows ? x[row_start(m, i / m.width) + i % m.width] : x[i]), e);
  return e;
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_pack(const T* x, int64_t n, int8_t* codes, uint8_t* exponents) {
  const ms_rows_t none = {};
  for (int64_t b = blockIdx.x * 256ll + threadIdx.x; b * kBlock < n; b += gridDim.x * 256ll)
    hold<T, false>(x, none, b * kBlock, n, codes, exponents);
}

template <typename T>
__global__ void __launch_bounds__(256)
    k_unpack(const int8_t* codes, const uint8_t* exponents, int64_t n, T* out) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
    out[i] = narrow<T>(static_cast<float>(codes[i]) * step_of(exponents[i / kBlock]));
}

template <typename T, int K>
__global__ void __launch_bounds__(256)
    k_act8(ms_rows_t h, ms_rows_t up, T* a, int8_t* codes, uint8_t* exponents, int8_t* up_codes,
           uint8_t* up_exponents) {
  const T* x = static_cast<const T*>(h.data);
  const T* u = static_cast<const T*>(up.data);
  const int64_t n = h.n * h.width;
  for (int64_t b = blockIdx.x * 256ll + threadIdx.x; b * kBlock < n; b += gridDim.x * 256ll) {
    hold<T, true>(x, h, b * kBlock, n, codes, exponents);
    if (K == MS_ACT_SWIGLU) hold<T, true>(u, up, b * kBlock, n, up_codes, up_exponents);
    for (int64_t i = b * kBlock; i < n && i < (b + 1) * kBlock; ++i) {
      float f = act<K>(widen(x[row_start(h, i / h.width) + i % h.width])).f;
      if (K == MS_ACT_SWIGLU) f *= widen(u[row_start(up, i / up.width) + i % up.width]);
      a[i] = narrow<T>(f);
    }
  }
}

template <typename T, int K>
__global__ void __launch_bounds__(256)
    k_act8_grad(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                const uint8_t* up_exponents, const T* grad, int64_t n, T* dh, T* dup, T* a) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const Act r = act<K>(static_cast<float>(codes[i]) * step_of(exponents[i / kBlock]));
    const float g = widen(grad[i]);
    if (K == MS_ACT_SWIGLU) {
      const float u = static_cast<float>(up_codes[i]) * step_of(up_exponents[i / kBlock]);
      dh[i] = narrow<T>(g * u * r.df);
      dup[i] = narrow<T>(g * r.f);
      if (a) a[i] = narrow<T>(r.f * u);
    } else {
      dh[i] = narrow<T>(g * r.df);
      if (a) a[i] = narrow<T>(r.f);
    }
  }
}

unsigned blocks_for(int64_t items) {
  const int64_t n = (items + 255) / 256, most = 1 << 20;
  return static_cast<unsigned>(n < most ? n : most);
}

template <typename T>
int act8_as(const ms_rows_t& h, const ms_rows_t& up, int kind, void* a, int8_t* codes,
            uint8_t* exponents, int8_t* up_codes, uint8_t* up_exponents, hipStream_t s) {
  const unsigned blocks = blocks_for((h.n * h.width + kBlock - 1) / kBlock);
  T* out = static_cast<T*>(a);
  switch (kind) {
    case MS_ACT_GELU:
      k_act8<T, MS_ACT_GELU><<<blocks, 256, 0, s>>>(h, up, out, codes, exponents, up_codes,
                                                    up_exponents);
      break;
    case MS_ACT_GELU_TANH:
      k_act8<T, MS_ACT_GELU_TANH><<<blocks, 256, 0, s>>>(h, up, out, codes, exponents, up_codes,
                                                         up_exponents);
      break;
    case MS_ACT_SILU:
      k_act8<T, MS_ACT_SILU><<<blocks, 256, 0, s>>>(h, up, out, codes, exponents, up_codes,
                                                    up_exponents);
      break;
    default:
      k_act8<T, MS_ACT_SWIGLU><<<blocks, 256, 0, s>>>(h, up, out, codes, exponents, up_codes,
                                                      up_exponents);
  }
  return launched();
}

template <typename T>
int act8_grad_as(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                 const uint8_t* up_exponents, const void* grad, int kind, int64_t n, void* dh,
                 void* dup, void* a, hipStream_t s) {
  const unsigned blocks = blocks_for(n);
  const T* g = static_cast<const T*>(grad);
  T *d = static_cast<T*>(dh), *du = static_cast<T*>(dup), *out = static_cast<T*>(a);
  switch (kind) {
    case MS_ACT_GELU:
      k_act8_grad<T, MS_ACT_GELU><<<blocks, 256, 0, s>>>(codes, exponents, up_codes, up_exponents,
                                                         g, n, d, du, out);
      break;
    case MS_ACT_GELU_TANH:
      k_act8_grad<T, MS_ACT_GELU_TANH><<<blocks, 256, 0, s>>>(codes, exponents, up_codes,
                                                              up_exponents, g, n, d, du, out);
      break;
    case MS_ACT_SILU:
      k_act8_grad<T, MS_ACT_SILU><<<blocks, 256, 0, s>>>(codes, exponents, up_codes, up_exponents,
                                                         g, n, d, du, out);
      break;
    default:
      k_act8_grad<T, MS_ACT_SWIGLU><<<blocks, 256, 0, s>>>(codes, exponents, up_codes,
                                                           up_exponents, g, n, d, du, out);
  }
  return launched();
}

bool good_kind(int32_t k) { return k >= MS_ACT_GELU && k <= MS_ACT_SWIGLU; }

}  // namespace

extern "C" int ms_pack8(const void* x, int32_t dtype, int64_t n, int8_t* codes, uint8_t* exponents,
                        void* stream) {
  if (!good_dtype(dtype) || n < 0) return MS_OPS_EINVAL;
  if (n == 0) return MS_OPS_OK;
  if (!x || !codes || !exponents) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for((n + kBlock - 1) / kBlock);
  switch (dtype) {
    case MS_OPS_F32:
      k_pack<float><<<blocks, 256, 0, s>>>(static_cast<const float*>(x), n, codes, exponents);
      break;
    case MS_OPS_F16:
      k_pack<f16><<<blocks, 256, 0, s>>>(static_cast<const f16*>(x), n, codes, exponents);
      break;
    default:
      k_pack<bf16><<<blocks, 256, 0, s>>>(static_cast<const bf16*>(x), n, codes, exponents);
  }
  return launched();
}

extern "C" int ms_unpack8(const int8_t* codes, const uint8_t* exponents, int64_t n, int32_t dtype,
                          void* out, void* stream) {
  if (!good_dtype(dtype) || n < 0) return MS_OPS_EINVAL;
  if (n == 0) return MS_OPS_OK;
  if (!out || !codes || !exponents) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for(n);
  switch (dtype) {
    case MS_OPS_F32:
      k_unpack<float><<<blocks, 256, 0, s>>>(codes, exponents, n, static_cast<float*>(out));
      break;
    case MS_OPS_F16:
      k_unpack<f16><<<blocks, 256, 0, s>>>(codes, exponents, n, static_cast<f16*>(out));
      break;
    default:
      k_unpack<bf16><<<blocks, 256, 0, s>>>(codes, exponents, n, static_cast<bf16*>(out));
  }
  return launched();
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
  if (!good_kind(kind) || !good_dtype(dtype) || n < 0) return MS_OPS_EINVAL;
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
