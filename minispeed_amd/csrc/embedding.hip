// embedding.hip — token embedding and its gradient (gfx950).
//
//   out[t, :]    = scale * table[id_t, :]
//   dtable[v, :] = scale * sum_{t: id_t = v} grad[t, :], t rising

#include "ops_common.h"

namespace {

using namespace ops;

template <typename T>
__global__ void __launch_bounds__(256) k_lookup(ms_tokens_t ids, ms_rows_t table, float scale,
                                                T* __restrict__ out) {
  const T* rows = static_cast<const T*>(table.data);
  for (int64_t t = blockIdx.x; t < ids.n; t += gridDim.x) {
    const int64_t id = token(ids, t);
    const bool good = id >= 0 && id < table.n;
    const T* src = rows + (good ? row_start(table, id) : 0);
    T* dst = out + t * table.width;
    for (int64_t c = threadIdx.x; c < table.width; c += blockDim.x)
      dst[c] = narrow<T>(good ? widen(src[c]) * scale : quiet_nan());
  }
}

// One block per row of the table: it walks the ids and adds its tokens' rows
// in order.
template <typename T>
__global__ void __launch_bounds__(256) k_lookup_grad(ms_tokens_t ids, ms_rows_t grad,
                                                     int64_t vocab, float scale, int64_t skip,
                                                     T* __restrict__ dtable) {
  const T* g = static_cast<const T*>(grad.data);
  for (int64_t v = blockIdx.x; v < vocab; v += gridDim.x) {
    for (int64_t c0 = 0; c0 < grad.width; c0 += blockDim.x) {
      const int64_t c = c0 + threadIdx.x;
      float sum = 0.f;
      for (int64_t t0 = 0; t0 < ids.n; t0 += kWave) {
        const int64_t t = t0 + (threadIdx.x & (kWave - 1));
        uint64_t hits = __ballot(t < ids.n && v != skip && token(ids, t < ids.n ? t : 0) == v);
        while (hits) {
          const int b = __ffsll(static_cast<unsigned long long>(hits)) - 1;
          hits &= hits - 1;
          if (c < grad.width) sum += widen(g[row_start(grad, t0 + b) + c]);
        }
      }
      if (c < grad.width) dtable[v * grad.width + c] = narrow<T>(sum * scale);
    }
  }
}

unsigned blocks_for(int64_t n) {
  const int64_t most = 1 << 20;
  return static_cast<unsigned>(n < most ? n : most);
}

}  // namespace

extern "C" int ms_embedding(const ms_tokens_t* ids, const ms_rows_t* table, float scale, void* out,
                            void* stream) {
  if (!good_tokens(ids) || !good_rows(table)) return MS_OPS_EINVAL;
  if (ids->n == 0 || table->width == 0) return MS_OPS_OK;
  if (!out || table->n < 1) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for(ids->n);
  switch (table->dtype) {
    case MS_OPS_F32:
      k_lookup<float><<<blocks, 256, 0, s>>>(*ids, *table, scale, static_cast<float*>(out));
      break;
    case MS_OPS_F16:
      k_lookup<f16><<<blocks, 256, 0, s>>>(*ids, *table, scale, static_cast<f16*>(out));
      break;
    default:
      k_lookup<bf16><<<blocks, 256, 0, s>>>(*ids, *table, scale, static_cast<bf16*>(out));
  }
  return launched();
}

extern "C" int64_t ms_embedding_grad_workspace(int64_t, int64_t, int64_t) { return 0; }

extern "C" int ms_embedding_grad(const ms_tokens_t* ids, const ms_rows_t* grad, int64_t vocab,
                                 float scale, int64_t padding_idx, void* dtable, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (!good_tokens(ids) || !good_rows(grad) || grad->n != ids->n || vocab < 0)
    return MS_OPS_EINVAL;
  if (vocab == 0 || grad->width == 0) return MS_OPS_OK;
  if (!dtable) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = blocks_for(vocab);
  switch (grad->dtype) {
    case MS_OPS_F32:
      k_lookup_grad<float><<<blocks, 256, 0, s>>>(*ids, *grad, vocab, scale, padding_idx,
                                                  static_cast<float*>(dtable));
      break;
    case MS_OPS_F16:
      k_lookup_grad<f16><<<blocks, 256, 0, s>>>(*ids, *grad, vocab, scale, padding_idx,
                                                static_cast<f16*>(dtable));
      break;
    default:
      k_lookup_grad<bf16><<<blocks, 256, 0, s>>>(*ids, *grad, vocab, scale, padding_idx,
                                                 static_cast<bf16*>(dtable));
  }
  return launched();
}

extern "C" int ms_ops_abi_version(void) { return MS_OPS_ABI_VERSION; }

extern "C" const char* ms_ops_error_string(int code) {
  switch (code) {
    case MS_OPS_OK: return "ok";
    case MS_OPS_EINVAL: return "invalid argument";
    case MS_OPS_EWORKSPACE: return "workspace smaller than needed or misaligned";
    default:
      return code > 0 ? hipGetErrorString(static_cast<hipError_t>(code)) : "unknown error code";
  }
}
