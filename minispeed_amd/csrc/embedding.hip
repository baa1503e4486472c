// embedding.hip — token embedding and its gradient (gfx950).
//
//   out[t, :]    = scale * table[id_t, :]
//   dtable[v, :] = scale * sum_{t: id_t = v} grad[t, :], t rising

#include <algorithm>

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

// The gradient's table, in three launches:
//
//   k_sort_tokens  kSortRows rows of the table or fewer to a block: it counts
//                  its rows' tokens in LDS, wave w over the w-th part of the
//                  list, and places their positions stably, so `position` ends
//                  up sorted by (id, t).  The other blocks of the same launch
//                  clear the table, which takes longer.
//   k_sum_spans    `span` sorted positions to a wave and a slice of the width:
//                  fp32 sums of each id's rows, written to the table where the
//                  id's tokens lie within the span, left as a partial sum where
//                  they go on before (slot 0) or behind (slot 1) it.  An id
//                  with half of the tokens costs what others cost.
//   k_join_spans   adds up the partial sums of ids that cross spans.
//
// Every order is that of (id, t) and of the spans: no atomics on sums.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRows = 1024;
constexpr int kSortSteps = 8;             // groups of 64 tokens in flight per wave

struct Sorted {
  int32_t* start;       // [vocab + 1]: where each id's tokens begin
  int32_t* id;          // [n]
  int32_t* position;    // [n]
  float* partial;       // [spans, 2, width]
};

__device__ __forceinline__ int wave_scan(int x) {
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) {
    const int y = __shfl_up(x, k);
    if ((threadIdx.x & 63) >= k) x += y;
  }
  return x;
}

__global__ void __launch_bounds__(kSortThreads)
    k_sort_tokens(ms_tokens_t ids, int64_t vocab, int64_t skip, int buckets, int rows_each,
                  Sorted out, uint4* table, int64_t table_bytes) {
  __shared__ int count[kSortWaves][kSortRows];
  __shared__ int wave_sum[kSortWaves];
  if (blockIdx.x >= static_cast<unsigned>(buckets)) {
    const int64_t step = static_cast<int64_t>(gridDim.x - buckets) * kSortThreads;
    int64_t i = static_cast<int64_t>(blockIdx.x - buckets) * kSortThreads + threadIdx.x;
    const int64_t vectors = table_bytes / 16, rest = (table_bytes & 15) / 2;
    if (i < rest) reinterpret_cast<uint16_t*>(table + vectors)[i] = 0;
    for (; i < vectors; i += step) table[i] = uint4{0, 0, 0, 0};
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * rows_each;
  const int rows = static_cast<int>(vocab - lo < rows_each ? vocab - lo : rows_each);
  for (int i = threadIdx.x; i < kSortWaves * kSortRows; i += kSortThreads) (&count[0][0])[i] = 0;
  const int64_t part = ((ids.n + kSortThreads - 1) / kSortThreads) * kWave;
  const int64_t first = wave * part, last = first + part < ids.n ? first + part : ids.n;
  __syncthreads();

  // row of my bucket, -1: below it, -2: no row of mine or above
  auto row_of = [&](int64_t t) {
    if (t >= last) return -2;
    const int64_t id = token(ids, t);
    if (id < 0 || id >= lo + rows || id == skip) return -2;
    return id < lo ? -1 : static_cast<int>(id - lo);
  };
  int below = 0;
  for (int64_t t0 = first; t0 < last; t0 += kWave * kSortSteps) {
    int row[kSortSteps];
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) row[k] = row_of(t0 + k * kWave + lane);
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) {
      below += row[k] == -1;
      if (row[k] >= 0) atomicAdd(&count[wave][row[k]], 1);
    }
  }
  for (int k = 32; k; k >>= 1) below += __shfl_xor(below, k);
  if (lane == 0) wave_sum[wave] = below;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += wave_sum[w];
  __syncthreads();

  // exclusive sum over the rows, then over the waves of each row
  const int r = threadIdx.x;
  int mine = 0;
  if (r < rows)
    for (int w = 0; w < kSortWaves; ++w) mine += count[w][r];
  const int upto = wave_scan(mine);
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int at = base + upto - mine;
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
  if (r < rows) {
    out.start[lo + r] = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w][r];
      count[w][r] = at;
      at += c;
    }
    if (lo + r == vocab - 1) out.start[vocab] = at;
  }
  __syncthreads();

  for (int64_t t0 = first; t0 < last; t0 += kWave * kSortSteps) {
    int row[kSortSteps];
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) row[k] = row_of(t0 + k * kWave + lane);
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) {
      uint64_t left = __ballot(row[k] >= 0);
      while (left) {                               // once per different id
        const int lead = __ffsll(static_cast<unsigned long long>(left)) - 1;
        const int which = read_lane(row[k], lead);
        const uint64_t same = __ballot(row[k] == which);
        const int to = count[wave][which];
        if (row[k] == which) {
          const int p = to + __popcll(same & ((1ull << lane) - 1));
          out.id[p] = static_cast<int32_t>(lo + which);
          out.position[p] = static_cast<int32_t>(t0 + k * kWave + lane);
        }
        if (lane == lead) count[wave][which] = to + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// My N values of a row; `whole`: none of the wave's reach past the width.
template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load_slice(const T* row, int64_t c, int64_t width,
                                                 bool whole) {
  if (whole) return load<N>(row + c);
  Pack<T, N> x;
#pragma unroll
  for (int k = 0; k < N; ++k) x.v[k] = c + k < width ? row[c + k] : static_cast<T>(0.f);
  return x;
}
template <int N, typename T>
__device__ __forceinline__ void store_slice(T* row, int64_t c, int64_t width, bool whole,
                                            const Pack<T, N>& x) {
  if (whole) {
    store<N>(row + c, x);
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (c + k < width) row[c + k] = x.v[k];
}

constexpr int kSumThreads = 256, kSumWaves = kSumThreads / kWave;
constexpr int kSumDepth = 8;              // rows in flight per wave

template <typename T, int N>
__global__ void __launch_bounds__(kSumThreads)
    k_sum_spans(ms_rows_t grad, int64_t vocab, float scale, int span, int slices, Sorted in,
                T* __restrict__ table) {
  const int lane = threadIdx.x & 63;
  const int64_t job = blockIdx.x * static_cast<int64_t>(kSumWaves) + (threadIdx.x >> 6);
  const int64_t s = job / slices, width = grad.width;
  const int64_t c = ((job - s * slices) * kWave + lane) * N;
  const int total = in.start[vocab];
  const int64_t first = s * span;
  if (first >= total) return;
  const int n = static_cast<int>(total - first < span ? total - first : span);
  const int mine = lane < n ? lane : n - 1;
  const int id = in.id[first + mine];
  const int64_t offset = row_start(grad, in.position[first + mine]);
  const int before = first > 0 ? in.id[first - 1] : -1;
  const int behind = first + n < total ? in.id[first + n] : -1;
  const int next = __shfl_down(id, 1);
  const uint64_t ends = __ballot(lane < n && (lane == n - 1 || next != id));
  const T* g = static_cast<const T*>(grad.data);

  const bool whole = __all(c + N <= width);
  float sum[N];
#pragma unroll
  for (int k = 0; k < N; ++k) sum[k] = 0.f;
  bool open = read_lane(id, 0) == before;
  for (int i0 = 0; i0 < n; i0 += kSumDepth) {
    Pack<T, N> x[kSumDepth];                        // past the last: the last again, not added
#pragma unroll
    for (int u = 0; u < kSumDepth; ++u)
      x[u] = load_slice<N>(g + read_lane(offset, i0 + u < n ? i0 + u : n - 1), c, width, whole);
#pragma unroll
    for (int u = 0; u < kSumDepth; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k] += widen(x[u].v[k]);
      if (!(ends >> i & 1)) continue;
      const int row = read_lane(id, i);
      if (open || (i == n - 1 && row == behind)) {
        Pack<float, N> y;
#pragma unroll
        for (int k = 0; k < N; ++k) y.v[k] = sum[k];
        store_slice<N>(in.partial + (s * 2 + (open ? 0 : 1)) * width, c, width, whole, y);
      } else {
        Pack<T, N> y;
#pragma unroll
        for (int k = 0; k < N; ++k) y.v[k] = narrow<T>(sum[k] * scale);
        store_slice<N>(table + row * width, c, width, whole, y);
      }
      open = false;
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k] = 0.f;
    }
  }
}

// One block per span that an id's tokens leave to the right, having begun in
// it, and per kWave values of the width: its waves take a part of the partial
// sums each.
template <typename T>
__global__ void __launch_bounds__(kSumThreads)
    k_join_spans(int64_t width, int64_t vocab, float scale, int span, Sorted in,
                 T* __restrict__ table) {
  __shared__ float part[kSumWaves][kWave];
  const int64_t s = blockIdx.x, end = (s + 1) * span;
  if (end >= in.start[vocab]) return;
  const int id = in.id[end - 1];
  if (in.id[end] != id || in.start[id] < s * span) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = blockIdx.y * static_cast<int64_t>(kWave) + lane;
  const int64_t parts = (in.start[id + 1] - 1) / span - s + 1;
  const int64_t each = (parts + kSumWaves - 1) / kSumWaves;
  float sum = 0.f;
  if (c < width)
    for (int64_t k = wave * each; k < (wave + 1) * each && k < parts; ++k)
      sum += in.partial[((s + k) * 2 + (k == 0)) * width + c];
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < width) {
    for (int w = 1; w < kSumWaves; ++w) sum += part[w][lane];
    table[id * width + c] = narrow<T>(sum * scale);
  }
}

int64_t align16(int64_t bytes) { return (bytes + 15) & ~15ll; }

// How the work is cut; a function of the sizes alone, as the order of the sums
// follows from it.
struct GradShape {
  int buckets, rows_each, vector, slices, span;
  int64_t spans, start_bytes, list_bytes, partial_bytes;
};

GradShape shape_of(int64_t n, int64_t vocab, int64_t width) {
  GradShape g;
  const int64_t wanted = std::max((vocab + kSortRows - 1) / kSortRows,
                                  std::min<int64_t>((vocab + 7) / 8, 64));
  g.rows_each = static_cast<int>((vocab + wanted - 1) / wanted);
  g.buckets = static_cast<int>((vocab + g.rows_each - 1) / g.rows_each);
  g.vector = width >= 2 * kWave ? 4 : width >= kWave ? 2 : 1;
  g.slices = static_cast<int>((width + g.vector * kWave - 1) / (g.vector * kWave));
  g.span = n * g.slices >= (1 << 18) ? 32 : 16;
  g.spans = (n + g.span - 1) / g.span;
  g.start_bytes = align16((vocab + 1) * 4);
  g.list_bytes = align16(n * 4);
  g.partial_bytes = align16(g.spans * 2 * width * 4);
  return g;
}

template <typename T>
int grad_as(const ms_tokens_t& ids, const ms_rows_t& grad, int64_t vocab, float scale,
            int64_t skip, void* dtable, void* workspace, hipStream_t s) {
  const GradShape g = shape_of(ids.n, vocab, grad.width);
  char* w = static_cast<char*>(workspace);
  Sorted sorted;
  sorted.start = reinterpret_cast<int32_t*>(w);
  sorted.id = reinterpret_cast<int32_t*>(w + g.start_bytes);
  sorted.position = reinterpret_cast<int32_t*>(w + g.start_bytes + g.list_bytes);
  sorted.partial = reinterpret_cast<float*>(w + g.start_bytes + 2 * g.list_bytes);
  T* table = static_cast<T*>(dtable);
  const int64_t bytes = vocab * grad.width * static_cast<int64_t>(sizeof(T));
  const int64_t clear =
      std::min<int64_t>((bytes / 16 + kSortThreads) / kSortThreads, 2048);
  k_sort_tokens<<<static_cast<unsigned>(g.buckets + clear), kSortThreads, 0, s>>>(
      ids, vocab, skip, g.buckets, g.rows_each, sorted, static_cast<uint4*>(dtable), bytes);
  if (int rc = launched()) return rc;
  if (ids.n == 0) return MS_OPS_OK;
  const unsigned blocks =
      static_cast<unsigned>((g.spans * g.slices + kSumWaves - 1) / kSumWaves);
  switch (g.vector) {
    case 4:
      k_sum_spans<T, 4><<<blocks, kSumThreads, 0, s>>>(grad, vocab, scale, g.span, g.slices,
                                                       sorted, table);
      break;
    case 2:
      k_sum_spans<T, 2><<<blocks, kSumThreads, 0, s>>>(grad, vocab, scale, g.span, g.slices,
                                                       sorted, table);
      break;
    default:
      k_sum_spans<T, 1><<<blocks, kSumThreads, 0, s>>>(grad, vocab, scale, g.span, g.slices,
                                                       sorted, table);
  }
  if (int rc = launched()) return rc;
  if (g.spans > 1) {
    const dim3 grid(static_cast<unsigned>(g.spans),
                    static_cast<unsigned>((grad.width + kWave - 1) / kWave));
    k_join_spans<T><<<grid, kSumThreads, 0, s>>>(grad.width, vocab, scale, g.span, sorted, table);
  }
  return launched();
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

extern "C" int64_t ms_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t width) {
  if (n < 0 || vocab < 0 || width < 0 || n > INT32_MAX || vocab > INT32_MAX) return -1;
  if (vocab == 0 || width == 0) return 0;
  const GradShape g = shape_of(n, vocab, width);
  return g.start_bytes + 2 * g.list_bytes + g.partial_bytes;
}

extern "C" int ms_embedding_grad(const ms_tokens_t* ids, const ms_rows_t* grad, int64_t vocab,
                                 float scale, int64_t padding_idx, void* dtable, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (!good_tokens(ids) || !good_rows(grad) || grad->n != ids->n || vocab < 0 ||
      vocab > INT32_MAX)
    return MS_OPS_EINVAL;
  if (vocab == 0 || grad->width == 0) return MS_OPS_OK;
  if (!dtable || (reinterpret_cast<uintptr_t>(dtable) & 15)) return MS_OPS_EINVAL;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
      workspace_bytes < ms_embedding_grad_workspace(ids->n, vocab, grad->width))
    return MS_OPS_EWORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (grad->dtype) {
    case MS_OPS_F32:
      return grad_as<float>(*ids, *grad, vocab, scale, padding_idx, dtable, workspace, s);
    case MS_OPS_F16:
      return grad_as<f16>(*ids, *grad, vocab, scale, padding_idx, dtable, workspace, s);
    default:
      return grad_as<bf16>(*ids, *grad, vocab, scale, padding_idx, dtable, workspace, s);
  }
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
