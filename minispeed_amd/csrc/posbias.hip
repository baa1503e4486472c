// The learned relative position bias of attention, and the gradient of its table.
//
//   bias[h, i, j] = table[bucket(j - i - first), h]
//   dtable[b, h]  = sum of grad[..., h, i, j] over the pairs with bucket(j - i - first) = b
//
// with query i at position first + i.  A side's n buckets: distances below n / 2 have one
// each, from there on bucket n / 2 + s begins at the least distance a with
// (a / (n/2)) ^ (n - n/2) >= (max_distance / (n/2)) ^ s, and the last one has no end.
// Keys before the query come first, then (not causal) those behind it; causal, keys behind
// the query get -inf and have no gradient.  The first distance of each bucket is worked out
// on the host.
//
// A value depends on j - i alone.  Forward, which only writes, a block sets down the
// values of its diagonals in LDS; a thread has 16 bytes of a row in registers and goes
// down the rows, each time shifting one value in.  Backward, which only reads, a thread
// follows its 16 bytes of neighbouring diagonals down the rows with one register for each
// (loads take any alignment); a block then adds up its diagonals' sums by bucket, each a
// run of neighbours, and a second kernel joins the blocks' sums in their order.
#include "ops_common.h"

#include <algorithm>
#include <cmath>

namespace ops {
namespace {

constexpr int kThreads = 256, kMaxRows = 64, kMaxBuckets = 512;

// First distance of each bucket of a side, n of them; edge[n] is beyond all.
struct edges_t {
  int32_t n, one;
  int32_t edge[kMaxBuckets + 1];
};

struct bias_args {
  const void* table;
  int64_t bucket_stride, head_stride;
  int64_t queries, keys, first;
  int32_t rows, causal;            // rows: of a block
  void* out;
};

// The bucket of a distance of 0 or more.
__device__ __forceinline__ int side_bucket(const int32_t* edge, int n, int one, int64_t away) {
  if (away < one) return static_cast<int>(away);
  if (away >= edge[n - 1]) return n - 1;
  int lo = one, hi = n - 1;          // edge[lo] <= away < edge[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (edge[mid] <= away) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T> __device__ __forceinline__ T minus_infinity() {
  return static_cast<T>(-__builtin_inff());
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_bias(bias_args a, edges_t edges) {
  constexpr int V = 16 / sizeof(T), kSpan = kThreads * V;
  __shared__ T strip[kSpan + kMaxRows];
  __shared__ T column[kMaxBuckets];
  __shared__ int32_t edge[kMaxBuckets + 1];
  const int tid = threadIdx.x, n = edges.n, one = edges.one;
  const int64_t spans = (a.keys + kSpan - 1) / kSpan, bands = (a.queries + a.rows - 1) / a.rows;
  const int64_t b = blockIdx.x, h = b / (spans * bands), rest = b - h * (spans * bands);
  const int64_t i0 = rest / spans * a.rows, j0 = rest % spans * kSpan;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.queries - i0));
  const T* table = static_cast<const T*>(a.table) + h * a.head_stride;
  for (int k = tid; k < n * (a.causal ? 1 : 2); k += kThreads) column[k] = table[k * a.bucket_stride];
  for (int k = tid; k <= n; k += kThreads) edge[k] = edges.edge[k];
  __syncthreads();
  // strip[s]: the value of j - i - first = s + low
  const int64_t low = j0 - (i0 + rows - 1) - a.first;
  const int64_t most = min(static_cast<int64_t>(kSpan), a.keys - j0) + rows - 1;
  for (int s = tid; s < most; s += kThreads) {
    const int64_t rel = low + s;
    if (rel <= 0) {
      strip[s] = column[side_bucket(edge, n, one, -rel)];
    } else {
      strip[s] = a.causal ? minus_infinity<T>() : column[n + side_bucket(edge, n, one, rel)];
    }
  }
  __syncthreads();
  const int64_t j = j0 + tid * V;
  if (j >= a.keys) return;
  const bool whole = j + V <= a.keys;
  T* out = static_cast<T*>(a.out) + (h * a.queries + i0) * a.keys + j;
  int at = tid * V + rows - 1;
  Pack<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = strip[at + e];
  for (int i = 0; i < rows; ++i) {
    if (i) {
      const T next = strip[at];
#pragma unroll
      for (int e = V - 1; e > 0; --e) x.v[e] = x.v[e - 1];
      x.v[0] = next;
    }
    if (whole) {
      store<V>(out, x);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e < a.keys) out[e] = x.v[e];
    }
    out += a.keys;
    --at;
  }
}

struct bias_grad_args {
  const void* grad;
  int64_t batch_stride, head_stride, row_stride;
  int64_t batch, heads, queries, keys, first;
  int64_t spans, bands;
  int32_t rows, causal;
  float* sums;                     // [head][block of the head][bucket]
};

template <typename T>
__global__ __launch_bounds__(kThreads) void k_bias_grad(bias_grad_args a, edges_t edges) {
  constexpr int V = 16 / sizeof(T), kSpan = kThreads * V;
  __shared__ float strip[kSpan];
  const int tid = threadIdx.x, n = edges.n;
  const int64_t each = a.batch * a.bands * a.spans;
  const int64_t h = blockIdx.x / each, of_head = blockIdx.x - h * each;
  const int64_t span = of_head % a.spans, band = of_head / a.spans % a.bands,
                batch = of_head / a.spans / a.bands;
  const int64_t i0 = band * a.rows, i1 = min(i0 + a.rows, a.queries);
  // this thread's diagonals: j - i from d to d + V - 1
  const int64_t d0 = span * kSpan - (i1 - 1), d = d0 + tid * V;
  const T* grad = static_cast<const T*>(a.grad) + batch * a.batch_stride + h * a.head_stride;
  float sum[V] = {};
  // rows where some of them lie within the keys, and where all do
  const int64_t some0 = max(i0, -(d + V - 1)), some1 = min(i1, a.keys - d);
  int64_t all0 = max(i0, -d), all1 = min(i1, a.keys - d - (V - 1));
  if (all1 <= all0) all0 = all1 = some1;
  if (!a.causal || d - a.first <= 0) {
    // towards the diagonal's ends: value by value, from addresses within the row
    auto part = [&](int64_t from, int64_t to) {
      for (int64_t i = from; i < to; ++i) {
        T x[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[e] = grad[i * a.row_stride + min(max(i + d + e, int64_t{0}), a.keys - 1)];
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + d + e >= 0 && i + d + e < a.keys) sum[e] += widen(x[e]);
      }
    };
    part(some0, min(all0, some1));
    const T* p = grad + all0 * (a.row_stride + 1) + d;
    const int64_t step = a.row_stride + 1;
    int64_t i = all0;
    for (; i + 8 <= all1; i += 8, p += 8 * step) {
      Pack<T, V> x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = load_stream_any<V>(p + k * step);
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += widen(x[k].v[e]);
    }
    for (; i < all1; ++i, p += step) {
      const Pack<T, V> x = load_stream_any<V>(p);
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] += widen(x.v[e]);
    }
    part(max(all1, some0), some1);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) strip[tid * V + e] = sum[e];
  __syncthreads();
  // Buckets: each a run of strip[s], j - i - first = s + d0 - first
  const int wave = uniform(tid >> 6), lane = tid & 63, buckets = n * (a.causal ? 1 : 2);
  const int64_t base = d0 - a.first;
  float* out = a.sums + static_cast<int64_t>(blockIdx.x) * buckets;
  for (int b = wave; b < buckets; b += kThreads / 64) {
    const int k = b < n ? b : b - n;
    int64_t from, to;                // distances, both ends within
    if (b < n) {
      from = k + 1 < n ? -static_cast<int64_t>(edges.edge[k + 1] - 1) : INT64_MIN / 2;
      to = -static_cast<int64_t>(edges.edge[k]);
    } else {
      from = max(edges.edge[k], 1);
      to = k + 1 < n ? edges.edge[k + 1] - 1 : INT64_MAX / 2;
    }
    from = max(from - base, int64_t{0});
    to = min(to - base, static_cast<int64_t>(kSpan) - 1);
    float x = 0.0f;
    for (int64_t s = from + lane; s <= to; s += 64) x += strip[s];
#pragma unroll
    for (int m = 32; m; m /= 2) x += __shfl_xor(x, m);
    if (lane == 0) out[b] = x;
  }
}

// The blocks' sums: 16 slices of them for 16 buckets each.
template <typename T>
__global__ __launch_bounds__(256) void k_bias_join(const float* sums, int64_t count, int64_t heads,
                                                   int buckets, T* out) {
  __shared__ float held[16][17];
  const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t h = blockIdx.x / ((buckets + 15) / 16);
  const int b = static_cast<int>(blockIdx.x % ((buckets + 15) / 16)) * 16 + lane;
  float sum = 0.0f;
  if (b < buckets) {
    const float* p = sums + h * count * buckets + b;
#pragma unroll 8
    for (int64_t k = slice; k < count; k += 16) sum += p[k * buckets];
  }
  held[slice][lane] = sum;
  __syncthreads();
  if (slice || b >= buckets) return;
  for (int k = 1; k < 16; ++k) sum += held[k][lane];
  out[b * heads + h] = narrow<T>(sum);
}

// ---------------------------------------------------------------------------
// Host.

int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }

bool good_buckets(int64_t buckets, int64_t max_distance, int32_t causal) {
  const int64_t n = causal ? buckets : buckets / 2;
  return buckets <= kMaxBuckets && n >= 2 && (causal || buckets % 2 == 0) && max_distance > n / 2 &&
         max_distance <= INT32_MAX;
}

// Where buckets begin.  A border that is a whole number is one also after the rounding of
// the power (2^-60 of it; the next whole numbers are 2^-31 away).
edges_t edges_of(int64_t buckets, int64_t max_distance, int32_t causal) {
  edges_t e;
  e.n = static_cast<int32_t>(causal ? buckets : buckets / 2);
  e.one = e.n / 2;
  for (int k = 0; k < e.one; ++k) e.edge[k] = k;
  const int steps = e.n - e.one;
  const long double ratio = static_cast<long double>(max_distance) / e.one;
  for (int s = 0; s < steps; ++s) {
    const long double at = e.one * std::pow(ratio, static_cast<long double>(s) / steps);
    const long double near = std::round(at);
    e.edge[e.one + s] = static_cast<int32_t>(std::fabs(at - near) < 1e-13L * at ? near : std::ceil(at));
  }
  e.edge[e.n] = INT32_MAX;
  return e;
}

bool good_plane(int64_t heads, int64_t queries, int64_t keys, int64_t first) {
  return heads >= 0 && queries >= 0 && keys >= 0 && heads <= INT32_MAX && queries <= INT32_MAX &&
         keys <= INT32_MAX && first >= -(int64_t{1} << 40) && first <= int64_t{1} << 40 &&
         (heads == 0 || queries == 0 || (countable(heads, queries) && countable(heads * queries, keys)));
}

int64_t span_of(int32_t dtype) { return kThreads * (16 / dtype_bytes(dtype)); }

// Rows of a block: many, as its diagonals are worked out once, but so few that there are
// blocks for all CUs.
int32_t rows_of(int64_t queries, int64_t blocks_of_a_row, int64_t least) {
  int32_t rows = kMaxRows;
  while (rows > least && ceil_div(queries, rows) * blocks_of_a_row < 2048) rows /= 2;
  return static_cast<int32_t>(std::min<int64_t>(rows, std::max<int64_t>(queries, 1)));
}

void lay_out(bias_grad_args& a, int32_t dtype) {
  const int64_t span = span_of(dtype);
  a.rows = rows_of(a.queries, a.batch * a.heads * ceil_div(a.keys, span), 16);
  a.bands = ceil_div(a.queries, a.rows);
  a.spans = ceil_div(a.keys + a.rows - 1, span);
}

}  // namespace
}  // namespace ops

extern "C" {

int ms_position_bias(const void* table, int32_t dtype, int64_t buckets, int64_t bucket_stride,
                     int64_t head_stride, int64_t heads, int64_t queries, int64_t keys, int64_t first,
                     int64_t max_distance, int32_t causal, void* out, void* stream) {
  using namespace ops;
  if (!good_dtype(dtype) || !good_buckets(buckets, max_distance, causal) ||
      !good_plane(heads, queries, keys, first))
    return MS_OPS_EINVAL;
  if (heads == 0 || queries == 0 || keys == 0) return MS_OPS_OK;
  if (!table || !out) return MS_OPS_EINVAL;
  bias_args a{table, bucket_stride, head_stride, queries, keys, first, 0, causal ? 1 : 0, out};
  const int64_t spans = ceil_div(keys, span_of(dtype));
  a.rows = rows_of(queries, heads * spans, 4);
  const int64_t blocks = heads * spans * ceil_div(queries, a.rows);
  if (!fits(blocks, kThreads)) return MS_OPS_EINVAL;
  const edges_t e = edges_of(buckets, max_distance, causal);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MS_OPS_F32: return launch(k_bias<float>, blocks, kThreads, s, a, e);
    case MS_OPS_F16: return launch(k_bias<f16>, blocks, kThreads, s, a, e);
    default: return launch(k_bias<bf16>, blocks, kThreads, s, a, e);
  }
}

int64_t ms_position_bias_grad_workspace(int32_t dtype, int64_t buckets, int64_t batch, int64_t heads,
                                        int64_t queries, int64_t keys) {
  using namespace ops;
  if (!good_dtype(dtype) || buckets < 1 || buckets > kMaxBuckets || batch < 0 || batch > INT32_MAX ||
      !good_plane(heads, queries, keys, 0) || !countable(batch, std::max<int64_t>(heads, 1)))
    return MS_OPS_EINVAL;
  if (!batch || !heads || !queries || !keys) return 0;
  bias_grad_args a{};
  a.batch = batch;
  a.heads = heads;
  a.queries = queries;
  a.keys = keys;
  lay_out(a, dtype);
  if (!countable(batch * heads, a.bands) || !countable(batch * heads * a.bands, a.spans * buckets))
    return MS_OPS_EINVAL;
  return batch * heads * a.bands * a.spans * buckets * 4;
}

int ms_position_bias_grad(const void* grad, int32_t dtype, int64_t batch, int64_t batch_stride,
                          int64_t heads, int64_t head_stride, int64_t queries, int64_t row_stride,
                          int64_t keys, int64_t first, int64_t buckets, int64_t max_distance,
                          int32_t causal, void* dtable, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  using namespace ops;
  if (!good_dtype(dtype) || !good_buckets(buckets, max_distance, causal) ||
      !good_plane(heads, queries, keys, first))
    return MS_OPS_EINVAL;
  const int64_t need = ms_position_bias_grad_workspace(dtype, buckets, batch, heads, queries, keys);
  if (need < 0) return MS_OPS_EINVAL;
  if (heads == 0) return MS_OPS_OK;
  if (!dtable || (need && !grad)) return MS_OPS_EINVAL;
  if (workspace_bytes < need || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)))
    return MS_OPS_EWORKSPACE;
  bias_grad_args a{grad, batch_stride, head_stride, row_stride, batch, heads, queries, keys, first,
                   0, 0, 0, causal ? 1 : 0, static_cast<float*>(workspace)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t count = 0;
  if (need) {
    lay_out(a, dtype);
    count = batch * a.bands * a.spans;
    const int64_t blocks = heads * count;
    if (!fits(blocks, kThreads)) return MS_OPS_EINVAL;
    const edges_t e = edges_of(buckets, max_distance, causal);
    int rc;
    switch (dtype) {
      case MS_OPS_F32: rc = launch(k_bias_grad<float>, blocks, kThreads, s, a, e); break;
      case MS_OPS_F16: rc = launch(k_bias_grad<f16>, blocks, kThreads, s, a, e); break;
      default: rc = launch(k_bias_grad<bf16>, blocks, kThreads, s, a, e);
    }
    if (rc) return rc;
  }
  // (without blocks to join, zeros)
  const int64_t blocks = heads * ceil_div(buckets, 16);
  if (!fits(blocks, 256)) return MS_OPS_EINVAL;
  const int nb = static_cast<int>(buckets);
  switch (dtype) {
    case MS_OPS_F32: return launch(k_bias_join<float>, blocks, 256, s, a.sums, count, heads, nb, static_cast<float*>(dtable));
    case MS_OPS_F16: return launch(k_bias_join<f16>, blocks, 256, s, a.sums, count, heads, nb, static_cast<f16*>(dtable));
    default: return launch(k_bias_join<bf16>, blocks, 256, s, a.sums, count, heads, nb, static_cast<bf16*>(dtable));
  }
}

}  // extern "C"
