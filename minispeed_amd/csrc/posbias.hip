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
// down the rows, each time shifting one value in.  Backward, which only reads, the sums of the
// diagonals move through the registers of a wave as the rows go by; a block then adds up its
// diagonals' sums by bucket, each a run of neighbours, and a second kernel joins the
// blocks' sums in their order.
//
// Memory bounds both.  Forward 16 x 2048 x 2048 fp16 23.9 us, 5.6 TB/s (floor at 6.9 TB/s of writes 19.5);
// backward 8 x 12 x 1024 x 1024 bf16 40 us (kernel 36 to 43, the join 4.6; floor at 7.3 TB/s of reads 27.6).
// A thread that follows its diagonals down the rows by loads that move along instead took 59 to
// 69 us: at every wave's edges they run out of the rows.
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
  int64_t chunks, bands, units;    // of a row, of the rows, of a head
  int32_t rows, causal;            // rows: of a band, a multiple of 8
  float* sums;                     // [head][block of the head][bucket]
};

// 16 bytes, taken apart where their values are used.
template <typename T>
struct Words {
  uint32_t w[4];
  __device__ float operator[](int e) const {
    Pack<T, 16 / sizeof(T)> x;
    __builtin_memcpy(&x, w, 16);
    return widen(x.v[e]);
  }
};
template <typename T>
__device__ __forceinline__ Words<T> load_words(const T* p) {
  const Pack<T, 16 / sizeof(T)> x = load_stream_any<16 / sizeof(T)>(p);
  Words<T> r;
  __builtin_memcpy(r.w, &x, 16);
  return r;
}

// A wave goes down a band of rows in a chunk of 64 V columns, a lane with V of them.  Its V sums
// are of diagonals: from row to row each moves one column on, the last one to the next
// lane, and out of lane 63 to LDS.  (The sums move by the names of their registers, but for
// the one that changes lanes.)
template <typename T>
__global__ __launch_bounds__(kThreads) void k_bias_grad(bias_grad_args a, edges_t edges) {
  constexpr int V = 16 / sizeof(T), kWide = 64 * V, kWaves = kThreads / 64;
  __shared__ float strips[kWaves][kWide + kMaxRows];
  __shared__ int32_t edge[kMaxBuckets + 1];
  __shared__ int64_t bases[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), n = edges.n;
  // (under way with the gradient's loads: arguments lie in memory too)
  int32_t held[kMaxBuckets / kThreads + 1];
#pragma unroll
  for (int k = 0; k <= kMaxBuckets / kThreads; ++k)
    held[k] = edges.edge[min(tid + k * kThreads, n)];
  const int64_t blocks = (a.units + kWaves - 1) / kWaves;
  const int64_t h = blockIdx.x / blocks, unit = (blockIdx.x - h * blocks) * kWaves + wave;
  const int64_t chunk = unit % a.chunks, band = unit / a.chunks % a.bands,
                batch = unit / a.chunks / a.bands;
  const int64_t i0 = band * a.rows, c0 = chunk * kWide, c = c0 + lane * V;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.queries - i0));
  const int turns = (rows + 7) / 8 * 8;
  float* strip = strips[wave];
  float sum[V] = {};
  // (a unit behind the last, or one with keys behind all of its queries alone, has no sums)
  const bool some = unit < a.units && !(a.causal && c0 - (i0 + rows - 1) - a.first > 0);
  if (some) {
    const T* row = static_cast<const T*>(a.grad) + batch * a.batch_stride + h * a.head_stride +
                   i0 * a.row_stride;
    // Beyond the last key a lane's 16 bytes run into the next row, and what lies there is
    // masked.  The last row, and rows closer than 16 bytes, are loaded value by value.
    const bool whole = c0 + kWide <= a.keys;
    const T* column = row + min(c, a.keys - 1);
    uint32_t mask[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mask[k] = 0;
#pragma unroll
      for (int e = 0; e < V / 4; ++e)
        if (c + k * (V / 4) + e < a.keys) mask[k] |= (V == 4 ? ~0u : 0xffffu) << (e * 16);
    }
    auto masked = [&](Words<T> x) {
#pragma unroll
      for (int q = 0; q < 4; ++q) x.w[q] &= mask[q];
      return x;
    };
    auto one_by_one = [&](int k) {
      Pack<T, V> values;
#pragma unroll
      for (int e = 0; e < V; ++e) values.v[e] = row[k * a.row_stride + min(c + e, a.keys - 1)];
      Words<T> x;
      __builtin_memcpy(x.w, &values, 16);
      return masked(x);
    };
    // rows that are loaded as vectors
    const int vectors =
        whole ? rows : a.row_stride < V ? 0 : i0 + rows == a.queries ? rows - 1 : rows;
    auto take = [&](const Words<T>& x, int k, int r) {     // r = k % V
#pragma unroll
      for (int e = 0; e < V; ++e) sum[(e - r) & (V - 1)] += x[e];
      float& out = sum[(V - 1 - r) & (V - 1)];
      if (lane == 63) strip[kWide - 1 + turns - k] = out;
      out = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(out), 0x138, 0xf, 0xf, false));
    };
    int k = 0;
    for (; k + 8 <= vectors; k += 8) {
      Words<T> x[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = load_words(column + (k + q) * a.row_stride);
#pragma unroll
      for (int q = 0; q < 8; ++q) take(whole ? x[q] : masked(x[q]), k + q, q & (V - 1));
    }
    // the rows left, and rows of nothing up to a multiple of 8; all sums move
#pragma unroll 1
    for (; k < turns; ++k) {
      Words<T> x = {{0, 0, 0, 0}};
      if (k < vectors) x = masked(load_words(column + k * a.row_stride));
      else if (k < rows) x = one_by_one(k);
      take(x, k, 0);
      const float first = sum[V - 1];
#pragma unroll
      for (int e = V - 1; e > 0; --e) sum[e] = sum[e - 1];
      sum[0] = first;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) strip[lane * V + e] = sum[e];
  }
  // strip[s] is the sum of j - i - first = s + bases[wave]
  if (lane == 0) bases[wave] = c0 - i0 - turns - a.first;
  const int length = some ? kWide + turns : 0;
  __shared__ int lengths[kWaves];
  if (lane == 0) lengths[wave] = length;
#pragma unroll
  for (int k = 0; k <= kMaxBuckets / kThreads; ++k)
    if (tid + k * kThreads <= n) edge[tid + k * kThreads] = held[k];
  __syncthreads();
  // Buckets: each a run of a strip; 16 lanes to one
  const int buckets = n * (a.causal ? 1 : 2);
  float* out = a.sums + static_cast<int64_t>(blockIdx.x) * buckets;
  for (int b = tid >> 4; b < buckets; b += kThreads / 16) {
    const int k = b < n ? b : b - n;
    int64_t from, to;                // distances, both ends within
    if (b < n) {
      from = k + 1 < n ? -static_cast<int64_t>(edge[k + 1] - 1) : INT64_MIN / 2;
      to = -static_cast<int64_t>(edge[k]);
    } else {
      from = max(edge[k], 1);
      to = k + 1 < n ? edge[k + 1] - 1 : INT64_MAX / 2;
    }
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int64_t base = bases[w], long_ = lengths[w];
      const int first = static_cast<int>(min(max(from - base, int64_t{0}), long_));
      const int end = static_cast<int>(min(max(to - base + 1, int64_t{0}), long_));
#pragma unroll 4
      for (int s = first + (tid & 15); s < end; s += 16) x += strips[w][s];
    }
#pragma unroll
    for (int m = 8; m; m /= 2) x += __shfl_xor(x, m);
    if ((tid & 15) == 0) out[b] = x;
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

// Where buckets begin.  A border that is a whole number is taken for one although up to 256
// powers of a rounded root lie behind it (512 2^-64 of it, 3e-17; other borders are 1e-13 from one
// by chance alone).
edges_t edges_of(int64_t buckets, int64_t max_distance, int32_t causal) {
  edges_t e;
  e.n = static_cast<int32_t>(causal ? buckets : buckets / 2);
  e.one = e.n / 2;
  for (int k = 0; k < e.one; ++k) e.edge[k] = k;
  const int steps = e.n - e.one;
  const long double root = std::pow(static_cast<long double>(max_distance) / e.one, 1.0L / steps);
  long double at = e.one;
  for (int s = 0; s < steps; ++s, at *= root) {
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

constexpr int64_t kGradUnits = 12 * 256;   // waves, 12 to a CU

int64_t span_of(int32_t dtype) { return kThreads * (16 / dtype_bytes(dtype)); }

// Rows of a block: many, as its diagonals are worked out once, but so few that there are
// blocks for all CUs.
int32_t rows_of(int64_t queries, int64_t blocks_of_a_row, int64_t least, int64_t blocks) {
  int32_t rows = kMaxRows;
  while (rows > least && ceil_div(queries, rows) * blocks_of_a_row < blocks) rows /= 2;
  return static_cast<int32_t>(std::min<int64_t>(rows, std::max<int64_t>(queries, 1)));
}

void lay_out(bias_grad_args& a, int32_t dtype) {
  a.chunks = ceil_div(a.keys, span_of(dtype) / (kThreads / 64));
  a.rows = (rows_of(a.queries, a.batch * a.heads * a.chunks, 16, kGradUnits) + 7) / 8 * 8;
  a.bands = ceil_div(a.queries, a.rows);
  a.units = a.batch * a.bands * a.chunks;
}

int64_t blocks_of_a_head(const bias_grad_args& a) { return ceil_div(a.units, kThreads / 64); }

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
  a.rows = rows_of(queries, heads * spans, 4, 2048);
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
  if (!countable(heads, blocks_of_a_head(a)) || !countable(heads * blocks_of_a_head(a), buckets))
    return MS_OPS_EINVAL;
  return heads * blocks_of_a_head(a) * buckets * 4;
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
                   0, 0, 0, 0, causal ? 1 : 0, static_cast<float*>(workspace)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t count = 0;
  if (need) {
    lay_out(a, dtype);
    count = blocks_of_a_head(a);
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
