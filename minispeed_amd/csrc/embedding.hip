// embedding.hip — token embedding and its gradient (gfx950).
//
//   out[t, :]    = scale * table[id_t, :]
//   dtable[v, :] = scale * sum_{t: id_t = v} grad[t, :], t rising

#include <algorithm>

#include "ops_common.h"

namespace {

using namespace ops;

// Token t of a list with one of its layouts: kWide 8-byte ids, kPlain
// consecutive ones (`token` without its branches, which would wait for one load
// after the other).
template <bool kWide, bool kPlain>
__device__ __forceinline__ int64_t token_of(const ms_tokens_t& ids, int64_t t) {
  if (!kPlain) return token(ids, t);
  return kWide ? static_cast<const int64_t*>(ids.data)[t]
               : static_cast<int64_t>(static_cast<const int32_t*>(ids.data)[t]);
}

// Where a row's vector of N values from column c on is taken: the last one ends
// with the row and covers again what the one before it has, which then is
// computed twice, the same.  (With a branch for a short last vector every load
// was waited for before the next.)  Columns beyond the row: the last vector.
template <int N>
__device__ __forceinline__ int64_t vector_at(int64_t c, int64_t width) {
  return c + N <= width ? c : width - N;
}

// The output is cut into vectors of 16 bytes, which go to the lanes one after
// the other whatever the width, kLookupEach of them in flight.  Bound by memory:
// 8192 x 2048 fp16 from 50257 rows 9.3 us, 33.5 MB written at 3.6 TB/s beside the
// rows read, most of them more than once and from the caches.
constexpr int kLookupThreads = 256, kLookupEach = 4;

// kShort: rows of less than a vector, value by value.
template <typename T, bool kWide, bool kPlain, bool kShort>
__global__ void __launch_bounds__(kLookupThreads)
    k_lookup(ms_tokens_t ids, ms_rows_t table, float scale, uint32_t vectors,
             T* __restrict__ out) {
  constexpr int N = kShort ? 1 : 16 / sizeof(T);
  const T* rows = static_cast<const T*>(table.data);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kLookupThreads * kLookupEach);
  const int64_t t0 = item / vectors;
  const uint32_t v0 = static_cast<uint32_t>(item - t0 * vectors) + threadIdx.x;
  int64_t t[kLookupEach], id[kLookupEach];
  uint32_t v[kLookupEach];
#pragma unroll
  for (int k = 0; k < kLookupEach; ++k) {
    const uint32_t i = v0 + k * kLookupThreads, down = i / vectors;
    v[k] = i - down * vectors;
    t[k] = t0 + down;
    id[k] = token_of<kWide, kPlain>(ids, t[k] < ids.n ? t[k] : ids.n - 1);
  }
  Pack<T, N> x[kLookupEach];
#pragma unroll
  for (int k = 0; k < kLookupEach; ++k) {
    const bool good = static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(table.n);
    const T* row = rows + (good ? id[k] : 0) * table.inner_stride;
    x[k] = load<N>(row + vector_at<N>(static_cast<int64_t>(v[k]) * N, table.width));
  }
#pragma unroll
  for (int k = 0; k < kLookupEach; ++k) {
    if (t[k] >= ids.n) continue;
    const bool good = static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(table.n);
    Pack<T, N> y;
#pragma unroll
    for (int j = 0; j < N; ++j)
      y.v[j] = narrow<T>(good ? widen(x[k].v[j]) * scale : quiet_nan());
    store<N>(out + t[k] * table.width +
                 vector_at<N>(static_cast<int64_t>(v[k]) * N, table.width), y);
  }
}

template <typename T>
int lookup_as(const ms_tokens_t& ids, const ms_rows_t& table, float scale, void* out,
              hipStream_t s) {
  const bool brief = table.width < static_cast<int64_t>(16 / sizeof(T));
  const int64_t n = brief ? 1 : 16 / sizeof(T);
  const int64_t vectors = (table.width + n - 1) / n, each = kLookupThreads * kLookupEach;
  if (vectors > INT32_MAX) return MS_OPS_EINVAL;
  const int64_t blocks = (ids.n * vectors + each - 1) / each;
  if (!fits(blocks, kLookupThreads)) return MS_OPS_EINVAL;
  const bool plain = ids.inner >= ids.n && ids.inner_stride == 1;
#define LOOKUP(W, P) (brief ? k_lookup<T, W, P, true> : k_lookup<T, W, P, false>)
  return launch(ids.wide ? plain ? LOOKUP(true, true) : LOOKUP(true, false)
                : plain  ? LOOKUP(false, true)
                         : LOOKUP(false, false),
                blocks, kLookupThreads, s, ids, table, scale, static_cast<uint32_t>(vectors),
                static_cast<T*>(out));
#undef LOOKUP
}

// The gradient's table.  Tokens are sorted by (id, t) on the device, then each
// id's rows are added in that order; no atomics touch a sum.
//
// Few tokens and a small table, one launch (k_grad_small): every block sorts
// all tokens for a few rows of the table in LDS, adds and clears them.
//
// Otherwise three:
//   k_sort_tokens  a bucket of ids to a block, which goes through all tokens:
//                  its ids' positions end up grouped by id and rising.  Other
//                  blocks of the launch clear the first rows of the table.
//                  Buckets take every 2^k-th id: the frequent tokens of a
//                  vocabulary often have neighbouring numbers, and one block
//                  with most of the tokens took 75 us where 13 are usual.
//   k_sum_spans    kSpan sorted positions to a wave and a slice of the width.
//                  Ids of up to kLight tokens belong to the span they begin in;
//                  of longer ones every span adds its piece, left as a partial
//                  sum, so that an id with half of the tokens costs what others
//                  cost.  Other blocks clear the remaining rows without tokens.
//   k_join_spans   adds up the partial sums.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRows = 1024;

struct Sorted {
  int32_t* start;       // [buckets * rows + 1]: where each id's tokens begin, by slot
  int32_t* id;          // [n]
  int32_t* position;    // [n]
  float* partial;       // [spans, 2, width]
  int32_t rows;         // ids to a bucket
  int32_t shift;        // 2^shift buckets
  int64_t slots;        // buckets * rows

  // ids in their sorted order
  __device__ __forceinline__ int64_t slot(int64_t id) const {
    return (id & ((1ll << shift) - 1)) * rows + (id >> shift);
  }
};

// A bucket, every 2^shift-th row of the table.  What is no row at all is 2^32 - 1;
// its top bit keeps it out of every bucket.
struct Bucket {
  uint32_t bucket, shift, vocab;

  __device__ __forceinline__ uint32_t key(uint32_t id) const {
    return id & ((1u << shift) - 1 | 0x80000000u);
  }
  __device__ __forceinline__ uint32_t row(uint32_t id) const { return id >> shift; }
};

__device__ __forceinline__ int wave_scan(int x) {
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) {
    const int y = __shfl_up(x, k);
    if ((threadIdx.x & 63) >= k) x += y;
  }
  return x;
}

// The tokens of a bucket of `rows` rows, stably sorted by a block of
// kSortThreads: wave w counts and then places the w-th part of the list.
// begin(r, p): row r's tokens begin at p of the whole sorted list (r = rows:
// they end there); place(p, r, t): token t of row r belongs at p.
// kWide: 8-byte ids.  kPlain: consecutive ids (`token` without its branches, so
// that a group's loads stay in flight together).  A block goes through all
// tokens, on one CU: what this costs is its instructions per token, so ids are
// compared as 32-bit words.
template <int kRows, int kSteps, bool kWide, bool kPlain, typename Begin, typename Place>
__device__ __forceinline__ void sort_bucket(const ms_tokens_t& ids, const Bucket bucket, int rows,
                                            int64_t skip, int (&count)[kSortWaves][kRows],
                                            int (&wave_sum)[kSortWaves], Begin begin,
                                            Place place) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = static_cast<int>(ids.n);
  const int part = ((n + kSortThreads - 1) / kSortThreads) * kWave;
  const int first = wave * part < n ? wave * part : n;
  const int last = n - first < part ? n : first + part;
  const uint32_t none = static_cast<uint32_t>(skip);

  // as an unsigned word, 2^32 - 1 for what is no row of any table
  auto one = [&](int t) -> uint32_t {
    if (kPlain && kWide) {
      const uint2 word = static_cast<const uint2*>(ids.data)[t];
      return word.y ? ~0u : word.x;
    }
    if (kPlain) return static_cast<const uint32_t*>(ids.data)[t];
    const int64_t x = token(ids, t);
    return static_cast<uint64_t>(x) >> 31 ? ~0u : static_cast<uint32_t>(x);
  };
  auto load_ids = [&](int t0, uint32_t (&id)[kSteps]) {
    if (last - t0 >= kSteps * kWave) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) id[k] = one(t0 + lane + k * kWave);
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int t = t0 + lane + k * kWave;
        id[k] = one(t < last ? t : last - 1);
        if (t >= last) id[k] = ~0u;
      }
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
      if (id[k] >= bucket.vocab) id[k] = ~0u;
    if (none != ~0u) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        if (id[k] == none) id[k] = ~0u;
    }
  };
  uint32_t id[kSteps];
  if (first < last) load_ids(first, id);
  for (int i = threadIdx.x; i < kSortWaves * rows; i += kSortThreads)
    count[i / rows][i % rows] = 0;
  __syncthreads();

  int below = 0;
  for (int t0 = first; t0 < last; t0 += kWave * kSteps) {
    if (t0 != first) load_ids(t0, id);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const uint32_t key = bucket.key(id[k]);
      below += key < bucket.bucket;
      // most often none, one or many of one id (padding): one addition for the first
      // id, which 64 to one address would serialise, and the rest by themselves
      const uint64_t mine = __ballot(key == bucket.bucket);
      if (!mine) continue;
      const int lead = __ffsll(static_cast<unsigned long long>(mine)) - 1;
      const uint32_t one = read_lane(static_cast<int>(id[k]), lead);
      const uint64_t same = __ballot(id[k] == one);
      if (lane == lead) count[wave][bucket.row(one)] += __popcll(same);
      if (key == bucket.bucket && id[k] != one) atomicAdd(&count[wave][bucket.row(id[k])], 1);
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
  int mine = 0, by_wave[kSortWaves];
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    by_wave[w] = r < rows ? count[w][r] : 0;
    mine += by_wave[w];
  }
  const int upto = wave_scan(mine);
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int at = base + upto - mine;
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
  if (r < rows) {
    begin(r, at);
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      count[w][r] = at;
      at += by_wave[w];
    }
    if (r == rows - 1) begin(rows, at);
  }
  __syncthreads();

  for (int t0 = first; t0 < last; t0 += kWave * kSteps) {
    if (part > kWave * kSteps) load_ids(t0, id);      // else they are still here
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      uint64_t left = __ballot(bucket.key(id[k]) == bucket.bucket);
      if (!left) continue;
      const uint32_t row = left >> (threadIdx.x & 63) & 1 ? bucket.row(id[k]) : ~0u;
      while (left) {                               // once per different id
        const int lead = __ffsll(static_cast<unsigned long long>(left)) - 1;
        const uint32_t which = read_lane(static_cast<int>(row), lead);
        const uint64_t same = __ballot(row == which);
        const int to = count[wave][which];
        if (row == which)
          place(to + __popcll(same & ((1ull << lane) - 1)), static_cast<int>(which),
                t0 + k * kWave + lane);
        if (lane == lead) count[wave][which] = to + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// kSteps: groups of 64 tokens in flight per wave.  No more than there are, as all are gone
// through: 4096 tokens (three launches) 23 us with 4 or 8, 27 with 16.
template <int kSteps, bool kWide, bool kPlain>
__global__ void __launch_bounds__(kSortThreads)
    k_sort_tokens(ms_tokens_t ids, int64_t vocab, int64_t skip, int buckets, Sorted out,
                  uint4* table, int64_t clear_bytes) {
  __shared__ int count[kSortWaves][kSortRows];
  __shared__ int wave_sum[kSortWaves];
  if (blockIdx.x >= static_cast<unsigned>(buckets)) {
    const int64_t step = static_cast<int64_t>(gridDim.x - buckets) * kSortThreads;
    int64_t i = static_cast<int64_t>(blockIdx.x - buckets) * kSortThreads + threadIdx.x;
    const int64_t vectors = clear_bytes / 16, rest = (clear_bytes & 15) / 2;
    if (i < rest) reinterpret_cast<uint16_t*>(table + vectors)[i] = 0;
    for (; i < vectors; i += step) table[i] = uint4{0, 0, 0, 0};
    return;
  }
  const uint32_t b = blockIdx.x;
  const Bucket bucket = {b, static_cast<uint32_t>(out.shift), static_cast<uint32_t>(vocab)};
  const int64_t slot = static_cast<int64_t>(b) * out.rows;
  sort_bucket<kSortRows, kSteps, kWide, kPlain>(
      ids, bucket, out.rows, skip, count, wave_sum,
      [&](int r, int p) {
        if (r < out.rows || b == static_cast<uint32_t>(buckets) - 1) out.start[slot + r] = p;
      },
      [&](int p, int r, int t) {
        out.id[p] = static_cast<int32_t>(static_cast<uint32_t>(r) << out.shift | b);
        out.position[p] = t;
      });
}

constexpr int kSumThreads = 256, kSumWaves = kSumThreads / kWave;
constexpr int kSpan = 16;                 // sorted positions to a block
constexpr int kSumDepth = 8;              // rows in flight per wave
// An id of up to kLight tokens is added by one wave.  A wave looks at 64
// positions from kLead before its span on, which is enough to tell for every
// id in the span whether it has more.
constexpr int kLight = 20, kLead = 24;
static_assert(kLead >= kLight && kLead + kSpan + kLight <= 63, "");
constexpr int kClearRows = 32, kClearBytes = 16384;     // of the table per clearing block

// fp32 sums of N columns in each of G chunks of kWave * N, from column c on.
template <typename T, int N, int G>
struct Tile {
  float sum[G][N];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int k = 0; k < N; ++k) sum[j][k] = 0.f;
  }
  // rows q0 .. q1 - 1, at most kSumDepth of them; row(q): its first element
  template <typename Row>
  __device__ __forceinline__ void add(int q0, int q1, int64_t c, int64_t width, Row row) {
    // as words until all are on their way: taken apart into values beside each
    // load, every one was waited for before the next
    typedef typename raw_of<N * sizeof(T)>::type raw;
    raw x[kSumDepth][G];
#pragma unroll
    for (int u = 0; u < kSumDepth; ++u)
      if (q0 + u < q1) {
        const T* src = row(q0 + u);
#pragma unroll
        for (int j = 0; j < G; ++j)
          x[u][j] = *reinterpret_cast<const raw*>(src + vector_at<N>(c + j * kWave * N, width));
      }
#pragma unroll
    for (int u = 0; u < kSumDepth; ++u)
      if (q0 + u < q1)
#pragma unroll
        for (int j = 0; j < G; ++j) {
          Pack<T, N> y;
          __builtin_memcpy(&y, &x[u][j], sizeof(y));
#pragma unroll
          for (int k = 0; k < N; ++k) sum[j][k] += widen(y.v[k]);
        }
  }
  __device__ __forceinline__ void write(T* row, int64_t c, int64_t width, float scale) const {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int64_t at = c + j * kWave * N;
      Pack<T, N> y;
#pragma unroll
      for (int k = 0; k < N; ++k) y.v[k] = narrow<T>(sum[j][k] * scale);
      if (at < width) store<N>(row + vector_at<N>(at, width), y);
    }
  }
  __device__ __forceinline__ void leave(float* row, int64_t c, int64_t width) const {
    constexpr int kVec = N < 4 ? N : 4;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int64_t at = c + j * kWave * N;
      if (at >= width) continue;
#pragma unroll
      for (int k0 = 0; k0 < N; k0 += kVec) {
        Pack<float, kVec> y;
#pragma unroll
        for (int k = 0; k < kVec; ++k) y.v[k] = sum[j][k0 + k];
        store<kVec>(row + vector_at<N>(at, width) + k0, y);
      }
    }
  }
};

// Zeros for `rows` rows of which bit r of `empty` is set, row(r) the r-th: the
// block's threads take consecutive vectors.
template <typename T, typename Row>
__device__ __forceinline__ void clear_rows_of(uint64_t empty, int rows, int64_t width, Row row) {
  constexpr int kVec = 16 / sizeof(T);
  if (width < kVec) {
    for (int64_t i = threadIdx.x; i < width * rows; i += blockDim.x)
      if (empty >> (i / width) & 1)
        row(static_cast<int>(i / width))[i % width] = static_cast<T>(0.f);
    return;
  }
  Pack<T, kVec> zero;
#pragma unroll
  for (int k = 0; k < kVec; ++k) zero.v[k] = static_cast<T>(0.f);
  const uint32_t vectors = static_cast<uint32_t>((width + kVec - 1) / kVec);
  for (uint32_t v = threadIdx.x; v < vectors * rows; v += blockDim.x) {
    const uint32_t r = rows == 1 ? 0 : v / vectors;
    if (empty >> r & 1)
      store<kVec>(row(static_cast<int>(r)) +
                      vector_at<kVec>(static_cast<int64_t>(v - r * vectors) * kVec, width), zero);
  }
}

// Block `block` of those that clear: `each` rows from `from` on, below `until`,
// those that have no tokens.
template <typename T>
__device__ __forceinline__ void clear_absent(const Sorted& in, int64_t block, int64_t from,
                                             int64_t until, int each, int64_t width, T* table) {
  const int lane = threadIdx.x & 63;
  const int64_t r0 = from + block * each;
  const int rows = static_cast<int>(until - r0 < each ? until - r0 : each);
  const int64_t slot = in.slot(r0 + (lane < rows ? lane : rows - 1));
  const uint64_t empty = __ballot(lane < rows && in.start[slot] == in.start[slot + 1]);
  clear_rows_of<T>(empty, rows, width, [&](int k) { return table + (r0 + k) * width; });
}

// What is left to clear: rows [from, until), `each` to a block, in the blocks from
// `first_block` on.
struct Clear {
  int64_t from, until;
  int each;
  unsigned first_block;
};

// Blocks below clear.first_block: a span and kWave * N * G columns; wave w adds the
// span's w-th, (w + kSumWaves)-th .. run of equal ids.  16384 x 768 bf16 into 12000 rows,
// uniform ids or falling off as 1 / rank: 11.1 and 10.8 us (39 and 32 MB moved), 15.5
// and 16.1 before the rows were loaded as words.  A wave to a span that keeps its
// 16 rows in registers, the loop over them unrolled: 16.5 and more; the rows
// set down in LDS for a short loop: 17.3 and 23.
template <typename T, int N, int G>
__global__ void __launch_bounds__(kSumThreads)
    k_sum_spans(ms_rows_t grad, float scale, int slices, Clear clear, Sorted in,
                T* __restrict__ table) {
  const int lane = threadIdx.x & 63;
  const int64_t width = grad.width;
  if (blockIdx.x >= clear.first_block) {
    clear_absent(in, blockIdx.x - clear.first_block, clear.from, clear.until, clear.each, width,
                 table);
    return;
  }
  const int64_t s = blockIdx.x / slices, first = s * kSpan;
  const int64_t c =
      static_cast<int64_t>(blockIdx.x - s * slices) * (kWave * N * G) + lane * N;
  // lane q has position first - kLead + q of the sorted list.  The lists beyond
  // `total` hold nothing; they are read with it, not after it.
  const int64_t at = first + lane - kLead;
  const int64_t in_list = at < 0 ? 0 : at < grad.n ? at : grad.n - 1;
  const int total = in.start[in.slots];
  int id = in.id[in_list];
  int position = in.position[in_list];
  if (first >= total) return;
  if (at < 0 || at >= total) id = -1, position = 0;
  const int64_t offset = row_start(grad, position);
  const int next = __shfl_down(id, 1);
  // bit q: lane q's id ends there (lane 63: not known, and not needed)
  const uint64_t ends = __ballot(lane < 63 && next != id);
  const int n = static_cast<int>(total - first < kSpan ? total - first : kSpan);
  const int last = kLead + n - 1;
  const T* g = static_cast<const T*>(grad.data);
  int run = 0;
  for (int from = kLead; from <= last; ++run) {
    // the run of equal ids that position `from` is in: all of it is
    // [begin, end], begin -1: before lane 0, end 64: behind lane 62
    const uint64_t before = ends & ((1ull << from) - 1), behind = ends >> from;
    const int begin = before ? 64 - __clzll(before) : -1;
    const int end = behind ? from + __ffsll(static_cast<unsigned long long>(behind)) - 1 : 64;
    const bool light = begin >= 0 && end < 64 && end - begin < kLight;
    const int to = light || end <= last ? end : last;
    const bool mine = (run & (kSumWaves - 1)) == static_cast<int>(threadIdx.x >> 6) &&
                      !(light && begin < kLead);          // else an earlier span's
    if (mine) {
      Tile<T, N, G> tile;
      tile.clear();
      for (int q = from; q <= to; q += kSumDepth)
        tile.add(q, to + 1, c, width, [&](int i) { return g + read_lane(offset, i); });
      if (light)
        tile.write(table + read_lane(id, from) * width, c, width, scale);
      else
        tile.leave(in.partial + (s * 2 + (begin >= kLead)) * width, c, width);
    }
    from = to + 1;
  }
}

constexpr int kJoinThreads = 1024, kJoinWaves = kJoinThreads / kWave;
constexpr int kJoinFew = 16;              // partial sums that one wave adds by itself
constexpr int kJoinDepth = 8;             // partial sums in flight per wave

// Every block looks at all spans, kJoinThreads at a time, for those that an id
// of many tokens begins in.  Such a span and a slice of the width make a job:
// a wave's (N columns to a lane) where there are few partial sums, the block's
// (1 column to a lane) where there are many; then its waves take a part of them
// each and are added in their order.  Jobs go round the waves and blocks.
template <typename T, int N>
__global__ void __launch_bounds__(kJoinThreads)
    k_join_spans(int64_t n, int64_t width, float scale, Clear clear, Sorted in,
                 T* __restrict__ table) {
  if (blockIdx.x >= clear.first_block) {
    clear_absent(in, blockIdx.x - clear.first_block, clear.from, clear.until, clear.each, width,
                 table);
    return;
  }
  struct Found {
    int span, id, parts;
  };
  __shared__ Found found[2][kJoinThreads];
  __shared__ int found_by[2][kJoinWaves];
  __shared__ float part[kJoinWaves][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned blocks = clear.first_block;
  const int total = in.start[in.slots];
  // partial sums [from, to) of the id that begins in span s
  auto add_parts = [&](auto& sum, int64_t s, int from, int to, int64_t c) {
    constexpr int M = sizeof(sum) / sizeof(float);
    for (int k0 = from; k0 < to; k0 += kJoinDepth) {
      Pack<float, M> x[kJoinDepth];
#pragma unroll
      for (int u = 0; u < kJoinDepth; ++u) {
        const int k = k0 + u < to ? k0 + u : to - 1;
        x[u] = load<M>(in.partial + ((s + k) * 2 + (k == 0)) * width + vector_at<M>(c, width));
      }
#pragma unroll
      for (int u = 0; u < kJoinDepth; ++u)
        if (k0 + u < to)
#pragma unroll
          for (int k = 0; k < M; ++k) sum[k] += x[u].v[k];
    }
  };
  for (int64_t s0 = 0; (s0 + 1) * kSpan < n; s0 += kJoinThreads) {
    const int64_t end = (s0 + threadIdx.x + 1) * kSpan, at = end < n ? end : n - 1;
    const int a = in.id[at - 1], b = in.id[at];               // n > kSpan here
    int kind = -1, parts = 0;
    if (end < total && a == b) {
      const int64_t slot = in.slot(a);
      const int from = in.start[slot], to = in.start[slot + 1];
      parts = (to - 1) / kSpan - static_cast<int>(end / kSpan - 1) + 1;
      if (from >= end - kSpan && to - from > kLight) kind = parts > kJoinFew;
    }
    __syncthreads();
    for (int u = 0; u < 2; ++u) {
      const uint64_t hits = __ballot(kind == u);
      if (lane == 0) found_by[u][wave] = __popcll(hits);
    }
    __syncthreads();
    int all[2] = {0, 0};
    for (int u = 0; u < 2; ++u) {
      const uint64_t hits = __ballot(kind == u);
      int to = __popcll(hits & ((1ull << lane) - 1));
      for (int w = 0; w < kJoinWaves; ++w) {
        if (w < wave) to += found_by[u][w];
        all[u] += found_by[u][w];
      }
      if (kind == u) found[u][to] = Found{static_cast<int>(s0 + threadIdx.x), a, parts};
    }
    __syncthreads();

    const int64_t lots = (width + kWave - 1) / kWave;
    for (int64_t j = blockIdx.x; j < all[1] * lots; j += blocks) {
      const Found f = found[1][j / lots];
      const int64_t s = f.span, id = f.id, c = (j % lots) * kWave + lane;
      const int each = (f.parts + kJoinWaves - 1) / kJoinWaves;
      const int from = wave * each, to = from + each < f.parts ? from + each : f.parts;
      float sum[1] = {0.f};
      add_parts(sum, s, from, to, c);
      part[wave][lane] = sum[0];
      __syncthreads();
      if (wave == 0 && c < width) {
        for (int w = 1; w < kJoinWaves; ++w) sum[0] += part[w][lane];
        table[id * width + c] = narrow<T>(sum[0] * scale);
      }
      __syncthreads();
    }
    // from the last block on, which has the fewest of the others
    const int64_t few = (width + N * kWave - 1) / (N * kWave);
    const int64_t waves = static_cast<int64_t>(blocks) * kJoinWaves;
    for (int64_t j = static_cast<int64_t>(wave) * blocks + blocks - 1 - blockIdx.x;
         j < all[0] * few; j += waves) {
      const Found f = found[0][j / few];
      const int64_t s = f.span, id = f.id, c = (j % few) * (N * kWave) + lane * N;
      float sum[N] = {};
      add_parts(sum, s, 0, f.parts, c);
      Pack<T, N> y;
#pragma unroll
      for (int k = 0; k < N; ++k) y.v[k] = narrow<T>(sum[k] * scale);
      if (c < width) store<N>(table + id * width + vector_at<N>(c, width), y);
    }
  }
}

// Few tokens: every block sorts all of them for its rows of the table, in LDS, and
// makes those rows' columns from part * columns on, the last part all that are left.  A wave
// takes a row with tokens and a slice of the columns at a time; the tokens of rows with more
// than kLight are cut into `pieces`, as many in every block, whose sums are added in their order.
constexpr int kSmallTokens = 1024, kSmallRows = 64, kSmallParts = 8;
constexpr int64_t kSmallBlocks = 256, kSmallBytes = 262144;

template <typename T, int N, bool kWide, bool kPlain>
__global__ void __launch_bounds__(kSortThreads)
    k_grad_small(ms_tokens_t ids, ms_rows_t grad, int64_t vocab, int64_t skip, float scale,
                 int shift, int column_parts, int columns, int pieces, T* __restrict__ table) {
  __shared__ int count[kSortWaves][kSmallRows];
  __shared__ int wave_sum[kSortWaves];
  __shared__ int start[kSmallRows + 1];
  __shared__ uint16_t position[kSmallTokens];
  __shared__ float part[kSortWaves][kWave * N];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const uint32_t b = blockIdx.x / column_parts;
  const int column_part = static_cast<int>(blockIdx.x - b * column_parts);
  const int64_t column = static_cast<int64_t>(column_part) * columns;
  // from here on a row is its columns of this block, N or more
  const int64_t width = column_part == column_parts - 1 ? grad.width - column : columns;
  const int rows = static_cast<int>((vocab - 1 - b) >> shift) + 1;      // b < vocab
  auto table_row = [&](int r) {
    return table + ((static_cast<int64_t>(r) << shift) + b) * grad.width + column;
  };
  sort_bucket<kSmallRows, kSmallTokens / kSortThreads, kWide, kPlain>(
      ids, Bucket{b, static_cast<uint32_t>(shift), static_cast<uint32_t>(vocab)}, rows, skip,
      count, wave_sum, [&](int r, int p) { start[r] = p; },
      [&](int p, int, int t) { position[p] = static_cast<uint16_t>(t); });
  __syncthreads();

  const T* g = static_cast<const T*>(grad.data) + column;
  // the sum of the sorted tokens [from, to), 64 positions looked up at a time
  auto add_rows = [&](int from, int to, int64_t c, float (&sum)[N]) {
    Tile<T, N, 1> tile;
    tile.clear();
    for (int p0 = from; p0 < to; p0 += kWave) {
      const int64_t offset = row_start(grad, position[p0 + lane < to ? p0 + lane : to - 1]);
      const int n = to - p0 < kWave ? to - p0 : kWave;
      for (int q = 0; q < n; q += kSumDepth)
        tile.add(q, n, c, width, [&](int i) { return g + read_lane(offset, i); });
    }
#pragma unroll
    for (int k = 0; k < N; ++k) sum[k] = tile.sum[0][k];
  };
  const int slices = static_cast<int>((width + kWave * N - 1) / (kWave * N));
  // the same in every wave: bit r for row r
  const int row_at = lane < rows ? lane : rows - 1;
  const int tokens = start[row_at + 1] - start[row_at];
  const uint64_t empty = __ballot(lane < rows && tokens == 0);
  const uint64_t heavy = __ballot(lane < rows && tokens > kLight);
  uint64_t some = __ballot(lane < rows && tokens > 0) & ~heavy;

  if (empty) clear_rows_of<T>(empty, rows, width, table_row);
  for (int item = wave; some; item -= slices, some &= some - 1) {
    const int r = __ffsll(static_cast<unsigned long long>(some)) - 1;
    const int from = uniform(start[r]), to = uniform(start[r + 1]);
    for (; item < slices; item += kSortWaves) {
      const int64_t c = (static_cast<int64_t>(item) * kWave + lane) * N;
      float sum[N];
      add_rows(from, to, c, sum);
      Pack<T, N> y;
#pragma unroll
      for (int k = 0; k < N; ++k) y.v[k] = narrow<T>(sum[k] * scale);
      if (c < width) store<N>(table_row(r) + vector_at<N>(c, width), y);
    }
  }
  // the waves share a row's slices and, where these are few, its tokens
  const int jobs = slices * pieces;                  // no more than `part` has, unless pieces is 1
  for (uint64_t left = heavy; left; left &= left - 1) {
    const int r = __ffsll(static_cast<unsigned long long>(left)) - 1;
    const int from = uniform(start[r]), end = uniform(start[r + 1]);
    const int each = (end - from + pieces - 1) / pieces;
    for (int j = wave; j < jobs; j += kSortWaves) {
      const int slice = j / pieces, first = from + (j - slice * pieces) * each;
      const int64_t c = (static_cast<int64_t>(slice) * kWave + lane) * N;
      float sum[N];
      add_rows(first, first + each < end ? first + each : end, c, sum);
      if (pieces == 1) {
        Pack<T, N> y;
#pragma unroll
        for (int k = 0; k < N; ++k) y.v[k] = narrow<T>(sum[k] * scale);
        if (c < width) store<N>(table_row(r) + vector_at<N>(c, width), y);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) part[j][lane * N + k] = sum[k];
      }
    }
    if (pieces == 1) continue;
    __syncthreads();
    for (int k = threadIdx.x; k < slices * kWave * N; k += kSortThreads) {
      const int slice = k / (kWave * N), at = k % (kWave * N);
      const int64_t c = k / N * N;                   // of the lane; its vector may be earlier
      if (c >= width) continue;
      float y = part[slice * pieces][at];
      for (int p = 1; p < pieces; ++p) y += part[slice * pieces + p][at];
      table_row(r)[vector_at<N>(c, width) + k % N] = narrow<T>(y * scale);
    }
    __syncthreads();
  }
}

int64_t align16(int64_t bytes) { return (bytes + 15) & ~15ll; }

// How the work is cut; a function of the sizes alone, as the order of the sums
// follows from it.
struct GradShape {
  int shift, rows;
  int64_t spans, start_bytes, list_bytes, partial_bytes;
};

GradShape shape_of(int64_t n, int64_t vocab, int64_t width) {
  GradShape g;
  // 256 buckets, a CU each: as many as go round beside each other, few ids to
  // each.  Small vocabularies: 8 ids; large ones: what fits the LDS.
  g.shift = 0;
  while (g.shift < 8 ? vocab >> g.shift > 8 : vocab > static_cast<int64_t>(kSortRows) << g.shift)
    ++g.shift;
  g.rows = static_cast<int>(((vocab - 1) >> g.shift) + 1);
  g.spans = (n + kSpan - 1) / kSpan;
  g.start_bytes = align16(((static_cast<int64_t>(g.rows) << g.shift) + 1) * 4);
  g.list_bytes = align16(n * 4);
  g.partial_bytes = align16(g.spans * 2 * width * 4);
  return g;
}

// What the sort's launch clears while it sorts, which takes it some 12 us.
constexpr int64_t kClearBesideSort = 40 << 20;

// Blocks that clear rows [from, until) behind `first` others; blocks: of the launch.
Clear clear_after(int64_t first, int64_t from, int64_t until, int64_t row_bytes, int64_t bytes,
                  int64_t& blocks) {
  Clear c;
  c.from = from;
  c.until = until;
  c.each = static_cast<int>(std::min<int64_t>(kClearRows, std::max<int64_t>(bytes / row_bytes, 1)));
  c.first_block = static_cast<unsigned>(first);
  blocks = first + (until - from + c.each - 1) / c.each;
  return c;
}

// Positions past the end of the list are 32-bit too.
constexpr int64_t kMostTokens = 1 << 30;

// One launch where three would mostly wait for each other: up to kSmallTokens
// tokens and kSmallTable bytes of table.  Ids that fall off as 1 / rank, and with 33% and
// 90% of them one id, bf16, in three launches in brackets: 12000 x 768, 316 tokens 9, 11
// and 15 us (16), 1024 tokens 11, 16 and 29 (17); 50257 x 768, 19, 20 and 19 (20 to 22), 20,
// 20 and 33 (22); 100000 x 1024, 41, 43 and 49 (37), 43, 52 and 68 (37).
constexpr int64_t kSmallTable = 96 << 20;

bool is_small(int64_t n, int64_t table_bytes) {
  return n <= kSmallTokens && table_bytes <= kSmallTable;
}

template <typename T, int N>
int small_as(const ms_tokens_t& ids, const ms_rows_t& grad, int64_t vocab, float scale,
             int64_t skip, T* table, hipStream_t s) {
  // A block for each CU at least, and no more than some 256 KB of the table to one
  // (50257 x 768 bf16 18 us, 24 with 64 KB).  Where the table is small, several take the
  // columns of its rows, or one had all tokens of a frequent id: 316 and 1024 tokens
  // of 1588 x 1344 bf16, 90% one id, 10.9 and 16.5 us, 19.8 and 46.9 without.
  const int64_t slices = (grad.width + kWave * N - 1) / (kWave * N);
  int64_t most_parts = kSmallParts;
  while (most_parts > 1 && vocab * most_parts > kSmallBlocks * kSmallRows) most_parts /= 2;
  const int64_t each = (slices + most_parts - 1) / most_parts;
  const int64_t columns = each * kWave * N;
  int parts = static_cast<int>((slices + each - 1) / each);
  // no part of less than a vector: that would begin in the one before
  if (parts > 1 && grad.width - (parts - 1) * columns < N) --parts;
  const int64_t widest = std::max(std::min(columns, grad.width), grad.width - (parts - 1) * columns);
  const int most_slices = static_cast<int>(
      std::min<int64_t>((widest + kWave * N - 1) / (kWave * N), kSortWaves));
  const int pieces = kSortWaves / most_slices;
  const int64_t bytes = widest * static_cast<int64_t>(sizeof(T));
  const int64_t most = std::min<int64_t>(kSmallRows, std::max<int64_t>(kSmallBytes / bytes, 1));
  int shift = 0;
  while (((parts << shift) < 256 && 1 << shift < vocab) || vocab > most << shift) ++shift;
  const int64_t blocks = std::min<int64_t>(vocab, 1ll << shift) * parts;
  const bool plain = ids.inner >= ids.n && ids.inner_stride == 1;
  return launch(ids.wide ? plain ? k_grad_small<T, N, true, true> : k_grad_small<T, N, true, false>
                : plain  ? k_grad_small<T, N, false, true>
                         : k_grad_small<T, N, false, false>,
                blocks, kSortThreads, s, ids, grad, vocab, skip, scale, shift, parts,
                static_cast<int>(columns), pieces, table);
}

template <typename T>
int grad_as(const ms_tokens_t& ids, const ms_rows_t& grad, int64_t vocab, float scale,
            int64_t skip, void* dtable, void* workspace, hipStream_t s) {
  const int64_t width = grad.width;
  const int64_t row_bytes = width * static_cast<int64_t>(sizeof(T));
  T* table = static_cast<T*>(dtable);
  if (skip < 0 || skip >= vocab) skip = -1;                // no row: compared as 32-bit words
  if (is_small(ids.n, vocab * row_bytes))
    return width >= 4 ? small_as<T, 4>(ids, grad, vocab, scale, skip, table, s)
                      : small_as<T, 1>(ids, grad, vocab, scale, skip, table, s);
  const GradShape g = shape_of(ids.n, vocab, width);
  char* w = static_cast<char*>(workspace);
  Sorted sorted;
  sorted.start = reinterpret_cast<int32_t*>(w);
  sorted.id = reinterpret_cast<int32_t*>(w + g.start_bytes);
  sorted.position = reinterpret_cast<int32_t*>(w + g.start_bytes + g.list_bytes);
  sorted.partial = reinterpret_cast<float*>(w + g.start_bytes + 2 * g.list_bytes);
  sorted.rows = g.rows;
  sorted.shift = g.shift;
  sorted.slots = static_cast<int64_t>(g.rows) << g.shift;
  const int buckets = 1 << g.shift;
  const int64_t clear_rows = std::min<int64_t>(vocab, kClearBesideSort / row_bytes);
  const int64_t clear_bytes = clear_rows * row_bytes;
  const int64_t clear = (clear_bytes / 16 + kSortThreads) / kSortThreads;
  const int64_t blocks = buckets + std::min<int64_t>(clear, 1024);
  // of what is left to clear, the last launch gets half where that is much
  const bool joins = ids.n > kLight;
  const int64_t left = vocab - clear_rows;
  const int64_t until =
      joins && left * row_bytes > 2 * kClearBesideSort ? clear_rows + left / 2 : vocab;
  // 512 columns to a wave (256 of a narrow fp32 table), 16 bytes to a lane
  constexpr int kVec = 16 / sizeof(T), kPair = sizeof(T) == 4 ? 2 : 1;
  const bool brief = width < kVec, pair = kPair == 2 && width > kVec * kWave;
  const int64_t columns = kWave * (brief ? 1 : pair ? kVec * kPair : kVec);
  const int64_t slices = (width + columns - 1) / columns;
  int64_t sum_blocks, join_blocks;
  const Clear first =
      clear_after(g.spans * slices, clear_rows, until, row_bytes, kClearBytes, sum_blocks);
  const int64_t jobs = g.spans * ((width + kWave - 1) / kWave);
  // (a block to a CU: 16384 tokens of 50257 x 768 bf16 35.1 us, 37.2 with two)
  const Clear rest = clear_after(std::min<int64_t>(jobs, 256), until, vocab, row_bytes,
                                 4 * kClearBytes, join_blocks);
  if (!fits(sum_blocks, kSumThreads) || !fits(join_blocks, kJoinThreads)) return MS_OPS_EINVAL;

  const bool plain = ids.inner >= ids.n && ids.inner_stride == 1;
#define SORT(W, P)                                         \
  (ids.n <= 4 * kSortThreads   ? k_sort_tokens<4, W, P>    \
   : ids.n <= 8 * kSortThreads ? k_sort_tokens<8, W, P>    \
                               : k_sort_tokens<16, W, P>)
  int rc = launch(ids.wide ? plain ? SORT(true, true) : SORT(true, false)
                  : plain  ? SORT(false, true)
                           : SORT(false, false),
                  blocks, kSortThreads, s, ids, vocab, skip, buckets, sorted,
                  static_cast<uint4*>(dtable), clear_bytes);
#undef SORT
  if (!rc && sum_blocks)
    rc = launch(brief  ? k_sum_spans<T, 1, 1>
                : pair ? k_sum_spans<T, kVec, kPair>
                       : k_sum_spans<T, kVec, 1>,
                sum_blocks, kSumThreads, s, grad, scale, static_cast<int>(slices), first, sorted,
                table);
  if (!rc && joins)
    rc = launch(width < 4 ? k_join_spans<T, 1> : k_join_spans<T, 4>, join_blocks, kJoinThreads, s,
                ids.n, width, scale, rest, sorted, table);
  return rc;
}

}  // namespace

extern "C" int ms_embedding(const ms_tokens_t* ids, const ms_rows_t* table, float scale, void* out,
                            void* stream) {
  if (!good_tokens(ids) || !good_rows(table)) return MS_OPS_EINVAL;
  if (ids->n == 0 || table->width == 0) return MS_OPS_OK;
  if (!out || table->n < 1 || !countable(ids->n, table->width)) return MS_OPS_EINVAL;
  if (table->n > 1 && table->inner < table->n) return MS_OPS_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (table->dtype) {
    case MS_OPS_F32: return lookup_as<float>(*ids, *table, scale, out, s);
    case MS_OPS_F16: return lookup_as<f16>(*ids, *table, scale, out, s);
    default: return lookup_as<bf16>(*ids, *table, scale, out, s);
  }
}

extern "C" int64_t ms_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t width) {
  if (n < 0 || vocab < 0 || width < 0 || n > kMostTokens || vocab > INT32_MAX ||
      !countable(std::max(n, vocab), width))
    return -1;
  if (vocab == 0 || width == 0) return 0;
  const GradShape g = shape_of(n, vocab, width);
  return g.start_bytes + 2 * g.list_bytes + g.partial_bytes;
}

extern "C" int ms_embedding_grad(const ms_tokens_t* ids, const ms_rows_t* grad, int64_t vocab,
                                 float scale, int64_t padding_idx, void* dtable, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (!good_tokens(ids) || !good_rows(grad) || grad->n != ids->n || ids->n > kMostTokens ||
      vocab < 0 || vocab > INT32_MAX || !countable(vocab, grad->width))
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
