// What lies between two blocks of a model: the norm after the one, its gate and
// residual scale, the residual sum, and the norm before the next.
//
//   u  = norm(block) * block_weight + block_bias     (or block itself)
//   x' = residual + scale * gate * u
//   y  = norm(x') * weight + bias
//   norm(x) = (x - mean) * rstd, rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   (kind rms: mean taken as 0)
//
// Backward, with dy and dx' the gradients of the two results, n(t, v, rstd) =
// rstd * (t - mean(t) - v mean(t v)) (rms: without mean(t)), v = norm(x'):
//   dresidual = dx' + n(dy * weight, v, rstd) =: d
//   dweight = sum dy v,  dbias = sum dy                   (over the rows)
//   dgate = sum scale d u                                 (over a gate's rows)
//   q = scale gate d;  dblock_weight = sum q w, dblock_bias = sum q, w = norm(block)
//   dblock = n(q * block_weight, w, block rstd)           (or q)
//
// Memory bounds all of it: two rows read and two written forward, four and two backward.
// A row is held in registers by its team of threads, 16 bytes a thread at a time, and
// read once.  Everything is fp32 and rounded once where it is stored; variances are sums of
// squared differences from the mean, not differences of sums.
//
// Sums over rows: a block's teams take rows in turn and add into registers; the block
// leaves one partial sum for each column, and a second kernel joins those in the order of
// the blocks, so that the same call gives the same bits.
//
// Measured: forward 8192 x 2048 fp16 24.6 us (22.4 the kernel alone, 6.0 TB/s; 134 MB at the rate of a copy,
// 6.27 TB/s, 21.4), 8192 x 4096 bf16 with both norms and a gate 46 us.  Backward 8192 x 4096 bf16 with
// both norms and a gate 85-89 us (kernel 79, 5.1 TB/s; the join 6; floor 63), 16384 x 768 bf16 with 16 gates
// 39 us (34 and 5; floor 24).  Backward is held up by its two sums to a row, each with a
// barrier; streaming loads took it from 100 to 84 us (loads that stay in no cache leave room for
// the stores), streaming stores back to 94.  Rows above 8192 2-byte or 4096 4-byte values run
// at half that rate: they load their operands where they use them.
#include "ops_common.h"

#include <algorithm>

namespace ops {
namespace {

constexpr int64_t kMaxWidth = 16384;

// The sum over each N neighbouring lanes (up to 16), in every lane.
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
#define MS_DPP_ADD(ctrl) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, true))
  if (N > 1) MS_DPP_ADD(0xB1);    // lanes 1 0 3 2
  if (N > 2) MS_DPP_ADD(0x4E);    // lanes 2 3 0 1
  if (N > 4) MS_DPP_ADD(0x141);   // each 8 lanes mirrored
  if (N > 8) MS_DPP_ADD(0x140);   // each 16 lanes mirrored
#undef MS_DPP_ADD
  return x;
}

// The sum over a wave's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float x) {
  x = lanes_sum<16>(x);
  const int b = __float_as_int(x);
  return (__int_as_float(read_lane(b, 0)) + __int_as_float(read_lane(b, 16))) +
         (__int_as_float(read_lane(b, 32)) + __int_as_float(read_lane(b, 48)));
}

// Sums over a team of W waves (a power of two).  Two places take turns, so that one barrier is
// enough: a wave reaches the second next sum only after all have read this one.
template <int W>
struct Team {
  float2 (*place)[16];
  int turn = 0, wave, slot;

  __device__ Team(float2 (*p)[16], int wave_of_block)
      : place(p), wave(wave_of_block), slot(wave_of_block / W * W + threadIdx.x % W) {}
  __device__ float2 sum(float2 x, bool both) {
    x.x = wave_sum(x.x);
    if (both) x.y = wave_sum(x.y);
    if (W == 1) return x;
    place[turn][wave] = x;
    __syncthreads();
    x = place[turn][slot];
    x.x = lanes_sum<W>(x.x);
    if (both) x.y = lanes_sum<W>(x.y);
    turn ^= 1;
    return x;
  }
  __device__ float sum(float x) { return sum(make_float2(x, 0.0f), false).x; }
};

// What a thread has of a row, 16 bytes at a time, kept as they were loaded until they are used:
// taken apart earlier, they would be waited for.
template <typename T>
struct Words {
  uint32_t w[4];
  __device__ float operator[](int e) const {
    Pack<T, 16 / sizeof(T)> x;
    __builtin_memcpy(&x, w, 16);
    return widen(x.v[e]);
  }
};

// A thread's values narrowed in pairs, each rounded to nearest even (bf16 has an instruction for
// two).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow_all(const float (&x)[V]) {
  Pack<T, V> o;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = x[e];
  } else {
    typedef float two __attribute__((ext_vector_type(2)));
    typedef T halves __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      two pair = {x[e], x[e + 1]};
      asm("" : "+v"(pair));      // (no product and narrowing in one instruction, as in narrow())
      const halves h = __builtin_convertvector(pair, halves);
      o.v[e] = h[0];
      o.v[e + 1] = h[1];
    }
  }
  return o;
}

// The columns of a thread: 16 bytes at each of C byte offsets in a row.  Rows are reached as
// buffers that end with them, so that what lies behind the end is neither loaded (zeros) nor
// stored, by words and without a branch: behind a branch a wave could no longer tell its
// loads from its stores, which are counted together, and would wait for both.  The last value
// of a row of an odd number of 2-byte ones is moved by itself.
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kNowhere = 0x7ffffff0;

template <typename T, int W, int C>
struct Columns {
  static constexpr int V = 16 / sizeof(T);
  uint32_t at[C], last_at, last_word;
  int width;
  bool odd, ragged;       // ragged: the row ends inside a thread's 16 bytes

  __device__ Columns(int lane, int width_of) : width(width_of), ragged(width_of % V != 0) {
    odd = sizeof(T) == 2 && width % 2 != 0;
    const uint32_t end = (width - 1) * sizeof(T);
    last_at = kNowhere;
    last_word = 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      at[c] = (c * W * 64 + lane) * 16;
      if (odd && end >= at[c] && end < at[c] + 16) last_at = end, last_word = c * 4 + (end - at[c]) / 4;
    }
    if (last_at == kNowhere) last_word = 4 * C;
  }
  __device__ int column(int c, int e) const { return static_cast<int>(at[c] / sizeof(T)) + e; }
  __device__ bool in(int c, int e = 0) const { return column(c, e) < width; }
  // Behind the row's end the zeros that were loaded stay zeros: a mean stands alone there, and times its
  // deviation's reciprocal it can pass fp32's range where no value of the row does.  A mean for group c,
  // and what is left to do where a thread has the end among its values.
  __device__ float level(int c, float mean) const { return in(c) ? mean : 0.0f; }
  __device__ void clear(float (&y)[C][V]) const {
    if (!ragged) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 1; e < V; ++e) y[c][e] = in(c, e) ? y[c][e] : 0.0f;
  }
  // A row's buffer, or with there = false one of nothing.
  __device__ __amdgpu_buffer_rsrc_t buffer(const T* row, bool there = true) const {
    const int bytes = width * static_cast<int>(sizeof(T));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row), 0, there ? bytes : 0, 0x00027000);
  }
  template <bool NT = false>
  __device__ void load(const T* row, Words<T> (&x)[C], bool there = true) const {
    const __amdgpu_buffer_rsrc_t b = buffer(row, there);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const words4 r = __builtin_amdgcn_raw_buffer_load_b128(b, at[c], 0, NT ? 2 : 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[c].w[k] = r[k];
    }
    if (odd) {
      const uint32_t last = __builtin_amdgcn_raw_buffer_load_b16(b, last_at, 0, 0);
#pragma unroll
      for (int k = 0; k < 4 * C; ++k)
        if (last_word == static_cast<uint32_t>(k)) x[k / 4].w[k % 4] = last;
    }
  }
  __device__ void store(T* row, const Pack<T, V> (&x)[C], bool there = true) const {
    const __amdgpu_buffer_rsrc_t b = buffer(row, there);
    uint32_t last = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      words4 r;
      __builtin_memcpy(&r, &x[c], 16);
      __builtin_amdgcn_raw_buffer_store_b128(r, b, at[c], 0, 0);
      if (odd) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (last_word == static_cast<uint32_t>(c * 4 + k)) last = r[k];
      }
    }
    if (odd) __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(last), b, last_at, 0, 0);
  }
};

struct forward_args {
  ms_rows_t residual, block;           // block.data NULL: none
  const void *weight, *bias, *block_weight, *block_bias, *gate;
  int64_t gate_rows;                   // rows that share a gate
  float scale, eps;
  void *next, *out;
  float* stats;                        // [rows][2 or 4], or NULL
};

// Mean and reciprocal deviation of the team's row, held as C groups of V.  (The sum is taken 2^-14
// times, a row's longest, so that it stays within fp32's range as each value does; the same bits.
// What lies behind the row's end are zeros, or with `Behind` numbers of no meaning.)
constexpr float kDown = 0x1p-14f;
static_assert(kMaxWidth <= 1 << 14, "");
template <bool Layer, bool Behind, int C, int V, typename Cols, typename Of>
__device__ __forceinline__ float2 row_stats(const float (&x)[C][V], const Cols& cols, float eps,
                                            Of& team) {
  const float width = static_cast<float>(cols.width);
  float mean = 0.0f, sq = 0.0f;
  if (Layer) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!Behind || cols.in(c, e)) s = fmaf(x[c][e], kDown, s);
    mean = team.sum(s) / width * (1.0f / kDown);
  }
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = x[c][e] - mean;
      // (columns behind the end are zeros, but for the mean)
      if (!Layer || cols.in(c, e)) sq = fmaf(d, d, sq);
    }
  const float var = team.sum(sq) / width;
  return make_float2(mean, 1.0f / sqrtf(var + eps));
}

// A team of W waves to a row; blocks of at least 4 waves.  Everything is loaded before the first
// sum, which all would wait for.
template <typename T, int W, int C, bool Layer, bool Post>
__global__ __launch_bounds__(W < 4 ? 256 : W * 64) void k_norm(forward_args a) {
  constexpr int V = 16 / sizeof(T), kWaves = W < 4 ? 4 : W;
  __shared__ float2 place[2][16];
  const int tid = threadIdx.x, wave = uniform(tid >> 6);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWaves / W) + wave / W;
  if (W == 1 && row >= a.residual.n) return;
  static_assert(W == 1 || W >= 4, "the waves of a block belong to one row, or each has its own");
  const int width = static_cast<int>(a.residual.width);
  const int lane = tid % (W * 64);
  Team<W> team(place, wave);
  const Columns<T, W, C> cols(lane, width);
  Words<T> residual[C], more[C], weight[C], bias[C], gate[C], block_weight[C], block_bias[C];
  const bool block_there = a.block.data != nullptr, gated = a.gate != nullptr;
  auto vector = [&](const void* p, Words<T>(&x)[C]) {
    const T* some = static_cast<const T*>(p ? p : a.weight);
    cols.load(some, x, p != nullptr);
  };
  cols.load(static_cast<const T*>(a.residual.data) + row_start(a.residual, row), residual);
  const T* rows = static_cast<const T*>(block_there ? a.block.data : a.residual.data);
  cols.load(rows + (block_there ? row_start(a.block, row) : 0), more, block_there);
  vector(a.weight, weight);
  if (Layer) vector(a.bias, bias);
  if (Post) vector(a.block_weight, block_weight);
  if (Post && Layer) vector(a.block_bias, block_bias);
  if (gated)
    cols.load(static_cast<const T*>(a.gate) +
                  static_cast<uint32_t>(row) / static_cast<uint32_t>(a.gate_rows) *
                      static_cast<int64_t>(width),
              gate);
  float x[C][V];
  Pack<T, V> o[C];
  float2 post = make_float2(0.0f, 1.0f);
  if (block_there) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = more[c][e];
    if (Post) {
      post = row_stats<Layer, false>(x, cols, a.eps, team);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[c][e] = fmaf((x[c][e] - post.x) * post.y, block_weight[c][e], Layer ? block_bias[c][e] : 0.0f);
    }
    if (gated) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) x[c][e] *= gate[c][e];
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = fmaf(x[c][e], a.scale, residual[c][e]);
      o[c] = narrow_all<T>(x[c]);
    }
    cols.store(static_cast<T*>(a.next) + row * width, o);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = residual[c][e];
  }
  const float2 pre = row_stats<Layer, Post>(x, cols, a.eps, team);
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      x[c][e] = fmaf((x[c][e] - pre.x) * pre.y, weight[c][e], Layer ? bias[c][e] : 0.0f);
    o[c] = narrow_all<T>(x[c]);
  }
  cols.store(static_cast<T*>(a.out) + row * width, o);
  if (a.stats && lane == 0) {
    float* s = a.stats + row * (Post ? 4 : 2);
    s[0] = pre.x;
    s[1] = pre.y;
    if (Post) {
      s[2] = post.x;
      s[3] = post.y;
    }
  }
}

// ---------------------------------------------------------------------------

struct backward_args {
  ms_rows_t dout, dnext, next, block;       // data NULL: none (dout and dnext not both)
  const float* stats;
  const void *weight, *block_weight, *block_bias, *gate;
  int64_t gate_rows, parts, item_rows, items;
  float scale;
  void *dresidual, *dblock;
  float* sums;              // [block][vector][width]
  float* gate_sums;         // [item][width], or NULL
  void* dgate;              // where each gate's rows are one item
};

// Waves of a block: eight, so that two blocks of a CU wait at different barriers, or a row's.
constexpr int block_waves(int w) { return w < 8 ? 8 : w; }

// Teams of W waves.  An item is up to item_rows neighbouring rows that share a gate;
// teams take items in turn, all the same number of rows, since the barriers are the
// block's.  Rows of up to 16 bytes a thread (C = 1): a row's loads are under way while
// the one before is worked on, and all sums are in registers.  Longer ones have neither
// registers: operands are loaded where they are used, and the first two sums are in LDS.
template <typename T, int W, int C, bool Layer, bool Post>
__global__ __launch_bounds__(block_waves(W) * 64, Layer && Post && W < 16 ? 2 : 4) void k_norm_grad(backward_args a) {
  constexpr int V = 16 / sizeof(T), kTeams = block_waves(W) / W;
  constexpr bool kShort = C == 1;
  constexpr int kVectors = (Layer ? 2 : 1) * (Post ? 2 : 1);
  constexpr int kInLds = kShort ? 0 : kVectors < 2 ? kVectors : 2, kInRegs = kVectors - kInLds;
  // weight, bias, block weight, block bias, as far as there are any
  constexpr int kWeight = 0, kBias = Layer, kBlockWeight = Post ? 1 + Layer : 0,
                kBlockBias = Layer && Post ? 3 : 0;
  __shared__ float2 place[2][16];
  __shared__ float joined[kShort ? (kTeams > 1 ? W * 64 * V : 1) : kInLds * W * 64 * C * V];
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid % (W * 64);
  const int width = static_cast<int>(a.next.width);
  const float inverse = 1.0f / static_cast<float>(width);
  Team<W> team(place, wave);
  const Columns<T, W, C> cols(lane, width);
  const T* const weights = static_cast<const T*>(a.weight);
  const T* const block_weights = static_cast<const T*>(a.block_weight);
  const T* const block_biases = static_cast<const T*>(a.block_bias);
  Words<T> weight[C], block_weight[C], block_bias[C], gate[C];
  auto load_block_vectors = [&] {
    if (Post) cols.load(block_weights, block_weight);
    if (Post && Layer) cols.load(block_biases ? block_biases : weights, block_bias, block_biases);
  };
  if (kShort) {
    cols.load(weights, weight);
    load_block_vectors();
  }
  float sums[kInRegs > 0 ? kInRegs : 1][C][V] = {}, gate_sum[C][V] = {};
  if (!kShort) {
    for (int k = tid; k < kInLds * W * 64 * C * V; k += W * 64) joined[k] = 0.0f;
  }
  // x y to sum k.  (A thread's own places in LDS, so that no barrier is needed.)
  auto add = [&](int k, int c, int e, float x, float y) {
    if (k < kInLds) {
      float* p = &joined[((k * C + c) * V + e) * W * 64 + lane];
      *p = fmaf(x, y, *p);
    } else {
      sums[k - kInLds][c][e] = fmaf(x, y, sums[k - kInLds][c][e]);
    }
  };
  const bool block_there = a.block.data != nullptr, gated = a.gate != nullptr;
  const bool dout_there = a.dout.data != nullptr, dnext_there = a.dnext.data != nullptr;
  constexpr int kFields = Post ? 4 : 2;

  // (Unsigned: what lies up to a turn of all teams, or an item's rows, behind the last of 2^31 - 1
  // is counted too.)
  const uint32_t teams = gridDim.x * kTeams, items = static_cast<uint32_t>(a.items);
  const uint32_t rounds = (items + teams - 1) / teams;
  const uint32_t parts = static_cast<uint32_t>(a.parts), gate_rows = static_cast<uint32_t>(a.gate_rows);
  const int item_rows = static_cast<int>(a.item_rows);
  // The team's item of a round, `count` rows from `row` on: none where it has no item.
  auto place_of = [&](uint32_t round, uint32_t& item, uint32_t& group, uint32_t& row, int& count) {
    item = static_cast<uint32_t>(uniform(static_cast<int>(round * teams + blockIdx.x * kTeams + wave / W)));
    const bool live = round < rounds && item < items;
    group = live ? item / parts : 0;
    const uint32_t begin = (live ? item - group * parts : 0) * static_cast<uint32_t>(item_rows);
    row = group * gate_rows + begin;
    count = live ? static_cast<int>(min(static_cast<uint32_t>(item_rows), gate_rows - begin)) : 0;
  };

  auto row_of = [](const ms_rows_t& m, uint32_t row) {
    return static_cast<const T*>(m.data) + row_start(m, row);
  };
  struct Row {
    Words<T> dy[C], dx[C], x[C], b[C];
    float mean, rstd, block_mean, block_rstd;
  };
  // The loads of a row, of nothing where there is none
  auto fetch = [&](uint32_t row, bool live, Row& r) {
    cols.template load<true>(row_of(a.next, row), r.x, live);
    cols.template load<true>(dout_there ? row_of(a.dout, row) : weights, r.dy, live && dout_there);
    if (kShort) {
      cols.template load<true>(dnext_there ? row_of(a.dnext, row) : weights, r.dx, live && dnext_there);
      cols.template load<true>(block_there ? row_of(a.block, row) : weights, r.b, live && block_there);
    }
    // (zeros, with which the row that is none adds nothing to any sum)
    const float* s = a.stats + (live ? static_cast<int64_t>(row) * kFields : 0);
    r.mean = live ? s[0] : 0.0f;
    r.rstd = live ? s[1] : 0.0f;
    if (Post) {
      r.block_mean = live ? s[2] : 0.0f;
      r.block_rstd = live ? s[3] : 0.0f;
    }
  };

  Row now, then;
  uint32_t item, group, row;
  int count;
  place_of(0, item, group, row, count);
  Pack<T, V> o[C];
  if (kShort) {
    fetch(row, count > 0, then);
    // Two stores of nothing: as many follow the loads of every later row, so that the wait
    // for loads is known not to be one for those stores.
    cols.store(static_cast<T*>(a.dresidual), o, false);
    cols.store(static_cast<T*>(a.dresidual), o, false);
  }
  for (uint32_t round = 0; round < rounds; ++round) {
    uint32_t next_item, next_group, next_row;
    int next_count;
    place_of(round + 1, next_item, next_group, next_row, next_count);
    const T* gates = static_cast<const T*>(a.gate) + static_cast<int64_t>(group) * width;
    if (gated && kShort) cols.load(gates, gate);
    for (int k = 0; k < item_rows; ++k, ++row) {
      const bool live = k < count;
      if (kShort) {
        now = then;
        const bool last = k + 1 == item_rows;
        fetch(last ? next_row : row + 1, last ? next_count > 0 : k + 1 < count, then);
      } else {
        fetch(row, live, now);
        cols.load(weights, weight);
      }
      // d: first the normalised row, then its gradient
      float2 s = make_float2(0.0f, 0.0f);
      float d[C][V];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float level = Layer ? cols.level(c, now.mean) : 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) d[c][e] = (now.x[c][e] - level) * now.rstd;
      }
      if (Layer) cols.clear(d);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float t = now.dy[c][e] * weight[c][e];
          s.x = fmaf(t, d[c][e], s.x);
          if (Layer) s.y += t;
        }
      s = team.sum(s, Layer);
      if (!kShort) {
        cols.load(weights, weight);
        cols.load(dnext_there ? row_of(a.dnext, row) : weights, now.dx, live && dnext_there);
      }
      float2 s2 = make_float2(0.0f, 0.0f);
      const float along = s.x * inverse, level = Layer ? s.y * inverse : 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = d[c][e], g = now.dy[c][e];
          add(kWeight, c, e, g, v);
          if (Layer) add(kBias, c, e, g, 1.0f);
          float r = fmaf(-v, along, g * weight[c][e]);
          if (Layer) r -= level;
          d[c][e] = fmaf(r, now.rstd, now.dx[c][e]);
        }
        o[c] = narrow_all<T>(d[c]);
      }
      cols.store(static_cast<T*>(a.dresidual) + (live ? static_cast<int64_t>(row) * width : 0), o, live);
      if (!kShort) {
        cols.load(block_there ? row_of(a.block, row) : weights, now.b, live && block_there);
        load_block_vectors();
        if (gated) cols.load(gates, gate);
      }
      float w[C][V] = {};
      if (Post) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float level = Layer ? cols.level(c, now.block_mean) : 0.0f;
#pragma unroll
          for (int e = 0; e < V; ++e) w[c][e] = (now.b[c][e] - level) * now.block_rstd;
        }
        if (Layer) cols.clear(w);
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float q = d[c][e] * a.scale;
          if (gated) {
            const float u = Post ? fmaf(w[c][e], block_weight[c][e], Layer ? block_bias[c][e] : 0.0f)
                                 : now.b[c][e];
            gate_sum[c][e] = fmaf(q, u, gate_sum[c][e]);
            q *= gate[c][e];
          }
          if (Post) {
            add(kBlockWeight, c, e, q, w[c][e]);
            if (Layer) add(kBlockBias, c, e, q, 1.0f);
            // (the weight is 0 behind the row's end)
            q *= block_weight[c][e];
            s2.x = fmaf(q, w[c][e], s2.x);
            if (Layer) s2.y += q;
          }
          d[c][e] = q;
        }
      if (Post) s2 = team.sum(s2, Layer);
      const float block_along = s2.x * inverse, block_level = Layer ? s2.y * inverse : 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (Post) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float q = fmaf(-w[c][e], block_along, d[c][e]);
            if (Layer) q -= block_level;
            d[c][e] = q * now.block_rstd;
          }
        }
        o[c] = narrow_all<T>(d[c]);
      }
      cols.store(static_cast<T*>(block_there ? a.dblock : a.dresidual) +
                     (live ? static_cast<int64_t>(row) * width : 0),
                 o, live && block_there);
    }
    if (gated && item < items) {
      float* sums_out = a.gate_sums + static_cast<int64_t>(item) * width;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (a.gate_sums && cols.in(c, e)) sums_out[cols.column(c, e)] = gate_sum[c][e];
          o[c].v[e] = narrow<T>(gate_sum[c][e]);
          gate_sum[c][e] = 0.0f;
        }
      cols.store(a.gate_sums ? static_cast<T*>(a.dresidual)
                             : static_cast<T*>(a.dgate) + static_cast<int64_t>(group) * width,
                 o, !a.gate_sums);
    }
    item = next_item;
    group = next_group;
    row = next_row;
    count = next_count;
  }

  // The block's sums: one team after the other adds in LDS.
  const int which = wave / W;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (kTeams > 1) {
      for (int t = 0; t < kTeams; ++t) {
        __syncthreads();
        if (which != t) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float* p = &joined[e * W * 64 + lane];
          if (t > 0) sums[k < kInRegs ? k : 0][0][e] += *p;
          *p = sums[k < kInRegs ? k : 0][0][e];
        }
      }
    }
    if (which == kTeams - 1) {
      float* out = a.sums + (static_cast<int64_t>(blockIdx.x) * kVectors + k) * width;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (cols.in(c, e))
            out[cols.column(c, e)] = k < kInLds ? joined[((k * C + c) * V + e) * W * 64 + lane]
                                                : sums[k - kInLds][c][e];
    }
  }
}

// Joins partial sums: out[g][column] = sum over p < count of from[g][p][column].
struct join_t {
  const float* from;
  int64_t groups, group_stride, part_stride;
  int32_t count;
  void* out;
};
struct joins_t {
  join_t of[5];
};

template <typename T>
__global__ __launch_bounds__(1024) void k_join_rows(joins_t joins, int64_t width) {
  __shared__ float held[16][64];
  const join_t j = joins.of[blockIdx.y];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int64_t bands = (width + 63) / 64;
  for (int64_t b = blockIdx.x; b < j.groups * bands; b += gridDim.x) {
    const int64_t g = b / bands, c = (b - g * bands) * 64 + lane;
    const float* p = j.from + g * j.group_stride + c;
    float sum = 0.0f;
    if (c < width) {
#pragma unroll 4
      for (int k = slice; k < j.count; k += 16) sum += p[k * j.part_stride];
    }
    __syncthreads();
    held[slice][lane] = sum;
    __syncthreads();
    if (slice == 0 && c < width) {
      for (int k = 1; k < 16; ++k) sum += held[k][lane];
      static_cast<T*>(j.out)[g * width + c] = narrow<T>(sum);
    }
  }
}

// No rows: gradients of zeros.
template <typename T>
__global__ __launch_bounds__(256) void k_zero_vectors(joins_t joins, int64_t width) {
  T* out = static_cast<T*>(joins.of[blockIdx.y].out);
  const int64_t n = joins.of[blockIdx.y].groups * width;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * 256)
    out[i] = static_cast<T>(0.0f);
}

// ---------------------------------------------------------------------------
// Host.

int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }

bool same_rows(const ms_rows_t* m, const ms_rows_t& like) {
  return !m || (good_rows(m) && m->n == like.n && m->width == like.width && m->dtype == like.dtype);
}

bool good_norm(const ms_rows_t* x, const ms_rows_t* block, int32_t kind, const void* weight,
               const void* bias, const void* block_weight, const void* block_bias, const void* gate,
               int64_t gates) {
  if (!good_rows(x) || !same_rows(block, *x) || x->width < 1 || x->width > kMaxWidth || !weight ||
      (kind != MS_NORM_RMS && kind != MS_NORM_LAYER))
    return false;
  if (kind == MS_NORM_RMS && (bias || block_bias)) return false;
  if (!block && (block_weight || gate)) return false;
  if (block_bias && !block_weight) return false;
  return gate ? gates >= 1 && (x->n == 0 || x->n % gates == 0) : gates == 0;
}

template <typename T, int W, int C>
int run_forward(const forward_args& a, bool layer, hipStream_t s) {
  constexpr int kWaves = W < 4 ? 4 : W;
  const int64_t blocks = ceil_div(a.residual.n, kWaves / W);
  if (!fits(blocks, kWaves * 64)) return MS_OPS_EINVAL;
  if (a.block_weight)
    return layer ? launch(k_norm<T, W, C, true, true>, blocks, kWaves * 64, s, a)
                 : launch(k_norm<T, W, C, false, true>, blocks, kWaves * 64, s, a);
  return layer ? launch(k_norm<T, W, C, true, false>, blocks, kWaves * 64, s, a)
               : launch(k_norm<T, W, C, false, false>, blocks, kWaves * 64, s, a);
}

// A wave to a row while it holds it in 32 bytes a lane, as no barrier is needed then; more
// waves rather than more registers for longer ones (2048 fp16: 64 bytes a lane 41.6 us).
template <typename T>
int choose_forward(const forward_args& a, bool layer, hipStream_t s) {
  const int64_t chunks = ceil_div(a.residual.width, 16 / static_cast<int>(sizeof(T)) * 64);
  if (chunks <= 1) return run_forward<T, 1, 1>(a, layer, s);
  if (chunks <= 2) return run_forward<T, 1, 2>(a, layer, s);
  if (chunks <= 4) return run_forward<T, 4, 1>(a, layer, s);
  if (chunks <= 8) return run_forward<T, 8, 1>(a, layer, s);
  if (chunks <= 16) return run_forward<T, 16, 1>(a, layer, s);
  if (chunks <= 32) return run_forward<T, 16, 2>(a, layer, s);
  if constexpr (sizeof(T) == 4) return run_forward<T, 16, 4>(a, layer, s);
  return MS_OPS_EINVAL;       // (no 2-byte row is that long)
}

// How backward cuts the rows: teams of `waves`, `blocks` of them, items of a gate's rows.
struct Shares {
  int waves;
  int64_t blocks, parts, item_rows, items;
};

Shares shares_of(int64_t n, int64_t width, int64_t bytes, int64_t gates) {
  Shares s{};
  const int64_t chunks = ceil_div(width * bytes, 16 * 64);
  s.waves = 1;
  while (s.waves < 16 && s.waves < chunks) s.waves *= 2;
  const int64_t teams_of_block = block_waves(s.waves) / s.waves;
  s.blocks = std::min<int64_t>(s.waves == 16 ? 256 : 512, ceil_div(n, teams_of_block));
  const int64_t teams = s.blocks * teams_of_block, groups = std::max<int64_t>(gates, 1);
  const int64_t rows = n / groups;
  // A gate's rows in as many parts as give the teams equal turns, one to four of them
  int64_t least = INT64_MAX;
  for (int64_t turns = 1; turns <= 4; ++turns) {
    const int64_t p = std::max<int64_t>(1, std::min(turns * teams / groups, rows));
    const int64_t each = ceil_div(rows, p), took = ceil_div(groups * ceil_div(rows, each), teams) * each;
    if (took < least) least = took, s.parts = p;
  }
  s.item_rows = ceil_div(rows, s.parts);
  s.parts = ceil_div(rows, s.item_rows);
  s.items = groups * s.parts;
  return s;
}

int vectors_of(bool layer, bool post) { return (layer ? 2 : 1) * (post ? 2 : 1); }

int64_t grad_workspace(const Shares& s, int64_t width, bool layer, bool post, bool gated) {
  return (s.blocks * vectors_of(layer, post) + (gated && s.parts > 1 ? s.items : 0)) * width * 4;
}

template <typename T, int W, int C>
int run_backward(const backward_args& a, bool layer, bool post, int64_t blocks, hipStream_t s) {
  if (layer)
    return post ? launch(k_norm_grad<T, W, C, true, true>, blocks, block_waves(W) * 64, s, a)
                : launch(k_norm_grad<T, W, C, true, false>, blocks, block_waves(W) * 64, s, a);
  return post ? launch(k_norm_grad<T, W, C, false, true>, blocks, block_waves(W) * 64, s, a)
              : launch(k_norm_grad<T, W, C, false, false>, blocks, block_waves(W) * 64, s, a);
}

template <typename T>
int choose_backward(const backward_args& a, bool layer, bool post, const Shares& sh, hipStream_t s) {
  const int64_t chunks = ceil_div(a.next.width * static_cast<int64_t>(sizeof(T)), 16 * 64);
  switch (sh.waves) {
    case 1: return run_backward<T, 1, 1>(a, layer, post, sh.blocks, s);
    case 2: return run_backward<T, 2, 1>(a, layer, post, sh.blocks, s);
    case 4: return run_backward<T, 4, 1>(a, layer, post, sh.blocks, s);
    case 8: return run_backward<T, 8, 1>(a, layer, post, sh.blocks, s);
  }
  if (chunks <= 16) return run_backward<T, 16, 1>(a, layer, post, sh.blocks, s);
  if (chunks <= 32) return run_backward<T, 16, 2>(a, layer, post, sh.blocks, s);
  if constexpr (sizeof(T) == 4) return run_backward<T, 16, 4>(a, layer, post, sh.blocks, s);
  return MS_OPS_EINVAL;
}

template <typename T>
int run_joins(joins_t joins, int count, int64_t width, hipStream_t s) {
  int64_t most = 1;
  for (int k = 0; k < count; ++k) most = std::max(most, joins.of[k].groups * ceil_div(width, 64));
  void* args[] = {&joins, &width};
  return static_cast<int>(hipLaunchKernel(reinterpret_cast<const void*>(k_join_rows<T>),
                                          dim3(std::min<int64_t>(most, 4096), count), dim3(1024), args,
                                          0, s));
}
template <typename T>
int run_zeros(joins_t joins, int count, int64_t width, hipStream_t s) {
  void* args[] = {&joins, &width};
  return static_cast<int>(hipLaunchKernel(reinterpret_cast<const void*>(k_zero_vectors<T>),
                                          dim3(ceil_div(width, 256), count), dim3(256), args, 0, s));
}

}  // namespace
}  // namespace ops

extern "C" {

int ms_norm(const ms_rows_t* residual, const ms_rows_t* block, int32_t kind, const void* weight,
            const void* bias, const void* block_weight, const void* block_bias, const void* gate,
            int64_t gates, float scale, float eps, void* next, void* out, float* stats, void* stream) {
  using namespace ops;
  if (!good_norm(residual, block, kind, weight, bias, block_weight, block_bias, gate, gates))
    return MS_OPS_EINVAL;
  if (residual->n == 0) return MS_OPS_OK;
  if (!out || (block && !next)) return MS_OPS_EINVAL;
  forward_args a{};
  a.residual = *residual;
  if (block) a.block = *block;
  a.weight = weight;
  a.bias = bias;
  a.block_weight = block_weight;
  a.block_bias = block_bias;
  a.gate = gate;
  a.gate_rows = gate ? residual->n / gates : 1;
  a.scale = scale;
  a.eps = eps;
  a.next = next;
  a.out = out;
  a.stats = stats;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool layer = kind == MS_NORM_LAYER;
  switch (residual->dtype) {
    case MS_OPS_F32: return choose_forward<float>(a, layer, s);
    case MS_OPS_F16: return choose_forward<f16>(a, layer, s);
    default: return choose_forward<bf16>(a, layer, s);
  }
}

int64_t ms_norm_grad_workspace(int64_t n, int64_t width, int32_t dtype, int32_t kind, int32_t post,
                               int64_t gates) {
  using namespace ops;
  if (n < 0 || n > INT32_MAX || width < 1 || width > kMaxWidth || !good_dtype(dtype) || gates < 0 ||
      (gates && n % gates))
    return MS_OPS_EINVAL;
  if (n == 0) return 0;
  return grad_workspace(shares_of(n, width, dtype_bytes(dtype), gates), width, kind == MS_NORM_LAYER,
                        post != 0, gates != 0);
}

int ms_norm_grad(const ms_rows_t* dout, const ms_rows_t* dnext, const ms_rows_t* next,
                 const float* stats, const ms_rows_t* block, int32_t kind, const void* weight,
                 const void* block_weight, const void* block_bias, const void* gate, int64_t gates,
                 float scale, void* dresidual, void* dblock, void* dweight, void* dbias,
                 void* dblock_weight, void* dblock_bias, void* dgate, void* workspace,
                 int64_t workspace_bytes, void* stream) {
  using namespace ops;
  if (!good_norm(next, block, kind, weight, dbias, block_weight, block_bias, gate, gates) ||
      !same_rows(dout, *next) || !same_rows(dnext, *next))
    return MS_OPS_EINVAL;
  const bool layer = kind == MS_NORM_LAYER, post = block_weight != nullptr;
  if (!dweight || (post && !dblock_weight) || (!post && (dblock_weight || dblock_bias)) ||
      (!layer && dblock_bias) || (gate != nullptr) != (dgate != nullptr))
    return MS_OPS_EINVAL;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t n = next->n, width = next->width;
  void* outs[] = {dweight, layer ? dbias : dblock_weight, dblock_weight, dblock_bias};
  const int vectors = vectors_of(layer, post);
  if (n == 0) {
    joins_t zeros{};
    int count = 0;
    for (int k = 0; k < vectors; ++k)
      if (outs[k]) zeros.of[count++] = {nullptr, 1, 0, 0, 0, outs[k]};
    if (gate) zeros.of[count++] = {nullptr, gates, 0, 0, 0, dgate};
    return next->dtype == MS_OPS_F32 ? run_zeros<float>(zeros, count, width, s)
                                     : run_zeros<f16>(zeros, count, width, s);
  }
  if ((!dout && !dnext) || !stats || !dresidual || (block && !dblock)) return MS_OPS_EINVAL;
  const Shares sh = shares_of(n, width, dtype_bytes(next->dtype), gates);
  if (workspace_bytes < grad_workspace(sh, width, layer, post, gate) || !workspace ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return MS_OPS_EWORKSPACE;
  backward_args a{};
  if (dout) a.dout = *dout;
  if (dnext) a.dnext = *dnext;
  a.next = *next;
  if (block) a.block = *block;
  a.stats = stats;
  a.weight = weight;
  a.block_weight = block_weight;
  a.block_bias = block_bias;
  a.gate = gate;
  a.gate_rows = gate ? n / gates : n;
  a.parts = sh.parts;
  a.item_rows = sh.item_rows;
  a.items = sh.items;
  a.scale = scale;
  a.dresidual = dresidual;
  a.dblock = dblock;
  a.sums = static_cast<float*>(workspace);
  const bool gate_parts = gate && sh.parts > 1;
  a.gate_sums = gate_parts ? a.sums + sh.blocks * vectors * width : nullptr;
  a.dgate = dgate;
  int rc;
  switch (next->dtype) {
    case MS_OPS_F32: rc = choose_backward<float>(a, layer, post, sh, s); break;
    case MS_OPS_F16: rc = choose_backward<f16>(a, layer, post, sh, s); break;
    default: rc = choose_backward<bf16>(a, layer, post, sh, s);
  }
  if (rc) return rc;
  joins_t joins{};
  int count = 0;
  for (int k = 0; k < vectors; ++k)
    if (outs[k])
      joins.of[count++] = {a.sums + k * width, 1, 0, vectors * width, static_cast<int32_t>(sh.blocks),
                           outs[k]};
  if (gate_parts)
    joins.of[count++] = {a.gate_sums, gates, sh.parts * width, width,
                         static_cast<int32_t>(sh.parts), dgate};
  switch (next->dtype) {
    case MS_OPS_F32: return run_joins<float>(joins, count, width, s);
    case MS_OPS_F16: return run_joins<f16>(joins, count, width, s);
    default: return run_joins<bf16>(joins, count, width, s);
  }
}

}  // extern "C"
