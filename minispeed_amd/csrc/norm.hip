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
#include "ops_common.h"

#include <algorithm>

namespace ops {
namespace {

constexpr int64_t kMaxWidth = 16384;

// The sum over a wave's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float x) {
#define MS_DPP_ADD(ctrl) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, true))
  MS_DPP_ADD(0xB1);    // lanes 1 0 3 2
  MS_DPP_ADD(0x4E);    // lanes 2 3 0 1
  MS_DPP_ADD(0x141);   // each 8 lanes mirrored
  MS_DPP_ADD(0x140);   // each 16 lanes mirrored
#undef MS_DPP_ADD
  const int b = __float_as_int(x);
  return (__int_as_float(read_lane(b, 0)) + __int_as_float(read_lane(b, 16))) +
         (__int_as_float(read_lane(b, 32)) + __int_as_float(read_lane(b, 48)));
}

// Sums over a team of W waves.  Two places take turns, so that one barrier is enough: a
// wave reaches the second next sum only after all have read this one.
template <int W>
struct Team {
  float2 (*place)[16];
  int turn = 0, wave, first;

  __device__ Team(float2 (*p)[16], int wave_of_block) : place(p), wave(wave_of_block) {
    first = wave / W * W;
  }
  __device__ float2 sum(float2 x, bool both) {
    x.x = wave_sum(x.x);
    if (both) x.y = wave_sum(x.y);
    if (W == 1) return x;
    place[turn][wave] = x;
    __syncthreads();
    float2 s = place[turn][first];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      const float2 o = place[turn][first + k];
      s.x += o.x;
      s.y += o.y;
    }
    turn ^= 1;
    return s;
  }
  __device__ float sum(float x) { return sum(make_float2(x, 0.0f), false).x; }
};

// V values at column c of a row of `width`; those behind its end are zeros.
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_columns(const T* p, int64_t c, int64_t width) {
  if (c + V <= width) return load<V>(p + c);
  Pack<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = c + e < width ? p[c + e] : static_cast<T>(0.0f);
  return x;
}
template <int V, typename T>
__device__ __forceinline__ void store_columns(T* p, int64_t c, int64_t width, const Pack<T, V>& x) {
  if (c + V <= width) {
    store<V>(p + c, x);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c + e < width) p[c + e] = x.v[e];
  }
}

struct forward_args {
  ms_rows_t residual, block;           // block.data NULL: none
  const void *weight, *bias, *block_weight, *block_bias, *gate;
  int64_t gate_rows;                   // rows that share a gate
  float scale, eps;
  void *next, *out;
  float* stats;                        // [rows][2 or 4], or NULL
};

// Mean and reciprocal deviation of the team's row, held as C groups of V.
template <bool Layer, int C, int V, typename Of>
__device__ __forceinline__ float2 row_stats(const float (&x)[C][V], const int64_t (&col)[C],
                                            int64_t width, float eps, Of& team) {
  float mean = 0.0f, sq = 0.0f;
  if (Layer) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) s += x[c][e];
    mean = team.sum(s) / static_cast<float>(width);
  }
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = x[c][e] - mean;
      // (columns behind the end are zeros, but for the mean)
      if (!Layer || col[c] + e < width) sq = fmaf(d, d, sq);
    }
  const float var = team.sum(sq) / static_cast<float>(width);
  return make_float2(mean, 1.0f / sqrtf(var + eps));
}

// A team of W waves to a row; blocks of at least 4 waves.
template <typename T, int W, int C, bool Layer>
__global__ __launch_bounds__(W < 4 ? 256 : W * 64) void k_norm(forward_args a) {
  constexpr int V = 16 / sizeof(T), kWaves = W < 4 ? 4 : W;
  __shared__ float2 place[2][16];
  const int tid = threadIdx.x, wave = uniform(tid >> 6);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWaves / W) + wave / W;
  if (W == 1 && row >= a.residual.n) return;
  static_assert(W == 1 || W >= 4, "the waves of a block belong to one row, or each has its own");
  const int64_t width = a.residual.width;
  const int lane = tid % (W * 64);
  Team<W> team(place, wave);
  int64_t col[C];
  float x[C][V];
  Pack<T, V> raw[C], more[C];
  const T* residual = static_cast<const T*>(a.residual.data) + row_start(a.residual, row);
  const T* block = static_cast<const T*>(a.block.data) + (a.block.data ? row_start(a.block, row) : 0);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (static_cast<int64_t>(c) * W * 64 + lane) * V;
    raw[c] = load_columns<V>(residual, col[c], width);
    if (a.block.data) more[c] = load_columns<V>(block, col[c], width);
  }
  float2 post = make_float2(0.0f, 1.0f);
  const T* gate = static_cast<const T*>(a.gate) + (a.gate ? row / a.gate_rows * width : 0);
  if (a.block.data) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = widen(more[c].v[e]);
    if (a.block_weight) {
      post = row_stats<Layer>(x, col, width, a.eps, team);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Pack<T, V> w = load_columns<V>(static_cast<const T*>(a.block_weight), col[c], width);
        Pack<T, V> b{};
        if (Layer && a.block_bias)
          b = load_columns<V>(static_cast<const T*>(a.block_bias), col[c], width);
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[c][e] = fmaf((x[c][e] - post.x) * post.y, widen(w.v[e]), widen(b.v[e]));
      }
    }
    if (a.gate) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Pack<T, V> g = load_columns<V>(gate, col[c], width);
#pragma unroll
        for (int e = 0; e < V; ++e) x[c][e] *= widen(g.v[e]);
      }
    }
    T* next = static_cast<T*>(a.next) + row * width;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      Pack<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] = fmaf(x[c][e], a.scale, widen(raw[c].v[e]));
        o.v[e] = narrow<T>(x[c][e]);
      }
      store_columns<V>(next, col[c], width, o);
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = widen(raw[c].v[e]);
  }
  const float2 pre = row_stats<Layer>(x, col, width, a.eps, team);
  T* out = static_cast<T*>(a.out) + row * width;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Pack<T, V> w = load_columns<V>(static_cast<const T*>(a.weight), col[c], width);
    Pack<T, V> b{}, o;
    if (Layer && a.bias) b = load_columns<V>(static_cast<const T*>(a.bias), col[c], width);
#pragma unroll
    for (int e = 0; e < V; ++e)
      o.v[e] = narrow<T>(fmaf((x[c][e] - pre.x) * pre.y, widen(w.v[e]), widen(b.v[e])));
    store_columns<V>(out, col[c], width, o);
  }
  if (a.stats && lane == 0) {
    const int fields = a.block.data && a.block_weight ? 4 : 2;
    float* s = a.stats + row * fields;
    s[0] = pre.x;
    s[1] = pre.y;
    if (fields == 4) {
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

// What a thread has of a row: 4 neighbouring columns C times, so that the sums and the
// next row's values fit in the registers beside it.
constexpr int kOwn = 4;
template <typename T, int C>
struct Row {
  Pack<T, kOwn> dy[C], dx[C], x[C], b[C];
  float mean, rstd, block_mean, block_rstd;
  bool live;
};

// Teams of W waves.  An item is up to item_rows neighbouring rows that share a gate;
// teams take items in turn, all the same number of rows, since the barriers are the
// block's.  A row's loads are under way while the one before is worked on.
template <typename T, int W, int C, bool Layer, bool Post>
__global__ __launch_bounds__(block_waves(W) * 64) void k_norm_grad(backward_args a) {
  constexpr int V = kOwn, kTeams = block_waves(W) / W;
  constexpr int kVectors = (Layer ? 2 : 1) * (Post ? 2 : 1);
  // weight, bias, block weight, block bias, as far as there are any
  constexpr int kWeight = 0, kBias = Layer, kBlockWeight = Post ? 1 + Layer : 0,
                kBlockBias = Layer && Post ? 3 : 0;
  __shared__ float2 place[2][16];
  __shared__ float joined[kTeams > 1 ? W * 64 * C * V : 1];
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid % (W * 64);
  const int64_t width = a.next.width;
  const float inverse = 1.0f / static_cast<float>(width);
  Team<W> team(place, wave);
  int64_t col[C];
  Pack<T, V> weight[C], block_weight[C], block_bias[C], gate[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (static_cast<int64_t>(c) * W * 64 + lane) * V;
    weight[c] = load_columns<V>(static_cast<const T*>(a.weight), col[c], width);
    if (Post) {
      block_weight[c] = load_columns<V>(static_cast<const T*>(a.block_weight), col[c], width);
      block_bias[c] = Pack<T, V>{};
      if (Layer && a.block_bias)
        block_bias[c] = load_columns<V>(static_cast<const T*>(a.block_bias), col[c], width);
    }
  }
  float sums[kVectors][C][V] = {}, gate_sum[C][V] = {};
  const bool block_there = a.block.data != nullptr, gated = a.gate != nullptr;
  constexpr int kFields = Post ? 4 : 2;

  const int64_t teams = static_cast<int64_t>(gridDim.x) * kTeams;
  const int64_t rounds = (a.items + teams - 1) / teams;
  const int64_t first_item = static_cast<int64_t>(blockIdx.x) * kTeams + wave / W;

  // row k of the team's item of a round; not live where there is none
  auto place_of = [&](int64_t round, int64_t k, bool& live) {
    const int64_t item = round * teams + first_item;
    const int64_t group = item / a.parts, part = item - group * a.parts;
    const int64_t in = part * a.item_rows + k;
    live = round < rounds && item < a.items && in < a.gate_rows && k < a.item_rows;
    return group * a.gate_rows + in;
  };
  auto fetch = [&](int64_t round, int64_t k, Row<T, C>& r) {
    const int64_t row = place_of(round, k, r.live);
    if (!r.live) return;
    const T* px = static_cast<const T*>(a.next.data) + row_start(a.next, row);
    const T* py = a.dout.data ? static_cast<const T*>(a.dout.data) + row_start(a.dout, row) : nullptr;
    const T* pn = a.dnext.data ? static_cast<const T*>(a.dnext.data) + row_start(a.dnext, row) : nullptr;
    const T* pb = block_there ? static_cast<const T*>(a.block.data) + row_start(a.block, row) : nullptr;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      r.x[c] = load_columns<V>(px, col[c], width);
      r.dy[c] = r.dx[c] = r.b[c] = Pack<T, V>{};
      if (py) r.dy[c] = load_columns<V>(py, col[c], width);
      if (pn) r.dx[c] = load_columns<V>(pn, col[c], width);
      if (pb) r.b[c] = load_columns<V>(pb, col[c], width);
    }
    const float* s = a.stats + row * kFields;
    r.mean = s[0];
    r.rstd = s[1];
    if (Post) {
      r.block_mean = s[2];
      r.block_rstd = s[3];
    }
  };

  Row<T, C> now, then;
  fetch(0, 0, then);
  for (int64_t round = 0; round < rounds; ++round) {
    const int64_t item = round * teams + first_item;
    const int64_t group = item / a.parts;
    if (gated && item < a.items) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        gate[c] = load_columns<V>(static_cast<const T*>(a.gate) + group * width, col[c], width);
    }
    for (int64_t k = 0; k < a.item_rows; ++k) {
      now = then;
      const bool last = k + 1 == a.item_rows;
      fetch(last ? round + 1 : round, last ? 0 : k + 1, then);
      bool live;
      const int64_t row = place_of(round, k, live);
      float2 s = make_float2(0.0f, 0.0f);
      if (live) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float v = (widen(now.x[c].v[e]) - now.mean) * now.rstd;
            const float t = widen(now.dy[c].v[e]) * widen(weight[c].v[e]);
            s.x = fmaf(t, v, s.x);
            s.y += t;
          }
      }
      s = team.sum(s, Layer);
      float d[C][V];
      float2 s2 = make_float2(0.0f, 0.0f);
      if (live) {
        const float along = s.x * inverse, level = Layer ? s.y * inverse : 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          Pack<T, V> o;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float v = (widen(now.x[c].v[e]) - now.mean) * now.rstd, g = widen(now.dy[c].v[e]);
            const float t = g * widen(weight[c].v[e]);
            sums[kWeight][c][e] = fmaf(g, v, sums[kWeight][c][e]);
            if (Layer) sums[kBias][c][e] += g;
            float r = fmaf(-v, along, t);
            if (Layer) r -= level;
            d[c][e] = fmaf(r, now.rstd, widen(now.dx[c].v[e]));
            o.v[e] = narrow<T>(d[c][e]);
          }
          store_columns<V>(static_cast<T*>(a.dresidual) + row * width, col[c], width, o);
        }
        if (block_there) {
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float q = d[c][e] * a.scale, u = widen(now.b[c].v[e]), w = 0.0f;
              if (Post) {
                w = (u - now.block_mean) * now.block_rstd;
                u = fmaf(w, widen(block_weight[c].v[e]), widen(block_bias[c].v[e]));
              }
              if (gated) {
                gate_sum[c][e] = fmaf(q, u, gate_sum[c][e]);
                q *= widen(gate[c].v[e]);
              }
              if (Post) {
                sums[kBlockWeight][c][e] = fmaf(q, w, sums[kBlockWeight][c][e]);
                if (Layer) sums[kBlockBias][c][e] += q;
                // (the weight is 0 behind the row's end)
                q *= widen(block_weight[c].v[e]);
                s2.x = fmaf(q, w, s2.x);
                s2.y += q;
              }
              d[c][e] = q;
            }
        }
      }
      if (Post) s2 = team.sum(s2, Layer);
      if (live && block_there) {
        const float along = s2.x * inverse, level = Layer ? s2.y * inverse : 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          Pack<T, V> o;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float q = d[c][e];
            if (Post) {
              const float w = (widen(now.b[c].v[e]) - now.block_mean) * now.block_rstd;
              q = fmaf(-w, along, q);
              if (Layer) q -= level;
              q *= now.block_rstd;
            }
            o.v[e] = narrow<T>(q);
          }
          store_columns<V>(static_cast<T*>(a.dblock) + row * width, col[c], width, o);
        }
      }
    }
    if (gated && item < a.items) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (a.gate_sums) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (col[c] + e < width) a.gate_sums[item * width + col[c] + e] = gate_sum[c][e];
        } else {
          Pack<T, V> o;
#pragma unroll
          for (int e = 0; e < V; ++e) o.v[e] = narrow<T>(gate_sum[c][e]);
          store_columns<V>(static_cast<T*>(a.dgate) + group * width, col[c], width, o);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) gate_sum[c][e] = 0.0f;
      }
    }
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
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float* p = &joined[(c * V + e) * W * 64 + lane];
            if (t > 0) sums[k][c][e] += *p;
            *p = sums[k][c][e];
          }
      }
    }
    if (which == kTeams - 1) {
      float* out = a.sums + (static_cast<int64_t>(blockIdx.x) * kVectors + k) * width;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (col[c] + e < width) out[col[c] + e] = sums[k][c][e];
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
  return layer ? launch(k_norm<T, W, C, true>, blocks, kWaves * 64, s, a)
               : launch(k_norm<T, W, C, false>, blocks, kWaves * 64, s, a);
}

// A wave to a row as long as it holds it in 64 bytes a lane, as no barrier is needed then.
template <typename T>
int choose_forward(const forward_args& a, bool layer, hipStream_t s) {
  const int64_t chunks = ceil_div(a.residual.width, 16 / static_cast<int>(sizeof(T)) * 64);
  if (chunks <= 1) return run_forward<T, 1, 1>(a, layer, s);
  if (chunks <= 2) return run_forward<T, 1, 2>(a, layer, s);
  if (chunks <= 4) return run_forward<T, 1, 4>(a, layer, s);
  if (chunks <= 8) return run_forward<T, 4, 2>(a, layer, s);
  if (chunks <= 16) return run_forward<T, 4, 4>(a, layer, s);
  if (chunks <= 32) return run_forward<T, 16, 2>(a, layer, s);
  return run_forward<T, 16, 4>(a, layer, s);
}

// How backward cuts the rows: teams of `waves`, `blocks` of them, items of a gate's rows.
struct Shares {
  int waves;
  int64_t blocks, parts, item_rows, items;
};

Shares shares_of(int64_t n, int64_t width, int64_t gates) {
  Shares s{};
  const int64_t chunks = ceil_div(width, kOwn * 64);
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
  const int64_t chunks = ceil_div(a.next.width, kOwn * 64);
  switch (sh.waves) {
    case 1: return run_backward<T, 1, 1>(a, layer, post, sh.blocks, s);
    case 2: return run_backward<T, 2, 1>(a, layer, post, sh.blocks, s);
    case 4: return run_backward<T, 4, 1>(a, layer, post, sh.blocks, s);
    case 8: return run_backward<T, 8, 1>(a, layer, post, sh.blocks, s);
  }
  if (chunks <= 16) return run_backward<T, 16, 1>(a, layer, post, sh.blocks, s);
  if (chunks <= 32) return run_backward<T, 16, 2>(a, layer, post, sh.blocks, s);
  return run_backward<T, 16, 4>(a, layer, post, sh.blocks, s);
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
  return grad_workspace(shares_of(n, width, gates), width, kind == MS_NORM_LAYER,
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
  const Shares sh = shares_of(n, width, gates);
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
