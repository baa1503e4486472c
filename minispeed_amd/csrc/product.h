// Matrix products with an epilogue of their own, for operators that use the
// product's values where they arise instead of storing them (linear.hip).
//
//   C[m, n] = sum over k of A[m, k] B[n, k],   elements of 2 (or 4) bytes, fp32 sums
//
// A block computes a tile of C; its waves hold it as 32 x 32 squares of matrix
// instructions (v_mfma_f32_32x32x16).  Of such a square a lane has one column
// n = lane % 32 and the rows m = 8 (i / 4) + 4 (lane / 32) + i % 4, i < 16: an
// epilogue that reduces over m stays within two lanes, and one that stores has four
// consecutive m of one n.
//
// Tiles of 64 k go from memory to LDS by loads that write LDS themselves, so that
// no register holds them; two of them take turns.  LDS is written in the order of the
// lanes, so each lane chooses which 16 bytes it fetches such that the reads of a
// fragment meet all banks:
//   along  k (rows of A or B lie along k): chunk c of row r lies at c ^ (r / 2 % 8);
//   across k (rows lie along m or n, one for each k): chunk c of row k at c ^ 4 (k % 4),
//            read by the transposing LDS load, 4 k of one m to a lane.
// Chunks beyond an operand's edge are fetched from beyond the buffer's range, which
// gives zeros.
//
// What bounds it: the matrix units, with the clock that their power leaves.  Of 16384 x 2048 x
// 4096 bf16 tiles of 256 x 256 make 1230 TFLOP/s where the library makes 1300, and across k on
// one side or both 1195; 128 x 128, two blocks to a CU, 1130.  Each wave has 128 x 64 of the tile:
// 6 fragment reads of LDS for 8 matrix instructions.  Fragments are read 16 k ahead of their
// use, and the one barrier for each tile lies between the last read and the last products.
// Tried and not kept: tiles of 32 k, five in LDS (1150), their loads spread between the
// products (1187); four waves of 128 x 128 (980); loads that the compiler knows of, which it
// waits for at the next read of LDS (across k on both sides 780).
#pragma once

#include "ops_common.h"

namespace ops {

constexpr int kStepBytes = 128;           // of k in one tile: 64 values of 2 bytes, 32 of 4
constexpr uint32_t kBeyond = 0x7f000000;  // an offset outside of every buffer
constexpr uint32_t kRange = 0x40000000;   // bytes that a tile's offsets stay within

enum Side { kAlong, kAcross };

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
#define MS_LDS __attribute__((address_space(3)))

template <typename T> struct frag_of;
template <> struct frag_of<f16> { typedef f16x8 type; };
template <> struct frag_of<bf16> { typedef bf16x8 type; };
template <> struct frag_of<float> { typedef f32x4 type; };

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// The instruction takes two k, one from each half of the wave: here value e of both halves' four.
__device__ __forceinline__ f32x16 mfma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// One operand: `rows` of m or n against k.  Along k: row r starts at r * ld, and ld and
// the address are multiples of 16 bytes.  Across k: k starts at k * ld, the same.
// A 32-bit operand is three planes of bf16 whose sum it is (plane: elements from one to
// the next); the product then runs over the six pairs of planes whose product is not
// below the last bit, as if k were six times as long.
struct operand {
  const void* data;
  int64_t ld;              // elements, as plane
  int64_t plane;
  int32_t rows;
};

struct product_args {
  operand a, b;
  int32_t k;
  int32_t pairs;                   // 1, or 6 pairs of planes
  int32_t tiles_m, tiles_n, splits;
};

// Which pair of planes: (0,0) (0,1) (1,0) (1,1) (0,2) (2,0), two bits each.
__device__ __forceinline__ int plane_a(int pair) { return 0x850 >> (2 * pair) & 3; }
__device__ __forceinline__ int plane_b(int pair) { return 0x244 >> (2 * pair) & 3; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes from each lane's offset to `to` + 16 lane in LDS.  In assembly, as the compiler
// would wait for it before the next read of LDS, of the other tile too; the wait is wait_loads().
// (An instruction between setting m0 and its use is required.  The compiler keeps nothing in m0
// and warns that it would not; the clobber orders the uses that it may make of it by itself.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, uint32_t offset, uint32_t to) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset),
      "s"(rsrc)
      : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// One operand's tile of R rows, fetched by NT threads.
template <typename T, int R, int NT, Side S>
struct Fetch {
  static constexpr int kIssues = R * kStepBytes / (NT * 16), kStep = kStepBytes / sizeof(T);
  static constexpr int V = 16 / sizeof(T);
  static constexpr int kChunks = R / V;              // across: 16-byte chunks of a row
  static constexpr int kRowsPer = S == kAlong ? NT / 8 : NT / kChunks;
  static constexpr int kTurn = sizeof(T) == 2 && kChunks >= 16 ? 3 : 0;
  static_assert(kIssues >= 1 && R * kStepBytes % (NT * 16) == 0, "");
  static_assert(S == kAlong ? kRowsPer % 16 == 0 : kRowsPer % 4 == 0, "");

  const char* base;
  int64_t ld_bytes;
  uint32_t offset[kIssues];
  int first_k;        // k of this thread's first chunk, within the tile

  __device__ Fetch(const operand& o, int row0, int tid) {
    ld_bytes = o.ld * static_cast<int64_t>(sizeof(T));
    if (S == kAlong) {
      base = reinterpret_cast<const char*>(o.data) + row0 * ld_bytes;
      const int r = tid >> 3, chunk = (tid & 7) ^ (r >> 1 & 7);
      first_k = chunk * V;
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int row = r + i * kRowsPer;
        offset[i] = row0 + row < o.rows
                        ? static_cast<uint32_t>(row * static_cast<int>(ld_bytes)) + chunk * 16
                        : kBeyond;
      }
    } else {
      base = reinterpret_cast<const char*>(o.data) + static_cast<int64_t>(row0) * sizeof(T);
      first_k = tid / kChunks;
      const int chunk = tid % kChunks ^ (first_k & kTurn) << 2;
#pragma unroll
      for (int i = 0; i < kIssues; ++i)
        offset[i] = row0 + chunk * V < o.rows
                        ? static_cast<uint32_t>((first_k + i * kRowsPer) * static_cast<int>(ld_bytes)) +
                              chunk * 16
                        : kBeyond;
    }
  }

  // The tile at k0 of plane `shift` elements further, into LDS at `to`; `left` is k - k0.
  __device__ void issue(int64_t shift, int k0, int left, uint32_t to, int wave) const {
    const char* p = base + shift * static_cast<int64_t>(sizeof(T)) +
                    (S == kAlong ? k0 * static_cast<int64_t>(sizeof(T)) : k0 * ld_bytes);
    const u32x4 rsrc = {static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)),
                        static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) >> 32) & 0xffff, kRange,
                        0x00027000};
    const uint32_t dst = to + wave * 1024;
    if (left >= kStep) {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) load_to_lds(rsrc, offset[i], dst + i * NT * 16);
    } else {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int k = S == kAlong ? first_k : first_k + i * kRowsPer;
        load_to_lds(rsrc, k < left ? offset[i] : kBeyond, dst + i * NT * 16);
      }
    }
  }
};

// Fragments of one operand: kept addresses of a lane, then one read for each square.
template <typename T, int R, Side S>
struct Frags {
  typedef typename frag_of<T>::type frag;
  uint32_t at[4];

  // first: the wave's first row of the tile.
  __device__ Frags(int first, int lane) {
    if (S == kAlong) {
      const int r = lane & 31;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        at[ks] = (first + r) * 128 + (((ks * 2 + (lane >> 5)) ^ (r >> 1 & 7)) << 4);
    } else if (sizeof(T) == 4) {
      // (a value of m for each lane, four k one after the other)
#pragma unroll
      for (int q = 0; q < 4; ++q) at[q] = (lane >> 5) * 4 * R * 4 + (first + q * 32 + (lane & 31)) * 4;
    } else {
      constexpr int kTurn = R / 8 >= 16 ? 3 : 0;
      const int k = (lane >> 5) * 8 + ((lane & 15) >> 2);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = first + q * 32 + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
        at[q] = k * R * 2 + (((m >> 3) ^ (k & kTurn) << 2) << 4) + (m & 7) * 2;
      }
    }
  }

  // Square q (32 rows further each), 32 bytes of k from 32 ks.
  __device__ frag read(const char MS_LDS* tile, int q, int ks) const {
    if (S == kAlong)
      return *reinterpret_cast<const frag MS_LDS*>(tile + at[ks] + q * 32 * 128);
    if constexpr (sizeof(T) == 4) {
      frag x;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = *reinterpret_cast<const float MS_LDS*>(tile + at[q & 3] + (ks * 8 + e) * R * 4);
      return x;
    } else {
      union { s16x4 half[2]; frag whole; } u;
      const char MS_LDS* p = tile + at[q & 3] + (q >> 2) * 256 + ks * 16 * R * 2;
      u.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<s16x4 MS_LDS*>(const_cast<char MS_LDS*>(p)));
      u.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<s16x4 MS_LDS*>(const_cast<char MS_LDS*>(p + 4 * R * 2)));
      return u.whole;
    }
  }
};

// Block b's place: neighbours in a tile order to one XCD (blocks go round the 8 XCDs),
// in that order bands of 8 columns of tiles, so that what runs at a time on an XCD shares
// its operands in the XCD's cache.
__device__ __forceinline__ void place(uint32_t b, uint32_t total, int tiles_m, int tiles_n,
                                      int& tm, int& tn, int& split) {
  const uint32_t q = total / 8, r = total % 8, x = b % 8;
  uint32_t t = x * q + min(x, r) + b / 8;
  const uint32_t each = static_cast<uint32_t>(tiles_m) * tiles_n;
  split = t / each;
  t -= split * each;
  const uint32_t band = t / (8 * tiles_m), first = band * 8;
  const uint32_t wide = min(8u, tiles_n - first);
  t -= first * tiles_m;
  tm = t / wide;
  tn = first + t % wide;
}

// A way to cut a product into tiles of BM x BN by WM x WN waves.
template <int BM_, int BN_, int WM_, int WN_>
struct Tiles {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kThreads = WM * WN * 64;
  static constexpr int kBytes = 2 * (BM + BN) * kStepBytes;     // of LDS
};

namespace {

// Block `block` of `blocks`: one tile, or one part of its k.
template <typename T, typename Tile, Side SA, Side SB, typename Epilogue>
__device__ __forceinline__ void multiply_tile(const product_args& p, const Epilogue& epilogue,
                                              uint32_t block, uint32_t blocks, char* memory) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host has none of the built-in functions)
  constexpr int BM = Tile::BM, BN = Tile::BN, WM = Tile::WM, WN = Tile::WN;
  constexpr int NT = Tile::kThreads, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int kStep = kStepBytes / sizeof(T);
  constexpr int kTileA = BM * kStepBytes, kTile = kTileA + BN * kStepBytes;
  static_assert(BM % (WM * 32) == 0 && BN % (WN * 32) == 0, "");
  char MS_LDS* const lds = (char MS_LDS*)memory;

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  int tm, tn, split;
  place(block, blocks, p.tiles_m, p.tiles_n, tm, tn, split);

  const Fetch<T, BM, NT, SA> fetch_a(p.a, tm * BM, tid);
  const Fetch<T, BN, NT, SB> fetch_b(p.b, tn * BN, tid);
  const Frags<T, BM, SA> frags_a(wm * MI * 32, lane);
  const Frags<T, BN, SB> frags_b(wn * NI * 32, lane);

  const int steps = (p.k + kStep - 1) / kStep;
  const int64_t all = static_cast<int64_t>(steps) * p.pairs;
  const int begin = static_cast<int>(all * split / p.splits);
  const int end = static_cast<int>(all * (split + 1) / p.splits);

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x16{};

  // Where no two blocks share a tile's rows, each begins elsewhere in k: in step they would
  // ask for the same columns of all rows at once, which lie in few of the memory's channels.
  const int turn = p.tiles_n == 1 ? tm % steps : 0;
  int pair = begin / steps, done = begin - pair * steps, k0 = (done + turn) % steps * kStep;
  auto issue = [&](int buffer) {
    const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + buffer * kTile;
    fetch_a.issue(plane_a(pair) * p.a.plane, k0, p.k - k0, to, wave);
    fetch_b.issue(plane_b(pair) * p.b.plane, k0, p.k - k0, to + kTileA, wave);
    k0 += kStep;
    if (k0 >= p.k) k0 = 0;
    if (++done == steps) done = 0, ++pair;
  };
  typedef typename frag_of<T>::type frag;
  frag a[2][MI], b[2][NI];
  auto read = [&](int buffer, int ks, int set) {
    const char MS_LDS* tile = lds + buffer * kTile;
#pragma unroll
    for (int i = 0; i < MI; ++i) a[set][i] = frags_a.read(tile, i, ks);
#pragma unroll
    for (int j = 0; j < NI; ++j) b[set][j] = frags_b.read(tile + kTileA, j, ks);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = mfma(a[set][i], b[set][j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };

  if (begin < end) {
    issue(0);
    wait_loads();
    __syncthreads();
    if (begin + 1 < end) issue(1);
    read(0, 0, 0);
  }
  for (int s = begin; s < end; ++s) {
    const int buffer = (s - begin) & 1;
#pragma unroll
    for (int ks = 0; ks < 3; ++ks) {
      read(buffer, ks + 1, (ks + 1) & 1);
      multiply(ks & 1);
    }
    // This tile's fragments are in registers and the next tile is in LDS, in all waves.  (The
    // barrier says nothing of memory to the compiler: nothing may be moved across it either way.)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 2 < end) issue(buffer);
    if (s + 1 < end) read(buffer ^ 1, 0, 0);
    multiply(1);
  }

  epilogue.template store<MI, NI>(acc, tm * BM + wm * MI * 32, tn * BN + wn * NI * 32,
                                  tm * WM + wm, split, lane, p.a.rows, p.b.rows);
#endif
}

template <typename T, typename Tile, Side SA, Side SB, typename Epilogue>
__global__ __launch_bounds__(Tile::kThreads, 2) void k_product(product_args p, Epilogue epilogue) {
  __shared__ __attribute__((aligned(1024))) char memory[Tile::kBytes];
  multiply_tile<T, Tile, SA, SB>(p, epilogue, blockIdx.x, gridDim.x, memory);
}

// Two products in one launch, the first `first` blocks and the others: so that the last
// tiles of the one do not leave CUs idle before the other begins.
template <typename T, typename Tile, Side SB1, Side SB2, typename Epilogue>
__global__ __launch_bounds__(Tile::kThreads, 2) void k_products(product_args p, Epilogue e,
                                                                product_args q, Epilogue f,
                                                                uint32_t first) {
  __shared__ __attribute__((aligned(1024))) char memory[Tile::kBytes];
  if (blockIdx.x < first)
    multiply_tile<T, Tile, kAcross, SB1>(p, e, blockIdx.x, first, memory);
  else
    multiply_tile<T, Tile, kAcross, SB2>(q, f, blockIdx.x - first, gridDim.x - first, memory);
}

}  // namespace
}  // namespace ops
