// Low-rank adapters of many requests beside one shared projection, for sm_100a:
//
//   h[t, s, r]  = sum_k x[t, k] A[a, s R + r, k]                      (shrink; a = the token's adapter, r < rank[a])
//   out[t, n]   = base[t, n] + scaling[a] sum_r h[t, s(n), r] B[a, n, r]        (expand; s(n) = the slice of column n)
//
// The plan groups the tokens by adapter (a stable counting sort), so that a tile of tokens shares one A and one B; it is made
// once for a batch of tokens and used by every projection of every layer.  Tiles have up to 16 tokens in small batches, where
// every adapter's weights are read for a few tokens each, and 128 in large ones.
//
// Both products are bound by memory: the shrink by x and A, the expand by base, out and B.  The large shrink, whose products
// would bind it on the older matrix instructions, runs on tcgen05 (lora_shrink_tiles_kernel).  The others use mma.m16n8k16; the
// order in which k is summed is free, so a lane's fragments of two consecutive k16 steps are one 16-byte vector (eight consecutive
// k) and nothing is transposed.  In small batches the weights are the 16-row operand and the tokens the 8-column one, so that a
// single token wastes no weight traffic.
//
// Sums are held in fp32.  h is rounded once, to the type of x, because the expand multiplies it with B on the tensor cores: half a
// step of h (2^-8 of it for bf16, 2^-11 for fp16) in the adapter's part of the sum; in fp16 an h beyond 65504 becomes infinite.
#include <cooperative_groups.h>

#include <atomic>

#include "gemm_common.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kSmallRows = 16, kLargeRows = 128;
// Rows of a tile: 128 from 256 tokens on, and 24 for every adapter that there may be.  K = 8192, qkv with R = 64, with 16 rows / 128:
// one adapter 128 tokens 17 / 20 us, 256 29 / 21; 8 adapters 128 tokens 17 / 21, 256 25 / 22; 32 adapters 512 tokens 52 / 68,
// 768 74 / 72.
__host__ __device__ inline int tile_rows(int64_t T, int64_t L) { return T >= 256 && T >= 24 * L ? kLargeRows : kSmallRows; }
constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr int kMaxAdapters = 1024;
constexpr int kMaxSlices = 8;
constexpr int64_t kMaxTokens = 1000000;     // max_tiles(kMaxTokens, kMaxAdapters) is a legal grid.y

__host__ __device__ inline int64_t max_tiles(int64_t T, int64_t L, int rows) { return T / rows + (L + 1 < T ? L + 1 : T); }
__host__ __device__ inline int64_t max_tiles(int64_t T, int64_t L) { return max_tiles(T, L, tile_rows(T, L)); }
// Device layout of a plan: int32 count[4] (tiles, -, -, -), int4 tiles[plan_tiles] (adapter or -1, first, rows, rank), int32 perm[T].
// The tiles have the room that small ones would need, so that a plan's size grows with every token and tells T: with the room
// of the tiles that there are, 212 tokens in tiles of 16 and 256 in tiles of 128 had plans of one size and different layouts.
__host__ __device__ inline int64_t plan_tiles(int64_t T, int64_t L) { return max_tiles(T, L, kSmallRows); }

struct PlanView {
  const int* count;
  const int4* tiles;
  const int* perm;
};
inline PlanView view_plan(const void* plan, int64_t T, int64_t L) {
  const char* b = static_cast<const char*>(plan);
  return {reinterpret_cast<const int*>(b), reinterpret_cast<const int4*>(b + 16),
          reinterpret_cast<const int*>(b + 16 + 16 * plan_tiles(T, L))};
}

// ------------------------------------------------------------------------------------------------------- plan
// One block.  Warp w owns the tokens [w * per, ...); bins [kPlanWarps][L + 1] in shared memory count its tokens per adapter
// (bin L: none), then hold where its next token of that adapter goes.  Stable: a token's place depends on nothing but the ids.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const int32_t* __restrict__ ids, int64_t T,
                                                                 const int32_t* __restrict__ ranks, int L, int rows,
                                                                 int* __restrict__ count, int4* __restrict__ tiles,
                                                                 int* __restrict__ perm) {
  pdl_start();
  extern __shared__ int sm[];
  const int E = L + 1;
  int* bins = sm;                       // [kPlanWarps][E]
  int* first = sm + kPlanWarps * E;     // [E + 1] first place of each adapter
  int* tile0 = first + E + 1;           // [E + 1] first tile of each adapter
  int* rank_of = tile0 + E + 1;         // [E]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < kPlanWarps * E; i += kPlanThreads) bins[i] = 0;
  for (int i = threadIdx.x; i < E; i += kPlanThreads) rank_of[i] = i < L ? max(__ldg(ranks + i), 0) : 0;
  __syncthreads();
  auto bin_of = [&](int64_t t) {
    const int a = __ldg(ids + t);
    return a >= 0 && a < L && rank_of[a] > 0 ? a : L;
  };
  const int64_t per = ((T + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t t0 = warp * per, t1 = t0 + per < T ? t0 + per : T;
  int* mine = bins + warp * E;
  for (int64_t t = t0; t < t1; t += 32) {
    const unsigned live = __ballot_sync(0xffffffffu, t + lane < t1);
    if (t + lane < t1) {
      const int a = bin_of(t + lane);
      const unsigned same = __match_any_sync(live, a);
      if (lane == __ffs(same) - 1) mine[a] += __popc(same);
    }
    __syncwarp();
  }
  __syncthreads();
  // per adapter: running sum over the warps, then over the adapters (by one warp)
  for (int a = threadIdx.x; a < E; a += kPlanThreads) {
    int run = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = bins[w * E + a];
      bins[w * E + a] = run;
      run += c;
    }
    first[a + 1] = run;
    tile0[a + 1] = (run + rows - 1) / rows;
  }
  __syncthreads();
  if (warp == 0) {
    int carry_f = 0, carry_t = 0;
    for (int base = 0; base < E; base += 32) {
      const bool in = base + lane < E;
      int f = in ? first[base + lane + 1] : 0, t = in ? tile0[base + lane + 1] : 0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int uf = __shfl_up_sync(0xffffffffu, f, off), ut = __shfl_up_sync(0xffffffffu, t, off);
        if (lane >= off) f += uf, t += ut;
      }
      if (in) first[base + lane + 1] = carry_f + f, tile0[base + lane + 1] = carry_t + t;
      carry_f += __shfl_sync(0xffffffffu, f, 31);
      carry_t += __shfl_sync(0xffffffffu, t, 31);
    }
    if (lane == 0) first[0] = 0, tile0[0] = 0, count[0] = carry_t;
  }
  __syncthreads();
  for (int64_t t = t0; t < t1; t += 32) {
    const unsigned live = __ballot_sync(0xffffffffu, t + lane < t1);
    if (t + lane < t1) {
      const int a = bin_of(t + lane);
      const unsigned same = __match_any_sync(live, a);
      const int place = first[a] + mine[a] + __popc(same & ((1u << lane) - 1));
      __syncwarp(live);
      if (lane == __ffs(same) - 1) mine[a] += __popc(same);
      perm[place] = static_cast<int>(t + lane);
    }
    __syncwarp();
  }
  for (int a = threadIdx.x; a < E; a += kPlanThreads)
    for (int i = tile0[a]; i < tile0[a + 1]; ++i) {
      const int at = first[a] + (i - tile0[a]) * rows;
      tiles[i] = make_int4(a < L ? a : -1, at, min(rows, first[a + 1] - at), rank_of[a]);
    }
}

// --------------------------------------------------------------------------------------------------- fragments
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 consecutive k at once: lo and hi are the 16-byte vectors (k = 8c .. 8c + 7, c = lane % 4) of rows lane / 4 and lane / 4 + 8
// of the 16-row operand, x the one of row lane / 4 of the other.
template <typename T>
__device__ __forceinline__ void mma_k32(float (&d)[4], const uint4& lo, const uint4& hi, const uint4& x) {
  mma16816<T>(d, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
  mma16816<T>(d, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
}
__device__ __forceinline__ uint4 load_if(bool p, const void* ptr) {
  return p ? __ldg(static_cast<const uint4*>(ptr)) : make_uint4(0, 0, 0, 0);
}
// Of a vector of eight elements only the first `keep` stay, the others become zero (an adapter's rank may end inside it).
__device__ __forceinline__ uint4 first_of(uint4 v, int keep) {
  uint32_t* w = &v.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] &= keep >= 2 * i + 2 ? 0xffffffffu : keep == 2 * i + 1 ? 0x0000ffffu : 0u;
  return v;
}

// ------------------------------------------------------------------------------------------------------- shrink
constexpr int kShrinkThreads = 128, kShrinkWarps = kShrinkThreads / 32;
template <int Z>
struct Shrink {
  static constexpr int kStages = Z == 1 ? 5 : 4, kStageBytes = (2 * Z + 2) * 512;
  static constexpr int kSmem = kShrinkWarps * kStages * kStageBytes;
};

// A cluster of up to eight blocks computes Z groups of 16 columns of h for one tile of up to 16 tokens, all its warps dividing K; the partial
// sums are added in a fixed order, first over a block's warps, then over the blocks through distributed shared memory.  A warp's
// operands come through a ring of k32 steps in shared memory in which each lane has its own place (nothing to synchronise):
// with loads into registers instead, 128 tokens of 32 adapters over K = 8192 and three slices of 64 took 25.6 us.
template <typename T, int Z>
__global__ void __launch_bounds__(kShrinkThreads) lora_shrink_kernel(const T* __restrict__ x, int64_t x_ld, const T* __restrict__ A,
                                                                     int64_t K, int R, int cols, PlanView plan,
                                                                     T* __restrict__ h, int64_t h_ld) {
  using S = Shrink<Z>;
  pdl_start();
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float part[kShrinkWarps][Z * 256];
  __shared__ float mine[Z * 256];
  const int tiles = plan.count[0];
  const int4 tile = plan.tiles[blockIdx.y];                          // in bounds whether or not it is one
  if (static_cast<int>(blockIdx.y) >= tiles) return;                 // the whole cluster leaves together, here and below
  const int splits = gridDim.x, c0 = blockIdx.z * (Z * 16);
  const int rows = tile.z, rank = tile.x < 0 ? 0 : min(tile.w, R);
  bool any = false;
#pragma unroll
  for (int i = c0; i < c0 + Z * 16; i += 8) any |= i < cols && i % R < rank;
  if (!any) {                                                        // behind the rank (R % 8 == 0), or no adapter: zeros
    if (blockIdx.x == 0)
      for (int e = threadIdx.x; e < Z * 256; e += kShrinkThreads) {
        const int row = e / 16 % 16, col = c0 + e / 256 * 16 + e % 16;
        if (row < rows && col < cols) h[static_cast<int64_t>(plan.perm[tile.y + row]) * h_ld + col] = static_cast<T>(0.f);
      }
    return;
  }
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int r0 = __ldg(plan.perm + tile.y + min(g, rows - 1)), r1 = __ldg(plan.perm + tile.y + min(g + 8, rows - 1));
  const int chunks = static_cast<int>((K + 31) / 32), per = (chunks + splits * kShrinkWarps - 1) / (splits * kShrinkWarps);
  const int begin = (blockIdx.x * kShrinkWarps + warp) * per, end = min(begin + per, chunks);
  // this lane's operands: rows lane / 4 and lane / 4 + 8 of A (of each group) and of x; absent ones are zero-filled copies of nothing
  const char* src[2 * Z + 2];
  bool there[2 * Z + 2];
#pragma unroll
  for (int i = 0; i < 2 * Z + 2; ++i) {
    const int row = g + 8 * (i % 2), col = c0 + i / 2 * 16 + row;
    const bool in = i < 2 * Z ? col < cols && col % R < rank : row < rows;
    const T* p = i < 2 * Z ? A + (static_cast<int64_t>(tile.x) * cols + col) * K : x + (i % 2 == 0 ? r0 : r1) * x_ld;
    src[i] = reinterpret_cast<const char*>(in ? p + static_cast<int64_t>(begin) * 32 + 8 * c : A);
    there[i] = in;
  }
  const bool both = rows > 8;
  float acc[Z][2][4] = {};
  const uint32_t ring = smem_u32(dyn) + warp * (S::kStages * S::kStageBytes) + lane * 16, ring_end = ring + S::kStages * S::kStageBytes;
  const int ragged = K % 32 != 0 && 8 * c >= K % 32 ? chunks - 1 : -1;       // the step of which this lane has nothing
  uint32_t to = ring, from = ring;
  auto fetch = [&](int i) {                                          // a stage: [A lo, A hi (of each group), x lo, x hi][lane]
    if (i == ragged) {
#pragma unroll
      for (int j = 0; j < 2 * Z + 2; ++j) there[j] = false, src[j] = reinterpret_cast<const char*>(A);
    }
#pragma unroll
    for (int j = 0; j < 2 * Z + 2; ++j) {
      if (j < 2 * Z + 1 || both) sa::cp_async_or_zero<16>(to + 512 * j, src[j], there[j]);
      src[j] += 64;
    }
    to = to + S::kStageBytes == ring_end ? ring : to + S::kStageBytes;
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (begin + i < end) fetch(begin + i);
    sa::cp_async_commit();
  }
#pragma unroll 2
  for (int i = begin; i < end; ++i) {
    if (i + S::kStages - 1 < end) fetch(i + S::kStages - 1);
    sa::cp_async_commit();
    sa::cp_async_wait<S::kStages - 1>();
    __syncwarp();
    const uint4 x0 = sa::ld_v4(from + 2 * Z * 512);
    uint4 x1 = make_uint4(0, 0, 0, 0);
    if (both) x1 = sa::ld_v4(from + (2 * Z + 1) * 512);
#pragma unroll
    for (int z = 0; z < Z; ++z) {
      const uint4 lo = sa::ld_v4(from + 2 * z * 512), hi = sa::ld_v4(from + (2 * z + 1) * 512);
      mma_k32<T>(acc[z][0], lo, hi, x0);
      if (both) mma_k32<T>(acc[z][1], lo, hi, x1);
    }
    from = from + S::kStageBytes == ring_end ? ring : from + S::kStageBytes;
  }
  // part[warp][group][token][column]
#pragma unroll
  for (int z = 0; z < Z; ++z)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][z * 256 + (8 * i + 2 * c + (j & 1)) * 16 + g + 8 * (j >> 1)] = acc[z][i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < Z * 256; e += kShrinkThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kShrinkWarps; ++w) sum += part[w][e];
    mine[e] = sum;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (splits > 1) cluster.sync();
  const int share = Z * 256 / splits;                                // one block: each thread reads what it has written
  for (int i = threadIdx.x; i < share; i += kShrinkThreads) {
    const int e = static_cast<int>(blockIdx.x) * share + i, row = e / 16 % 16, col = c0 + e / 256 * 16 + e % 16;
    float sum = 0.f;
    if (splits == 1) {
      sum = mine[e];
    } else {
#pragma unroll 8
      for (int b = 0; b < splits; ++b) sum += *cluster.map_shared_rank(mine + e, b);
    }
    if (row < rows && col < cols)
      h[static_cast<int64_t>(plan.perm[tile.y + row]) * h_ld + col] = static_cast<T>(col % R < rank ? sum : 0.f);
  }
  if (splits > 1) cluster.sync();
}

// A cluster of `splits` blocks computes up to n_alloc columns of h for one tile of up to 128 tokens, each block a part of K.
// tcgen05: D [128 tokens x columns] += x [128 x 64] A^T [64 x columns], both operands K-major in shared memory with the
// 128-byte swizzle.  Warps 0 and 2 fetch half of the tile's x each, with one TMA box where its tokens are neighbours, else with
// smaller ones or gathered four by four; warp 3 fetches the rows of A below the adapter's rank, box by box, the slices packed
// one behind the other; warp 1 issues the products.  Then all four warps read the sums out of tensor memory and, with several
// blocks, add them in block order through distributed shared memory.  The number of TMA instructions counts: with one warp
// issuing forty boxes of eight rows per k-block, a k-block took 2.2 us (8191 x 8192 and 192 columns: 141 us; rows copied by all
// threads with 16-byte asynchronous copies: 174 us; four warps with boxes of 32 rows: 45 us, two with 64: 38).
constexpr int kTileThreads = 128, kTileSmem = 201 * 1024, kBlockK = 64, kMaxTileStages = 8, kMaxColumns = 256;
constexpr uint32_t kXBytes = kLargeRows * kBlockK * 2;

struct ShrinkMaps {
  CUtensorMap x[5], a, a_whole;        // x in boxes of 1, 8, 16, 32 and 64 rows; A in boxes of a_box rows, and of an adapter's all
};
struct ShrinkTiles {
  int64_t K, h_ld;
  int R, slices, n_alloc, splits, stages, a_box;
  bool a_whole;
  int* status;
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status, int code) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = sa::wait(bar, parity, status, code);
  return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n) {   // fp32 sums; both operands K-major, bf16 (1) or fp16 (0)
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((kLargeRows >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads) lora_shrink_tiles_kernel(const __grid_constant__ ShrinkMaps maps,
                                                                         PlanView plan, T* __restrict__ h,
                                                                         const __grid_constant__ ShrinkTiles p) {
  pdl_wait();
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxTileStages + 1];
  __shared__ uint32_t tmem_slot;
  const int tiles = plan.count[0];
  const int4 tile = plan.tiles[blockIdx.y];                     // in bounds whether or not it is one
  if (static_cast<int>(blockIdx.y) >= tiles) return;            // the whole cluster leaves together, here and below
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rows = tile.z, split = blockIdx.x;
  const int rank = tile.x < 0 ? 0 : min(tile.w, p.R), width = (rank + p.a_box - 1) / p.a_box * p.a_box;    // of a slice
  const int c0 = blockIdx.z * p.n_alloc, n = min(p.slices * width - c0, p.n_alloc);      // packed columns of this block
  if (blockIdx.z == 0 && split == 0) {                          // zeros behind the rank, 16 bytes at a time
    const int vecs = (p.R - width) / 8, all = rows * p.slices * vecs;
    for (int e = threadIdx.x; e < all; e += kTileThreads) {
      const int v = e % vecs, s = e / vecs % p.slices, r = e / vecs / p.slices;
      *reinterpret_cast<uint4*>(h + plan.perm[tile.y + r] * p.h_ld + s * p.R + width + 8 * v) = make_uint4(0, 0, 0, 0);
    }
  }
  if (n <= 0) return;
  const int n16 = (n + 15) / 16 * 16;
  const uint32_t ring = (smem_u32(dyn) + 1023u) & ~1023u, stage_bytes = kXBytes + p.n_alloc * (kBlockK * 2);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxTileStages, done = empty + 8 * kMaxTileStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      sa::init(full + 8 * i, 3);
      sa::init(empty + 8 * i, 1);
    }
    sa::init(done, 1);
    fence_mbar_init();
  }
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(n16)) tmem_cols *= 2;
  if (warp == 1) {
    tmem_alloc(&tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before every block of this kernel that goes on has its tensor memory: a following kernel that takes all of it and then
  // waits for this one would otherwise be waited for.
  pdl_trigger();
  const uint32_t tmem = tmem_slot;
  const int64_t nkb = (p.K + kBlockK - 1) / kBlockK;
  const int kb0 = static_cast<int>(nkb * split / p.splits), count = static_cast<int>(nkb * (split + 1) / p.splits) - kb0;
  bool ok = true;
  if (warp != 1) {
    // x: 64 of the tile's rows, lanes 0-7 with eight each (tokens are in ascending order, so the ends of a run tell whether it has
    // gaps; rows behind the tile's last are any rows, their sums are not used).  The largest boxes that have none are taken: box is
    // the number of rows that this lane fetches in one, 4 for two gathers, 0 if an earlier lane has its rows.
    const int half = 64 * (warp / 2), first = half + 8 * (lane % 8);
    int y[8], box = 0;
    if (warp != 3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __ldg(plan.perm + tile.y + min(first + i, rows - 1));
      box = y[7] - y[0] == min(first + 7, rows - 1) - min(first, rows - 1) ? 8 : 4;
#pragma unroll
      for (int size = 16; size <= 64; size *= 2) {
        const int lanes = size / 8, from = lane % 8 / lanes * lanes, begin = half + 8 * from;
        const int y0 = __shfl_sync(0xffffffffu, y[0], from), y1 = __shfl_sync(0xffffffffu, y[7], from + lanes - 1);
        if (y1 - y0 == min(begin + size - 1, rows - 1) - min(begin, rows - 1)) box = lane % 8 == from ? size : 0;
      }
      if (lane >= 8) box = 0;
    }
    // A: lane by lane one box, or one for all of it where the adapter has the full rank
    const bool whole = p.a_whole && rank == p.R;
    const int boxes = whole ? 1 : n / p.a_box, j = c0 + lane * p.a_box;
    const int ay = warp == 3 && lane < boxes ? tile.x * p.slices * p.R + j / width * p.R + j % width : 0;
    const uint32_t bytes = warp == 3 ? n * (kBlockK * 2) : kXBytes / 2;
    int stage = 0, phase = 1;
    for (int i = 0; i < count; ++i) {
      ok = warp_wait(empty + 8 * stage, phase, p.status, 51);
      if (!ok) {                                                // let what is under way land before shared memory is given up
        for (int b = 0; b < min(i, p.stages); ++b) {
          if (stage-- == 0) stage = p.stages - 1, phase ^= 1;
          warp_wait(full + 8 * stage, phase ^ 1, p.status, 54);
        }
        break;
      }
      const uint32_t bar = full + 8 * stage, to = ring + stage * stage_bytes + (warp == 3 ? kXBytes : half * 128);
      const int k = (kb0 + i) * kBlockK;
      if (lane == 0) sa::expect_tx(bar, bytes);
      __syncwarp();
      if (warp == 3) {
        if (lane < boxes) sa::tma_load_2d(to + lane * p.a_box * 128, whole ? &maps.a_whole : &maps.a, bar, k, ay);
      } else if (box == 4) {
        sa::tma_gather4(to + lane * 1024, &maps.x[0], bar, k, y[0], y[1], y[2], y[3]);
        sa::tma_gather4(to + lane * 1024 + 512, &maps.x[0], bar, k, y[4], y[5], y[6], y[7]);
      } else if (box != 0) {
        sa::tma_load_2d(to + lane * 1024, box == 64 ? &maps.x[4] : box == 32 ? &maps.x[3] : box == 16 ? &maps.x[2] : &maps.x[1], bar, k, y[0]);
      }
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
  } else {
    const uint32_t idesc = idesc_f16<T>(n16);
    for (int i = 0, stage = 0, phase = 0; i < count; ++i) {
      ok = warp_wait(full + 8 * stage, phase, p.status, 52);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t xs = ring + stage * stage_bytes;
        const uint64_t xd = umma_desc_k128(xs), ad = umma_desc_k128(xs + kXBytes);
#pragma unroll
        for (int k = 0; k < kBlockK / 16; ++k) umma_f16(tmem, xd + 2 * k, ad + 2 * k, idesc, i > 0 || k > 0);
        sa::commit(empty + 8 * stage);
        if (i + 1 == count) sa::commit(done);
      }
      __syncwarp();
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
  }
  if (ok) ok = warp_wait(done, 0, p.status, 53);
  tc_fence_after();
  const uint32_t mine = tmem + (static_cast<uint32_t>(warp * 32) << 16);         // this thread's row of the sums
  const int row = threadIdx.x;
  // Each block of the cluster adds up a share of the columns, in groups of eight: the others' sums of them arrive in its shared
  // memory, where the ring was, as [block][column][row].
  const int groups = n / 8, share = (groups + p.splits - 1) / p.splits;
  const int g0 = split * share, g1 = min(g0 + share, groups);
  float* recv = reinterpret_cast<float*>(dyn + (ring - smem_u32(dyn))) + row;
  if (p.splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                             // nobody's ring is in use any more
    for (int b = 1; b < p.splits; ++b) {
      const int to = (split + b) % p.splits;
      float* theirs = cluster.map_shared_rank(recv, to) + split * share * (8 * kLargeRows);
      for (int q = to * share; q < min(to * share + share, groups); ++q) {
        float v[8];
        tmem_ld8(mine + 8 * q, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i) theirs[((q - to * share) * 8 + i) * kLargeRows] = v[i];
      }
    }
    cluster.sync();
  }
  const int64_t token = row < rows ? plan.perm[tile.y + row] : -1;
  int s = (c0 + 8 * g0) / width, r = (c0 + 8 * g0) % width;
  for (int q = g0; q < g1; ++q) {
    float v[8];
    tmem_ld8(mine + 8 * q, v);
    tmem_ld_wait();
    // in the order of the blocks, whoever adds
    if (p.splits > 1) {
      float sum[8] = {};
      for (int b = 0; b < p.splits; ++b) {
        const float* part = recv + (b * share + q - g0) * (8 * kLargeRows);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += b == split ? v[i] : part[i * kLargeRows];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = sum[i];
    }
    if (ok && token >= 0) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = pack2(static_cast<T*>(nullptr), r + 2 * i < rank ? v[2 * i] : 0.f, r + 2 * i + 1 < rank ? v[2 * i + 1] : 0.f);
      *reinterpret_cast<uint4*>(h + token * p.h_ld + s * p.R + r) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if ((r += 8) == width) r = 0, ++s;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------------------------------------------- expand
struct Slices {
  int n, first_col[kMaxSlices + 1], first_block[kMaxSlices + 1];     // columns; blocks of the columns of a warp
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
constexpr int kExpandThreads = 128;

// A warp takes `per` neighbouring blocks of 64 columns (each within a slice) for one tile of up to 16 tokens.  Weight row (tile i,
// half f, lane / 4) of its four 16-row operands is column 8 (lane / 4) + 2 i + f, so that the eight sums that a lane holds for a
// token are neighbours: base and out move 16 bytes at a time.  B comes through a ring of (block, 32 ranks) steps in shared memory in
// which each lane has its own places; base and h go straight into registers.  What bounds it is how many warps fit: with base and
// h in a ring of three steps, 8 warps an SM, 128 tokens of 32 adapters (ranks 16 to 64, N = 10240) took 12.3 us, now 9.6; with
// three steps and 16 warps 9.7, with two and 20 warps, whose registers spill, 10.3.
// early: the shrink before it is this library's own, launched in the same call, and triggered after its wait; what was there
// before the shrink (the plan, B and base) may then be read ahead of the wait, which only h has to be behind.
constexpr int kExpandStages = 2, kExpandStageBytes = 8 * 512;
constexpr int kExpandSmem = kExpandThreads / 32 * kExpandStages * kExpandStageBytes;

template <typename T>
__global__ void __launch_bounds__(kExpandThreads, 4) lora_expand_kernel(const T* h, int h_ld, const T* __restrict__ B, int64_t N, int R,
                                                                     const float* __restrict__ scalings, PlanView plan,
                                                                     const __grid_constant__ Slices sl, const T* base, int base_ld,
                                                                     T* out, int out_ld, int per, bool early) {
  if (!early) pdl_wait();
  extern __shared__ __align__(128) uint8_t dyn[];
  const int tiles = plan.count[0];
  const int4 tile = plan.tiles[blockIdx.y];                  // in bounds whether or not it is one
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int first = (blockIdx.x * (kExpandThreads / 32) + warp) * per, blocks = min(per, sl.first_block[sl.n] - first);
  const int rows = tile.z;
  const bool none = tile.x < 0;
  if (static_cast<int>(blockIdx.y) >= tiles || blocks <= 0 || (none && base == out)) {
    if (early) pdl_wait();                                   // no block ends before the shrink has: what follows relies on it
    return;
  }
  const bool both = rows > 8;
  const int* perm = plan.perm + tile.y;
  const int h_row[2] = {__ldg(perm + min(g, rows - 1)), __ldg(perm + min(g + 8, rows - 1))};
  int token[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) token[i] = __ldg(perm + min(8 * (i / 2) + 2 * c + i % 2, rows - 1));
  const int rank = none ? 0 : min(tile.w, R), chunks = max(1, (rank + 31) / 32), steps = blocks * chunks;
  const float scaling = none ? 0.f : __ldg(scalings + tile.x);
  const uint32_t ring = smem_u32(dyn) + warp * (kExpandStages * kExpandStageBytes) + lane * 16;
  // Where a walk over the steps (block, 32 ranks) stands: once for the copies, once for the products.
  struct At {
    int block, j, s, n;
    bool live;
    uint32_t place;
  };
  auto enter = [&](At& p) {                                  // slice and first column (of this lane's eight) of its block
    while (p.s + 1 < sl.n && p.block >= sl.first_block[p.s + 1]) ++p.s;
    p.n = sl.first_col[p.s] + (p.block - sl.first_block[p.s]) * 64 + 8 * g;
    p.live = p.n < sl.first_col[p.s + 1];
  };
  auto advance = [&](At& p) {
    p.place = p.place + kExpandStageBytes == ring + kExpandStages * kExpandStageBytes ? ring : p.place + kExpandStageBytes;
    if (++p.j == chunks) {
      p.j = 0;
      ++p.block;
      enter(p);
    }
  };
  At in_flight = {first, 0, 0, 0, false, ring}, at = in_flight;
  enter(in_flight);
  at = in_flight;
  const int64_t row_bytes = static_cast<int64_t>(R) * sizeof(T);
  const char* b0 = reinterpret_cast<const char*>(B + static_cast<int64_t>(none ? 0 : tile.x) * N * R + 8 * c);
  auto fetch_weights = [&](const At& p) {
    const bool in = p.live && rank - 32 * p.j - 8 * c > 0;
    const char* src = in ? b0 + p.n * row_bytes + p.j * (32 * sizeof(T)) : b0 - 8 * c * sizeof(T);
    const uint32_t ld = static_cast<uint32_t>(row_bytes);
#pragma unroll
    for (int i = 0; i < 8; ++i) sa::cp_async_or_zero<16>(p.place + i * 512, src + i * ld, in);
  };
  uint4 v[4];                                                // base, of a block ahead
  auto fetch_base = [&](const At& p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = make_uint4(0, 0, 0, 0);
      if (base != nullptr && p.live && 8 * (i / 2) + 2 * c + i % 2 < rows)
        v[i] = *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(token[i]) * base_ld + p.n);
    }
  };
  const T* h0[2] = {h + static_cast<int64_t>(h_row[0]) * h_ld + 8 * c, h + static_cast<int64_t>(h_row[1]) * h_ld + 8 * c};
  uint4 hv[2];
  auto fetch_h = [&](const At& p) {
    const bool in = rank - 32 * p.j - 8 * c > 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      hv[i] = make_uint4(0, 0, 0, 0);
      if (in && g + 8 * i < rows) hv[i] = *reinterpret_cast<const uint4*>(h0[i] + p.s * R + 32 * p.j);
    }
  };
  static_assert(kExpandStages == 2, "one step is fetched ahead");
  fetch_weights(in_flight);
  sa::cp_async_commit();
  fetch_base(at);
  if (early) pdl_wait();
  pdl_trigger();
  fetch_h(at);
  float acc[2][4][4];
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    if (step + kExpandStages - 1 < steps) {
      advance(in_flight);
      fetch_weights(in_flight);
    }
    sa::cp_async_commit();
    sa::cp_async_wait<kExpandStages - 1>();
    __syncwarp();                                            // lanes that stored come back to those that had nothing to store
    const uint32_t from = at.place;
    const int j = at.j;
    if (j == 0) {
#pragma unroll
      for (int m = 0; m < 32; ++m) acc[m / 16][m / 4 % 4][m % 4] = 0.f;
    }
    if (!none) {
      const int keep = rank - 32 * j - 8 * c;
      // Zeros of B alone would not do: h may be NaN behind the rank.  Here and not behind its load, which would be waited for.
      if (keep > 0 && keep < 8) hv[0] = first_of(hv[0], keep), hv[1] = first_of(hv[1], keep);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 lo = sa::ld_v4(from + 2 * i * 512), hi = sa::ld_v4(from + (2 * i + 1) * 512);
        if (keep > 0 && keep < 8) lo = first_of(lo, keep), hi = first_of(hi, keep);
        mma_k32<T>(acc[0][i], lo, hi, hv[0]);
        if (both) mma_k32<T>(acc[1][i], lo, hi, hv[1]);
      }
    }
    const At old = at;
    advance(at);
    if (step + 1 < steps && (at.j != old.j || at.s != old.s)) fetch_h(at);
    if (j + 1 < chunks) continue;
    if (old.live) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (8 * (i / 2) + 2 * c + i % 2 >= rows) continue;
        if (!none) {
          uint32_t* q = &v[i].x;
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 b = unpack2<T>(q[m]);
            q[m] = pack2(static_cast<T*>(nullptr), fmaf(scaling, acc[i / 2][m][i % 2], b.x), fmaf(scaling, acc[i / 2][m][i % 2 + 2], b.y));
          }
        }
        *reinterpret_cast<uint4*>(out + static_cast<int64_t>(token[i]) * out_ld + old.n) = v[i];
      }
    }
    if (step + 1 < steps) fetch_base(at);
  }
}

// A handful of tokens and a small rank: both products in one launch.  A cluster of eight blocks computes all of a tile's h -- up to
// 16 Z columns, K divided among its 32 warps, added up in the order of the separate kernels -- and every warp then expands one
// block of 64 columns.  Clusters of the same tile repeat the shrink out of L2, which up to 32 columns costs less than a second
// launch and h's way through memory: 1 token, K = N = 8192, rank 16 takes 5.0 us against 5.4, and the host one launch less (2.5 us).
// With 48 or 64 columns it does not pay (7.6 and 8.2 against 5.7 and 5.9), nor with many clusters (18 for N = 36864: 6.6 against
// 5.6; 17 tiles of four: 11.8 against 9.0).  B and base are fetched first and arrive under the shrink.
constexpr int kFusedThreads = 128, kFusedWarps = kFusedThreads / 32, kFusedCluster = 8, kFusedColumns = 32;
constexpr int64_t kFusedParts = 8, kFusedClusters = 36;
template <int Z>
struct Fused {
  static constexpr int kStages = Z == 1 ? 5 : 3, kStageBytes = (2 * Z + 2) * 512;
  static constexpr int kOwn = 12 * 512;                              // a warp's B and base
  static constexpr int kRing = kFusedWarps * kStages * kStageBytes, kSmem = kRing + kFusedWarps * kOwn;
};

template <typename T, int Z>
__global__ void __launch_bounds__(kFusedThreads) lora_fused_kernel(const T* __restrict__ x, int64_t x_ld, const T* __restrict__ A,
                                                                   const T* __restrict__ B, int64_t K, int64_t N, int R, int cols,
                                                                   const float* __restrict__ scalings, PlanView plan,
                                                                   const __grid_constant__ Slices sl, const T* base, int base_ld,
                                                                   T* out, int out_ld) {
  using F = Fused<Z>;
  pdl_start();
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float part[kFusedWarps][Z * 256], mine[Z * 256];
  __shared__ __align__(16) T hs[16][Z * 16 + 8];                     // padded: eight rows' vectors lie in different banks
  const int tiles = plan.count[0];
  const int4 tile = plan.tiles[blockIdx.y];                          // in bounds whether or not it is one
  if (static_cast<int>(blockIdx.y) >= tiles) return;                 // the whole cluster leaves together, here and below
  const bool none = tile.x < 0;
  if (none && base == out) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int rows = tile.z, rank = none ? 0 : min(tile.w, R);
  const bool both = rows > 8;
  const int* perm = plan.perm + tile.y;
  // ---- this warp's 64 columns: B and base
  const int block = (blockIdx.z * kFusedCluster + blockIdx.x) * kFusedWarps + warp;
  const bool busy = block < sl.first_block[sl.n];
  int s = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i) s += i < sl.n && block >= sl.first_block[i];
  const int n = busy ? sl.first_col[s] + (block - sl.first_block[s]) * 64 + 8 * g : 0;      // the first of this lane's eight columns
  const bool live = busy && n < sl.first_col[s + 1];
  int token[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) token[i] = __ldg(perm + min(8 * (i / 2) + 2 * c + i % 2, rows - 1));
  const uint32_t own = smem_u32(dyn) + F::kRing + warp * F::kOwn + lane * 16;
  const bool some = live && rank - 8 * c > 0;                        // of the at most 32 ranks
  const T* bp = some ? B + (static_cast<int64_t>(tile.x) * N + n) * R + 8 * c : B;
#pragma unroll
  for (int i = 0; i < 8; ++i) sa::cp_async_or_zero<16>(own + i * 512, some ? bp + i * R : B, some);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = base != nullptr && live && 8 * (i / 2) + 2 * c + i % 2 < rows;
    sa::cp_async_or_zero<16>(own + (8 + i) * 512, in ? base + static_cast<int64_t>(token[i]) * base_ld + n : B, in);
  }
  sa::cp_async_commit();
  // ---- shrink
  const int r0 = __ldg(perm + min(g, rows - 1)), r1 = __ldg(perm + min(g + 8, rows - 1));
  constexpr int kAll = kFusedCluster * kFusedWarps;
  const int chunks = none ? 0 : static_cast<int>((K + 31) / 32), per = (chunks + kAll - 1) / kAll;
  const int begin = (blockIdx.x * kFusedWarps + warp) * per, end = min(begin + per, chunks);
  const char* src[2 * Z + 2];
  bool there[2 * Z + 2];
#pragma unroll
  for (int i = 0; i < 2 * Z + 2; ++i) {
    const int col = i < 2 * Z ? g + 8 * i : 0, row = i < 2 * Z ? 0 : g + 8 * (i - 2 * Z);
    const bool in = i < 2 * Z ? col < cols && col % R < rank : row < rows;
    const T* p = i < 2 * Z ? A + (static_cast<int64_t>(none ? 0 : tile.x) * cols + col) * K : x + (i == 2 * Z ? r0 : r1) * x_ld;
    src[i] = reinterpret_cast<const char*>(in ? p + static_cast<int64_t>(begin) * 32 + 8 * c : A);
    there[i] = in;
  }
  float acc[Z][2][4] = {};
  const uint32_t ring = smem_u32(dyn) + warp * (F::kStages * F::kStageBytes) + lane * 16, ring_end = ring + F::kStages * F::kStageBytes;
  const int ragged = K % 32 != 0 && 8 * c >= K % 32 ? chunks - 1 : -1;       // the step of which this lane has nothing
  uint32_t to = ring, from = ring;
  auto fetch = [&](int i) {
    if (i == ragged) {
#pragma unroll
      for (int j = 0; j < 2 * Z + 2; ++j) there[j] = false, src[j] = reinterpret_cast<const char*>(A);
    }
#pragma unroll
    for (int j = 0; j < 2 * Z + 2; ++j) {
      if (j < 2 * Z + 1 || both) sa::cp_async_or_zero<16>(to + 512 * j, src[j], there[j]);
      src[j] += 64;
    }
    to = to + F::kStageBytes == ring_end ? ring : to + F::kStageBytes;
  };
#pragma unroll 1
  for (int i = 0; i < F::kStages - 1; ++i) {
    if (begin + i < end) fetch(begin + i);
    sa::cp_async_commit();
  }
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    if (i + F::kStages - 1 < end) fetch(i + F::kStages - 1);
    sa::cp_async_commit();
    sa::cp_async_wait<F::kStages - 1>();
    __syncwarp();
    const uint4 x0 = sa::ld_v4(from + 2 * Z * 512);
    uint4 x1 = make_uint4(0, 0, 0, 0);
    if (both) x1 = sa::ld_v4(from + (2 * Z + 1) * 512);
#pragma unroll
    for (int z = 0; z < Z; ++z) {
      const uint4 lo = sa::ld_v4(from + 2 * z * 512), hi = sa::ld_v4(from + (2 * z + 1) * 512);
      mma_k32<T>(acc[z][0], lo, hi, x0);
      if (both) mma_k32<T>(acc[z][1], lo, hi, x1);
    }
    from = from + F::kStageBytes == ring_end ? ring : from + F::kStageBytes;
  }
#pragma unroll
  for (int z = 0; z < Z; ++z)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][z * 256 + (8 * i + 2 * c + (j & 1)) * 16 + g + 8 * (j >> 1)] = acc[z][i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < Z * 256; e += kFusedThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFusedWarps; ++w) sum += part[w][e];
    mine[e] = sum;
  }
  // each block adds up an eighth of h and gives it to all
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = threadIdx.x; i < Z * 256 / kFusedCluster; i += kFusedThreads) {
    const int e = static_cast<int>(blockIdx.x) * (Z * 256 / kFusedCluster) + i, z = e / 256, row = e / 16 % 16, col = 16 * z + e % 16;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < kFusedCluster; ++b) sum += *cluster.map_shared_rank(mine + e, b);
    const T v = static_cast<T>(col < cols && col % R < rank ? sum : 0.f);
#pragma unroll
    for (int b = 0; b < kFusedCluster; ++b) *cluster.map_shared_rank(&hs[row][col], b) = v;
  }
  cluster.sync();                                                    // h is everywhere, and nobody reads or writes others' memory again
  if (!busy) return;
  // ---- expand
  sa::cp_async_wait<0>();
  __syncwarp();
  float sum[2][4][4] = {};
  if (!none) {
    const int keep = rank - 8 * c;
    uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
    if (keep > 0) x0 = *reinterpret_cast<const uint4*>(&hs[g][s * R + 8 * c]), x1 = *reinterpret_cast<const uint4*>(&hs[g + 8][s * R + 8 * c]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 lo = sa::ld_v4(own + 2 * i * 512), hi = sa::ld_v4(own + (2 * i + 1) * 512);
      if (keep > 0 && keep < 8) lo = first_of(lo, keep), hi = first_of(hi, keep);
      mma_k32<T>(sum[0][i], lo, hi, x0);
      if (both) mma_k32<T>(sum[1][i], lo, hi, x1);
    }
  }
  if (!live) return;
  const float scaling = none ? 0.f : __ldg(scalings + tile.x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (8 * (i / 2) + 2 * c + i % 2 >= rows) continue;
    uint4 v = sa::ld_v4(own + (8 + i) * 512);
    if (!none) {
      uint32_t* q = &v.x;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const float2 b = unpack2<T>(q[m]);
        q[m] = pack2(static_cast<T*>(nullptr), fmaf(scaling, sum[i / 2][m][i % 2], b.x), fmaf(scaling, sum[i / 2][m][i % 2 + 2], b.y));
      }
    }
    *reinterpret_cast<uint4*>(out + static_cast<int64_t>(token[i]) * out_ld + n) = v;
  }
}

// Tiles of up to 128 tokens: a warp holds the B of NT x 8 columns of one slice in registers (tokens are the 16-row operand here)
// and walks down the tile, 16 tokens at a time.  Row g of the 8-column operand i is column 2 NT (g / 2) + 2 i + g % 2, so that a
// lane's 2 NT sums of a token are neighbours and base and out move 16 bytes at a time (8 with NT = 2).  RJ = ceil(R / 32).
// The tile's h lies in shared memory, for all of the block's warps; base comes through a ring of kWalkStages steps in shared
// memory in which each lane has its own place, so that three steps are under way without registers being held for them.
constexpr int kWalkThreads = 128, kWalkStages = 4;
template <int RJ, int NT>
constexpr int walk_smem() { return kLargeRows * RJ * 64 + kWalkThreads * kWalkStages * 2 * NT * 4; }

template <typename T, int RJ, int NT>
__global__ void __launch_bounds__(kWalkThreads) lora_expand_tiles_kernel(const T* __restrict__ h, int h_ld, const T* __restrict__ B,
                                                                         int64_t N, int R, const float* __restrict__ scalings,
                                                                         PlanView plan, const __grid_constant__ Slices sl,
                                                                         const T* base, int base_ld, T* out, int out_ld) {
  pdl_start();
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ int row_of[kLargeRows];
  const int tiles = plan.count[0];
  const int4 tile = plan.tiles[blockIdx.y];                  // in bounds whether or not it is one
  if (static_cast<int>(blockIdx.y) >= tiles) return;
  const int rows = tile.z;
  const bool none = tile.x < 0;
  if (none && base == out) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int rank = none ? 0 : min(tile.w, R);
  // a block's four warps have neighbouring columns, of one slice (Slices::first_block counts in fours)
  const int block = blockIdx.x * (kWalkThreads / 32) + warp;
  int s = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i) s += i < sl.n && block >= sl.first_block[i];
  const int n0 = sl.first_col[s] + (block - sl.first_block[s]) * (8 * NT), n_end = sl.first_col[s + 1];
  const int n = n0 + 2 * NT * c;                             // the first of this lane's 2 NT columns
  const bool live = n < n_end;
  const uint32_t hs = smem_u32(dyn);
  const uint32_t ring = hs + kLargeRows * RJ * 64 + threadIdx.x * (4 * NT);
  constexpr uint32_t kHalf = kWalkThreads * 4 * NT, kStage = 2 * kHalf;    // [stage][row half][thread]
  row_of[threadIdx.x] = static_cast<int>(threadIdx.x) < rows ? __ldg(plan.perm + tile.y + threadIdx.x) : 0;
  uint4 w[NT][RJ];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int col = n0 + 2 * NT * (g / 2) + 2 * i + g % 2, keep = rank - 32 * j - 8 * c;
      w[i][j] = load_if(col < n_end && keep > 0, B + (static_cast<int64_t>(tile.x) * N + col) * R + 32 * j + 8 * c);
    }
  const float scaling = none ? 0.f : __ldg(scalings + tile.x);
  __syncthreads();
  // the 16-byte vectors of a row of h, those of odd rows with halves of 64 bytes exchanged: eight lanes then read all banks
  auto h_at = [&](int row, int v) { return hs + row * (RJ * 64) + ((RJ == 1 ? v : v ^ ((row & 1) << 2)) << 4); };
  if (!none) {
    for (int e = threadIdx.x; e < kLargeRows * RJ * 4; e += kWalkThreads) {
      const int row = e / (RJ * 4), v = e % (RJ * 4);
      const bool in = row < rows && v * 8 < rank;
      sa::cp_async_or_zero<16>(h_at(row, v), h + (in ? static_cast<int64_t>(row_of[row]) * h_ld + s * R + v * 8 : 0), in);
    }
  }
  auto fetch = [&](int step) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = step * 16 + g + 8 * i;
      const bool in = base != nullptr && r < rows && live;
      const T* src = in ? base + static_cast<int64_t>(row_of[r]) * base_ld + n : h;
      const uint32_t to = ring + step % kWalkStages * kStage + i * kHalf;
      if constexpr (NT == 4) sa::cp_async_or_zero<16>(to, src, in);
      else sa::cp_async_or_zero<8>(to, src, in);
    }
  };
  const int steps = (rows + 15) / 16;
  sa::cp_async_commit();
#pragma unroll
  for (int i = 0; i < kWalkStages - 1; ++i) {
    if (i < steps) fetch(i);
    sa::cp_async_commit();
  }
  sa::cp_async_wait<kWalkStages - 1>();                      // h
  if (rank % 8 != 0) {                                       // what is behind the rank may be NaN; each thread looks after what it copied
    for (int e = threadIdx.x; e < kLargeRows * RJ * 4; e += kWalkThreads) {
      if (e % (RJ * 4) != rank / 8) continue;
      const uint32_t at = h_at(e / (RJ * 4), rank / 8);
      const uint4 v = first_of(sa::ld_v4(at), rank % 8);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int keep = rank - 32 * j - 8 * c;
      if (keep > 0 && keep < 8) w[i][j] = first_of(w[i][j], keep);
    }
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    if (step + kWalkStages - 1 < steps) fetch(step + kWalkStages - 1);
    sa::cp_async_commit();
    __syncwarp();                                            // lanes that stored come back to those that had nothing to store
    float acc[NT][4] = {};
    if (!none) {
#pragma unroll
      for (int j = 0; j < RJ; ++j) {
        if (32 * j >= rank) break;                           // the same for the whole block
        const uint4 lo = sa::ld_v4(h_at(step * 16 + g, 4 * j + c)), hi = sa::ld_v4(h_at(step * 16 + g + 8, 4 * j + c));
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_k32<T>(acc[i], lo, hi, w[i][j]);
      }
    }
    sa::cp_async_wait<kWalkStages - 1>();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = step * 16 + g + 8 * i;
      uint32_t v[NT];
      const uint32_t from = ring + step % kWalkStages * kStage + i * kHalf;
      if constexpr (NT == 4) {
        const uint4 q = sa::ld_v4(from);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
      } else {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(from) : "memory");
      }
      if (r >= rows || !live) continue;
      if (!none) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 y = __ffma2_rn(make_float2(scaling, scaling), make_float2(acc[j][2 * i], acc[j][2 * i + 1]), unpack2<T>(v[j]));
          v[j] = pack2(static_cast<T*>(nullptr), y.x, y.y);
        }
      }
      T* dst = out + static_cast<int64_t>(row_of[r]) * out_ld + n;
      if constexpr (NT == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
    }
  }
}

// launch_pdl with clusters of `blocks` blocks along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, int blocks, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// How many clusters of n blocks of the large shrink, one block an SM, run at once on the current device; asked once for each n.
constexpr int kMaxSplits = 8;
template <typename Kern>
int cluster_slots(Kern kern, int n) {
  static std::atomic<int> known[64][kMaxSplits + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int v = known[dev][n].load(std::memory_order_relaxed);
  if (v != 0) return v;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(n);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = kTileSmem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&v, kern, &cfg) != cudaSuccess)
    return 0;
  known[dev][n].store(v, std::memory_order_relaxed);
  return v;
}

template <typename T>
int shrink(const T* x, int64_t x_ld, const T* A, int adapters, PlanView plan, int64_t tokens, int64_t tiles, int64_t K, int R, int slices, T* h,
           int64_t h_ld, cudaStream_t st) {
  const int cols = slices * R, sms = sm_count();
  if (sms <= 0) return B200_ERR_CUDA;
  if (K == 0) {
    B200_CUDA_TRY(cudaMemset2DAsync(h, h_ld * sizeof(T), 0, cols * sizeof(T), tokens, st));
    return B200_OK;
  }
  if (tile_rows(tokens, adapters) == kSmallRows) {
    // K is divided as far as five blocks for every SM go, if it has a k32 step for each of their warps.  Two groups of columns a
    // block, and four blocks for an SM, where single ones would not be divided at all, or full tiles not by eight.  Shared memory,
    // the static part counted, holds one block less of either kind; but the number of tiles is an estimate that errs upwards, and blocks
    // behind a rank leave at once.  Counted with four and three instead, 81 random batches took 3.8 % longer than with the best
    // division of each (at worst 1.56 times as long), with five and four 3.3 % (1.50); with the sums where the rings are, so that five
    // and four fit, the blocks of most batches crowd on fewer SMs (128 tokens of 32 adapters, 3 slices of 64: 16.2 -> 18.9 us).
    // Blocks of one group divided by 8 / 4 / 2, and of two by 8 / 4 / 2 (us; K = 8192, with the expand, 4 and 5 stages): 128 tokens of 32
    // adapters, 3 slices of 16: 18.6 15.6 17.5, 19.8 16.1 18.3; of 64 34.4 27.8 24.9, 37.2 29.6 25.5 with mixed ranks, 42.0 36.8
    // 34.8, 45.1 36.8 33.6 with rank 64 only; 200 tokens of one adapter 21.9 19.5 17.2, 19.1 14.8 19.
    const int passes = (cols + 15) / 16;
    const int64_t few = adapters < tokens ? adapters : tokens, half = (tokens + kSmallRows - 1) / kSmallRows + few / 2, about = few > half ? few : half;
    auto divided = [&](int64_t blocks, int64_t most) {
      int n = 1;
      while (n < 8 && 2 * n * blocks <= most && n * 32 * kShrinkWarps < K) n *= 2;
      return n;
    };
    auto go = [&](auto z, int splits) -> int {
      constexpr int Z = decltype(z)::value;
      B200_CUDA_TRY(cudaFuncSetAttribute(lora_shrink_kernel<T, Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shrink<Z>::kSmem));
      B200_CUDA_TRY(launch_cluster(lora_shrink_kernel<T, Z>, dim3(splits, static_cast<unsigned>(tiles), (passes + Z - 1) / Z),
                                   dim3(kShrinkThreads), Shrink<Z>::kSmem, splits, st, x, x_ld, A, K, R, cols, plan, h, h_ld));
      return B200_OK;
    };
    const int64_t blocks = about * passes, most = 5LL * sms;
    if (2 * blocks > most || (8 * blocks > most && tokens >= kSmallRows * static_cast<int64_t>(adapters)))
      return go(std::integral_constant<int, 2>(), divided((blocks + 1) / 2, 4LL * sms));
    return go(std::integral_constant<int, 1>(), divided(blocks, most));
  }
  if (gemm_sticky_status() != 0) return B200_ERR_DEVICE_TIMEOUT;
  ShrinkTiles p = {K, h_ld, R, slices};
  p.status = gemm_status_ptr();
  if (!p.status) return B200_ERR_CUDA;
  p.a_box = R % 32 == 0 ? 32 : R % 16 == 0 ? 16 : 8;       // rows of A that are fetched at a time; slices begin at multiples
  p.n_alloc = cols < kMaxColumns ? (cols + 15) / 16 * 16 : kMaxColumns;
  const int passes = (cols + kMaxColumns - 1) / kMaxColumns;
  // As many blocks a tile as let all tiles run at once, one block an SM.  Of a cluster's blocks no two may lie in different
  // processing clusters of the chip, so fewer clusters fit than SMs / size (of four blocks 33, of three 45); a batch has about an
  // eighth to a quarter more tiles than whole ones.  37 tiles of 4096 x 7168 x 64: four blocks in two waves 38 us, three in one 28.
  const int64_t whole = (tokens + kLargeRows - 1) / kLargeRows, about = passes * (whole + (adapters < whole / 4 ? adapters : whole / 4));
  p.splits = 1;
  for (int n = 2; n <= kMaxSplits; ++n)
    if (static_cast<int64_t>(n) * kBlockK <= K && about <= cluster_slots(lora_shrink_tiles_kernel<T>, n)) p.splits = n;
  const int stage_bytes = static_cast<int>(kXBytes) + p.n_alloc * kBlockK * 2;
  p.stages = (kTileSmem - 1024) / stage_bytes < kMaxTileStages ? (kTileSmem - 1024) / stage_bytes : kMaxTileStages;
  ShrinkMaps maps;
  const int64_t a_rows = static_cast<int64_t>(adapters) * cols;
  p.a_whole = cols <= kMaxColumns;
  int rc = make_map_u16_2d(&maps.a, A, a_rows, K, K, p.a_box);
  if (rc == B200_OK) rc = make_map_u16_2d(&maps.a_whole, A, a_rows, K, K, p.a_whole ? cols : p.a_box);
  for (int i = 0; i < 5 && rc == B200_OK; ++i) rc = make_map_u16_2d(&maps.x[i], x, tokens, K, x_ld, i == 0 ? 1 : 4 << i);
  if (rc != B200_OK) return rc;
  B200_CUDA_TRY(cudaFuncSetAttribute(lora_shrink_tiles_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem));
  B200_CUDA_TRY(launch_cluster(lora_shrink_tiles_kernel<T>, dim3(p.splits, static_cast<unsigned>(tiles), passes), dim3(kTileThreads), kTileSmem,
                               p.splits, st, maps, plan, h, p));
  return B200_OK;
}

// Slices in blocks of warp_cols columns, a whole number of block_cols for each.
Slices make_slices(const int64_t* sizes, int n, int warp_cols, int block_cols) {
  Slices sl = {};
  sl.n = n;
  for (int i = 0; i < n; ++i) {
    sl.first_col[i + 1] = sl.first_col[i] + static_cast<int>(sizes[i]);
    sl.first_block[i + 1] = sl.first_block[i] + static_cast<int>((sizes[i] + block_cols - 1) / block_cols) * (block_cols / warp_cols);
  }
  return sl;
}

// Columns of a warp of the expand.
int expand_columns(int64_t tokens, int adapters, int R) { return tile_rows(tokens, adapters) == kSmallRows ? 64 : R <= 128 ? 32 : 16; }

template <typename T>
int expand(const T* h, int64_t h_ld, const T* B, int64_t N, int R, const float* scalings, int adapters, PlanView plan, const Slices& sl, int64_t tokens,
           int64_t tiles, const T* base, int64_t base_ld, T* out, int64_t out_ld, bool early, cudaStream_t st) {
  static_assert(kExpandThreads == kWalkThreads, "one grid for both");
  const int sms = sm_count();
  if (sms <= 0) return B200_ERR_CUDA;
  constexpr int kWarps = kExpandThreads / 32;
  // small batches: as many blocks of columns a warp as leave 24 warps for each SM (16 are resident), at most eight.  1, 2, 4, 8 of
  // them: 41 tiles of N = 36864, R = 32: 21.3, 20.6, 19.0, 17.9 us; of 10240, ranks 16 to 64: 9.6, 10.7, 11.9, 16.1
  int per = 1;
  if (tile_rows(tokens, adapters) == kSmallRows) {
    const int64_t most = tiles * sl.first_block[sl.n] / (24LL * sms);
    per = static_cast<int>(most < 1 ? 1 : most < 8 ? most : 8);
  }
  const dim3 grid(static_cast<unsigned>((sl.first_block[sl.n] + kWarps * per - 1) / (kWarps * per)), static_cast<unsigned>(tiles));
  auto go = [&](auto kern, int smem, auto... more) -> int {
    if (smem > 40 * 1024) B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CUDA_TRY(launch_pdl(kern, grid, dim3(kExpandThreads), smem, st, h, static_cast<int>(h_ld), B, N, R, scalings, plan, sl, base,
                             static_cast<int>(base_ld), out, static_cast<int>(out_ld), more...));
    return B200_OK;
  };
  if (tile_rows(tokens, adapters) == kSmallRows) return go(lora_expand_kernel<T>, kExpandSmem, per, early);
  if (R <= 32) return go(lora_expand_tiles_kernel<T, 1, 4>, walk_smem<1, 4>());
  if (R <= 64) return go(lora_expand_tiles_kernel<T, 2, 4>, walk_smem<2, 4>());
  if (R <= 128) return go(lora_expand_tiles_kernel<T, 4, 4>, walk_smem<4, 4>());
  return go(lora_expand_tiles_kernel<T, 8, 2>, walk_smem<8, 2>());
}

// Clusters of a tile in the fused form, one block of 64 columns a warp; 0 where it is not used.
int fused_parts(int64_t tokens, int adapters, int64_t tiles, int cols, const Slices& sl) {
  if (tile_rows(tokens, adapters) != kSmallRows || cols > kFusedColumns) return 0;
  const int parts = (sl.first_block[sl.n] + kFusedCluster * kFusedWarps - 1) / (kFusedCluster * kFusedWarps);
  return parts <= kFusedParts && tiles * parts <= kFusedClusters ? parts : 0;
}

template <typename T, int Z>
int fused(const T* x, int64_t x_ld, const T* A, const T* B, int64_t K, int64_t N, int R, int cols, const float* scalings, PlanView plan,
          const Slices& sl, int64_t tiles, int parts, const T* base, int base_ld, T* out, int out_ld, cudaStream_t st) {
  B200_CUDA_TRY(cudaFuncSetAttribute(lora_fused_kernel<T, Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fused<Z>::kSmem));
  B200_CUDA_TRY(launch_cluster(lora_fused_kernel<T, Z>, dim3(kFusedCluster, static_cast<unsigned>(tiles), parts), dim3(kFusedThreads),
                               Fused<Z>::kSmem, kFusedCluster, st, x, x_ld, A, B, K, N, R, cols, scalings, plan, sl, base, base_ld, out,
                               out_ld));
  return B200_OK;
}
template <typename T>
int fused(const void* x, int64_t x_ld, const void* A, const void* B, int64_t K, int64_t N, int R, int cols, const float* scalings,
          PlanView plan, const Slices& sl, int64_t tiles, int parts, const void* base, int64_t base_ld, void* out, int64_t out_ld,
          cudaStream_t st) {
  auto go = [&](auto z) {
    return fused<T, decltype(z)::value>(static_cast<const T*>(x), x_ld, static_cast<const T*>(A), static_cast<const T*>(B), K, N, R,
                                        cols, scalings, plan, sl, tiles, parts, static_cast<const T*>(base), static_cast<int>(base_ld),
                                        static_cast<T*>(out), static_cast<int>(out_ld), st);
  };
  if (cols <= 16) return go(std::integral_constant<int, 1>());
  return go(std::integral_constant<int, 2>());
}

int check_plan(const void* plan, size_t bytes, int64_t T, int64_t L) {
  if (!plan) return B200_ERR_NULL_PTR;
  if (!aligned16(plan)) return B200_ERR_MISALIGNED;
  return bytes >= b200_lora_plan_bytes(T, static_cast<int>(L)) ? B200_OK : B200_ERR_BAD_SHAPE;
}
int check_sizes(int64_t T, int64_t L, int64_t R) {
  if (T < 0 || L <= 0 || R <= 0 || R % 8 != 0) return B200_ERR_BAD_SHAPE;
  if (T > kMaxTokens || L > kMaxAdapters || R > 256) return B200_ERR_TOO_LARGE;
  return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" size_t b200_lora_plan_bytes(int64_t T, int L) {
  if (T < 0 || L <= 0) return 0;
  return static_cast<size_t>(16 + 16 * b200::plan_tiles(T, L) + 4 * T);
}

extern "C" int b200_lora_plan(const int32_t* token_adapters, int64_t T, const int32_t* ranks, int L, void* plan,
                              size_t plan_bytes, void* stream) {
  using namespace b200;
  int rc = check_sizes(T, L, 8);
  if (rc != B200_OK) return rc;
  if ((rc = check_plan(plan, plan_bytes, T, L)) != B200_OK) return rc;
  if ((T > 0 && !token_adapters) || !ranks) return B200_ERR_NULL_PTR;
  // The large shrink reports into the status ring, whose first use allocates: here rather than in a capture of the shrink.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  B200_CUDA_TRY(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture));
  if (capture == cudaStreamCaptureStatusNone && tile_rows(T, L) == kLargeRows) gemm_sticky_status();
  const PlanView v = view_plan(plan, T, L);
  auto smem_of = [](int n) { return static_cast<int>(sizeof(int)) * ((kPlanWarps + 1) * (n + 1) + 2 * (n + 2)); };
  const int smem = smem_of(L);
  // Always the most that there can be: the limit is the kernel's, for all threads, and a smaller one of another thread could come
  // between this call and the launch.
  if (smem > 48 * 1024) B200_CUDA_TRY(cudaFuncSetAttribute(lora_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of(kMaxAdapters)));
  B200_CUDA_TRY(launch_pdl(lora_plan_kernel, dim3(1), dim3(kPlanThreads), smem, static_cast<cudaStream_t>(stream), token_adapters, T,
                           ranks, L, tile_rows(T, L), const_cast<int*>(v.count), const_cast<int4*>(v.tiles), const_cast<int*>(v.perm)));
  return B200_OK;
}

namespace b200 {
namespace {

// check_only, here and in expand_entry: the arguments are looked at, nothing is launched.
int shrink_entry(const void* x, int64_t x_ld, const void* A, int dtype, const void* plan, size_t plan_bytes, int64_t T, int L,
                 int64_t K, int R, int num_slices, void* h, int64_t h_ld, bool check_only, void* stream) {
  int rc = check_sizes(T, L, R);
  if (rc != B200_OK) return rc;
  if (num_slices <= 0 || K < 0 || K % 8 != 0) return B200_ERR_BAD_SHAPE;
  if (num_slices > kMaxSlices || K > (1LL << 30)) return B200_ERR_TOO_LARGE;
  if (dtype != B200_DT_BF16 && dtype != B200_DT_F16) return B200_ERR_BAD_DTYPE;
  const int cols = num_slices * R;
  if (x_ld < K || x_ld % 8 != 0 || h_ld < cols || h_ld % 8 != 0) return B200_ERR_BAD_STRIDE;
  if (T == 0) return B200_OK;
  if ((rc = check_plan(plan, plan_bytes, T, L)) != B200_OK) return rc;
  if ((K > 0 && (!x || !A)) || !h) return B200_ERR_NULL_PTR;
  if (!aligned16(x) || !aligned16(A) || !aligned16(h)) return B200_ERR_MISALIGNED;
  if (check_only) return B200_OK;
  const int64_t tiles = max_tiles(T, L);
  const PlanView v = view_plan(plan, T, L);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200_DT_BF16)
    return shrink(static_cast<const __nv_bfloat16*>(x), x_ld, static_cast<const __nv_bfloat16*>(A), L, v, T, tiles, K, R, num_slices,
                  static_cast<__nv_bfloat16*>(h), h_ld, st);
  return shrink(static_cast<const __half*>(x), x_ld, static_cast<const __half*>(A), L, v, T, tiles, K, R, num_slices,
                static_cast<__half*>(h), h_ld, st);
}

int expand_entry(const void* h, int64_t h_ld, const void* B, int dtype, const void* plan, size_t plan_bytes, const float* scalings,
                 int64_t T, int L, int R, const int64_t* slice_sizes, int num_slices, const void* base, int64_t base_ld, void* out,
                 int64_t out_ld, bool early, bool check_only, void* stream) {
  int rc = check_sizes(T, L, R);
  if (rc != B200_OK) return rc;
  if (num_slices <= 0 || !slice_sizes) return num_slices <= 0 ? B200_ERR_BAD_SHAPE : B200_ERR_NULL_PTR;
  if (num_slices > kMaxSlices) return B200_ERR_TOO_LARGE;
  if (dtype != B200_DT_BF16 && dtype != B200_DT_F16) return B200_ERR_BAD_DTYPE;
  int64_t N = 0;
  for (int i = 0; i < num_slices; ++i) {
    if (slice_sizes[i] < 0 || slice_sizes[i] % 8 != 0) return B200_ERR_BAD_SHAPE;
    if (slice_sizes[i] > (1 << 30) || N + slice_sizes[i] > (1 << 30)) return B200_ERR_TOO_LARGE;
    N += slice_sizes[i];
  }
  const int warp_cols = expand_columns(T, L, R);
  const Slices sl = make_slices(slice_sizes, num_slices, warp_cols, tile_rows(T, L) == kSmallRows ? warp_cols : 4 * warp_cols);
  if (h_ld < num_slices * static_cast<int64_t>(R) || h_ld % 8 != 0 || out_ld < N || out_ld % 8 != 0 ||
      (base && (base_ld < N || base_ld % 8 != 0)))
    return B200_ERR_BAD_STRIDE;
  if (h_ld > 0x7fffffffLL || base_ld > 0x7fffffffLL || out_ld > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  if (T == 0 || N == 0) return B200_OK;
  if ((rc = check_plan(plan, plan_bytes, T, L)) != B200_OK) return rc;
  if (!h || !B || !scalings || !out) return B200_ERR_NULL_PTR;
  if (!aligned16(h) || !aligned16(B) || !aligned16(base) || !aligned16(out)) return B200_ERR_MISALIGNED;
  if (check_only) return B200_OK;
  const int64_t tiles = max_tiles(T, L);
  const PlanView v = view_plan(plan, T, L);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200_DT_BF16)
    return expand(static_cast<const __nv_bfloat16*>(h), h_ld, static_cast<const __nv_bfloat16*>(B), N, R, scalings, L, v, sl, T, tiles,
                  static_cast<const __nv_bfloat16*>(base), base_ld, static_cast<__nv_bfloat16*>(out), out_ld, early, st);
  return expand(static_cast<const __half*>(h), h_ld, static_cast<const __half*>(B), N, R, scalings, L, v, sl, T, tiles,
                static_cast<const __half*>(base), base_ld, static_cast<__half*>(out), out_ld, early, st);
}

}  // namespace
}  // namespace b200

extern "C" int b200_lora_shrink(const void* x, int64_t x_ld, const void* A, int dtype, const void* plan, size_t plan_bytes,
                                int64_t T, int L, int64_t K, int R, int num_slices, void* h, int64_t h_ld, void* stream) {
  return b200::shrink_entry(x, x_ld, A, dtype, plan, plan_bytes, T, L, K, R, num_slices, h, h_ld, false, stream);
}

extern "C" int b200_lora_expand(const void* h, int64_t h_ld, const void* B, int dtype, const void* plan, size_t plan_bytes,
                                const float* scalings, int64_t T, int L, int R, const int64_t* slice_sizes, int num_slices,
                                const void* base, int64_t base_ld, void* out, int64_t out_ld, void* stream) {
  return b200::expand_entry(h, h_ld, B, dtype, plan, plan_bytes, scalings, T, L, R, slice_sizes, num_slices, base, base_ld, out, out_ld,
                            false, false, stream);
}

extern "C" int b200_lora_apply(const void* x, int64_t x_ld, const void* A, const void* B, int dtype, const void* plan,
                               size_t plan_bytes, const float* scalings, int64_t T, int L, int64_t K, int R,
                               const int64_t* slice_sizes, int num_slices, const void* base, int64_t base_ld, void* out,
                               int64_t out_ld, void* h, void* stream) {
  using namespace b200;
  const int64_t h_ld = static_cast<int64_t>(num_slices) * R;
  int rc = expand_entry(h, h_ld, B, dtype, plan, plan_bytes, scalings, T, L, R, slice_sizes, num_slices, base, base_ld, out, out_ld, true,
                        true, stream);
  if (rc != B200_OK) return rc;
  if ((rc = shrink_entry(x, x_ld, A, dtype, plan, plan_bytes, T, L, K, R, num_slices, h, h_ld, true, stream)) != B200_OK) return rc;
  const Slices sl = make_slices(slice_sizes, num_slices, 64, 64);
  if (T > 0 && sl.first_col[num_slices] > 0 && K > 0) {
    const int64_t tiles = max_tiles(T, L), N = sl.first_col[num_slices];
    const int parts = fused_parts(T, L, tiles, static_cast<int>(h_ld), sl);
    if (parts > 0)
      return (dtype == B200_DT_BF16 ? fused<__nv_bfloat16> : fused<__half>)(
          x, x_ld, A, B, K, N, R, static_cast<int>(h_ld), scalings, view_plan(plan, T, L), sl, tiles, parts, base, base_ld, out, out_ld,
          static_cast<cudaStream_t>(stream));
  }
  if ((rc = shrink_entry(x, x_ld, A, dtype, plan, plan_bytes, T, L, K, R, num_slices, h, h_ld, false, stream)) != B200_OK) return rc;
  // with K = 0 there is no kernel before the expand that would make reading ahead sound
  return expand_entry(h, h_ld, B, dtype, plan, plan_bytes, scalings, T, L, R, slice_sizes, num_slices, base, base_ld, out, out_ld, K > 0,
                      false, stream);
}
