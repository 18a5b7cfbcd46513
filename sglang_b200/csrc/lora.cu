// Low-rank adapters of many requests beside one shared projection, for sm_100a:
//
//   h[t, s, r]  = sum_k x[t, k] A[a, s R + r, k]                      (shrink; a = the token's adapter, r < rank[a])
//   out[t, n]   = base[t, n] + scaling[a] sum_r h[t, s(n), r] B[a, n, r]        (expand; s(n) = the slice of column n)
//
// The plan groups the tokens by adapter (a stable counting sort), so that a tile of up to kTileRows tokens shares one A and
// one B; it is made once for a batch of tokens and used by every projection of every layer.
//
// Both products are bound by memory: the shrink by x and A, the expand by base, out and B.  Operands go from global memory
// straight into the fragments of mma.m16n8k16: the order in which k is summed is free, so a lane's fragment of two
// consecutive k16 steps is one 16-byte load (eight consecutive k), and no shared memory or transposition is needed.  The
// weights are the 16-row operand, the tokens the 8-column one, so a single token wastes no weight traffic.
//
// Sums are held in fp32.  h is rounded once, to the type of x, because the expand multiplies it with B on the tensor cores;
// that adds at most half a step of h (2^-9 for bf16) to the adapter's part of the sum, less than the rounding of out adds.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kTileRows = 16;
constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr int kMaxAdapters = 1024;
constexpr int kMaxSlices = 8;
constexpr int64_t kMaxTokens = 1000000;     // max_tiles(kMaxTokens, kMaxAdapters) is a legal grid.y

// Device layout of a plan: int32 count[4] (tiles, -, -, -), int4 tiles[max_tiles] (adapter or -1, first, rows, rank), int32 perm[T]
__host__ __device__ inline int64_t max_tiles(int64_t T, int64_t L) {
  return T / kTileRows + (L + 1 < T ? L + 1 : T);
}

struct PlanView {
  const int* count;
  const int4* tiles;
  const int* perm;
};
inline PlanView view_plan(const void* plan, int64_t T, int64_t L) {
  const char* b = static_cast<const char*>(plan);
  return {reinterpret_cast<const int*>(b), reinterpret_cast<const int4*>(b + 16),
          reinterpret_cast<const int*>(b + 16 + 16 * max_tiles(T, L))};
}

// ------------------------------------------------------------------------------------------------------- plan
// One block.  Warp w owns the tokens [w * per, ...); bins [kPlanWarps][L + 1] in shared memory count its tokens per adapter
// (bin L: none), then hold where its next token of that adapter goes.  Stable: a token's place depends on nothing but the ids.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const int32_t* __restrict__ ids, int64_t T,
                                                                 const int32_t* __restrict__ ranks, int L,
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
    tile0[a + 1] = (run + kTileRows - 1) / kTileRows;
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
      const int at = first[a] + (i - tile0[a]) * kTileRows;
      tiles[i] = make_int4(a < L ? a : -1, at, min(kTileRows, first[a + 1] - at), rank_of[a]);
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
// 32 consecutive k at once: lo and hi are the 16-byte vectors (k = 8c .. 8c + 7, c = lane % 4) of the weight rows lane / 4 and
// lane / 4 + 8, x the one of token lane / 4.
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
constexpr int kShrinkThreads = 128, kShrinkCluster = 8;

// A cluster of eight blocks computes 16 columns of h for one tile of up to 16 tokens, its 32 warps dividing K; the partial
// sums are added in a fixed order, first over a block's warps, then over the blocks through distributed shared memory.
template <typename T>
__global__ void __cluster_dims__(kShrinkCluster, 1, 1) __launch_bounds__(kShrinkThreads)
lora_shrink_kernel(const T* __restrict__ x, int64_t x_ld, const T* __restrict__ A, int64_t K, int R, int cols,
                   PlanView plan, T* __restrict__ h, int64_t h_ld) {
  pdl_start();
  __shared__ float part[kShrinkThreads / 32][256];
  __shared__ float mine[256];
  if (static_cast<int>(blockIdx.y) >= plan.count[0]) return;        // the whole cluster leaves together
  const int4 tile = plan.tiles[blockIdx.y];
  const int c0 = blockIdx.z * 16;
  if (tile.x < 0) {                                                 // tokens without an adapter: zeros
    if (blockIdx.x == 0)
      for (int e = threadIdx.x; e < 256; e += kShrinkThreads)
        if (e / 16 < tile.z && c0 + e % 16 < cols)
          h[static_cast<int64_t>(plan.perm[tile.y + e / 16]) * h_ld + c0 + e % 16] = static_cast<T>(0.f);
    return;
  }
  const int rank = min(tile.w, R);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int rows = tile.z;
  const T* wp[2];
  bool wok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int col = c0 + g + 8 * i;
    wok[i] = col < cols && col % R < rank;
    wp[i] = A + (static_cast<int64_t>(tile.x) * cols + col) * K + 8 * c;
  }
  const T* xp[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    xp[i] = r < rows ? x + static_cast<int64_t>(__ldg(plan.perm + tile.y + r)) * x_ld + 8 * c : nullptr;
  }
  const bool both = rows > 8;
  float acc[2][4] = {};
  const int64_t chunks = (K + 31) / 32;
  const int64_t per = (chunks + kShrinkCluster * (kShrinkThreads / 32) - 1) / (kShrinkCluster * (kShrinkThreads / 32));
  const int64_t begin = (blockIdx.x * (kShrinkThreads / 32) + warp) * per, end = begin + per < chunks ? begin + per : chunks;
  for (int64_t i = begin; i < end; i += 4) {
    uint4 w0[4], w1[4], x0[4], x1[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t k = (i + u) * 32;
      const bool in = i + u < end && k + 8 * c < K;
      w0[u] = load_if(in && wok[0], wp[0] + k);
      w1[u] = load_if(in && wok[1], wp[1] + k);
      x0[u] = load_if(in && xp[0] != nullptr, xp[0] + k);
      x1[u] = load_if(both && in && xp[1] != nullptr, xp[1] + k);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      mma_k32<T>(acc[0], w0[u], w1[u], x0[u]);
      if (both) mma_k32<T>(acc[1], w0[u], w1[u], x1[u]);
    }
  }
  // part[warp][token][column]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[warp][(8 * i + 2 * c + (j & 1)) * 16 + g + 8 * (j >> 1)] = acc[i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < 256; e += kShrinkThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kShrinkThreads / 32; ++w) s += part[w][e];
    mine[e] = s;
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (threadIdx.x < 256 / kShrinkCluster) {
    const int e = static_cast<int>(cluster.block_rank()) * (256 / kShrinkCluster) + threadIdx.x;
    float s = 0.f;
#pragma unroll
    for (int b = 0; b < kShrinkCluster; ++b) s += *cluster.map_shared_rank(mine + e, b);
    const int row = e / 16, col = c0 + e % 16;
    if (row < rows && col < cols)
      h[static_cast<int64_t>(plan.perm[tile.y + row]) * h_ld + col] = static_cast<T>(col % R < rank ? s : 0.f);
  }
  cluster.sync();
}

// ------------------------------------------------------------------------------------------------------- expand
struct Slices {
  int n, first_col[kMaxSlices + 1], first_block[kMaxSlices + 1];     // columns; blocks of 64 columns
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
__device__ __forceinline__ uint32_t pack2_as(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack2_as(float a, float b, __half*) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

constexpr int kExpandThreads = 128;

// A warp: 64 columns of one slice for one tile of up to 16 tokens.  Weight row (tile i, half f, lane / 4) of its four 16-row
// operands is column 8 (lane / 4) + 2 i + f, so that the eight sums that a lane holds for a token are neighbours: base and out
// move 16 bytes at a time.
template <typename T>
__global__ void __launch_bounds__(kExpandThreads) lora_expand_kernel(const T* __restrict__ h, int64_t h_ld, const T* __restrict__ B,
                                                                     int64_t N, int R, const float* __restrict__ scalings,
                                                                     PlanView plan, const __grid_constant__ Slices sl,
                                                                     const T* base, int64_t base_ld, T* out, int64_t out_ld) {
  pdl_start();
  if (static_cast<int>(blockIdx.y) >= plan.count[0]) return;
  const int4 tile = plan.tiles[blockIdx.y];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int block = blockIdx.x * (kExpandThreads / 32) + warp;
  if (block >= sl.first_block[sl.n]) return;
  int s = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i) s += i < sl.n && block >= sl.first_block[i];
  const int n = sl.first_col[s] + (block - sl.first_block[s]) * 64 + 8 * g;   // the first of this lane's eight columns
  const bool live = n < sl.first_col[s + 1];
  const int rows = tile.z;
  const bool none = tile.x < 0;
  if (none && base == out) return;
  const bool both = rows > 8;
  float acc[2][4][4] = {};
  float scaling = 0.f;
  if (!none) {
    const int rank = min(tile.w, R);
    scaling = __ldg(scalings + tile.x);
    const T* bp = B + (static_cast<int64_t>(tile.x) * N + n) * R + 8 * c;
    const T* hp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      hp[i] = r < rows ? h + static_cast<int64_t>(__ldg(plan.perm + tile.y + r)) * h_ld + s * R + 8 * c : nullptr;
    }
    for (int r0 = 0; r0 < rank; r0 += 32) {
      const int keep = rank - r0 - 8 * c;
      const uint4 x0 = load_if(keep > 0 && hp[0] != nullptr, hp[0] + r0);
      const uint4 x1 = load_if(both && keep > 0 && hp[1] != nullptr, hp[1] + r0);
      uint4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = load_if(live && keep > 0, bp + i * R + r0);
        if (keep < 8) w[i] = first_of(w[i], keep);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mma_k32<T>(acc[0][i], w[2 * i], w[2 * i + 1], x0);
        if (both) mma_k32<T>(acc[1][i], w[2 * i], w[2 * i + 1], x1);
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * i + 2 * c + j;
      if (r >= rows) continue;
      const int64_t t = __ldg(plan.perm + tile.y + r);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (base != nullptr) v = *reinterpret_cast<const uint4*>(base + t * base_ld + n);
      if (!none) {
        uint32_t* w = &v.x;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float2 b = unpack2<T>(w[m]);
          w[m] = pack2_as(fmaf(scaling, acc[i][m][j], b.x), fmaf(scaling, acc[i][m][j + 2], b.y), static_cast<T*>(nullptr));
        }
      }
      *reinterpret_cast<uint4*>(out + t * out_ld + n) = v;
    }
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
  return static_cast<size_t>(16 + 16 * b200::max_tiles(T, L) + 4 * T);
}

extern "C" int b200_lora_plan(const int32_t* token_adapters, int64_t T, const int32_t* ranks, int L, void* plan,
                              size_t plan_bytes, void* stream) {
  using namespace b200;
  int rc = check_sizes(T, L, 8);
  if (rc != B200_OK) return rc;
  if ((rc = check_plan(plan, plan_bytes, T, L)) != B200_OK) return rc;
  if ((T > 0 && !token_adapters) || !ranks) return B200_ERR_NULL_PTR;
  const PlanView v = view_plan(plan, T, L);
  const size_t smem = sizeof(int) * ((kPlanWarps + 1) * (L + 1) + 2 * (L + 2));
  if (smem > 48 * 1024) B200_CUDA_TRY(cudaFuncSetAttribute(lora_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  B200_CUDA_TRY(launch_pdl(lora_plan_kernel, dim3(1), dim3(kPlanThreads), smem, static_cast<cudaStream_t>(stream), token_adapters, T,
                           ranks, L, const_cast<int*>(v.count), const_cast<int4*>(v.tiles), const_cast<int*>(v.perm)));
  return B200_OK;
}

extern "C" int b200_lora_shrink(const void* x, int64_t x_ld, const void* A, int dtype, const void* plan, size_t plan_bytes,
                                int64_t T, int L, int64_t K, int R, int num_slices, void* h, int64_t h_ld, void* stream) {
  using namespace b200;
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
  const int64_t tiles = max_tiles(T, L);
  const dim3 grid(kShrinkCluster, static_cast<unsigned>(tiles), static_cast<unsigned>((cols + 15) / 16));
  const PlanView v = view_plan(plan, T, L);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200_DT_BF16)
    B200_CUDA_TRY(launch_pdl(lora_shrink_kernel<__nv_bfloat16>, grid, dim3(kShrinkThreads), 0, st, static_cast<const __nv_bfloat16*>(x),
                             x_ld, static_cast<const __nv_bfloat16*>(A), K, R, cols, v, static_cast<__nv_bfloat16*>(h), h_ld));
  else
    B200_CUDA_TRY(launch_pdl(lora_shrink_kernel<__half>, grid, dim3(kShrinkThreads), 0, st, static_cast<const __half*>(x), x_ld,
                             static_cast<const __half*>(A), K, R, cols, v, static_cast<__half*>(h), h_ld));
  return B200_OK;
}

extern "C" int b200_lora_expand(const void* h, int64_t h_ld, const void* B, int dtype, const void* plan, size_t plan_bytes,
                                const float* scalings, int64_t T, int L, int R, const int64_t* slice_sizes, int num_slices,
                                const void* base, int64_t base_ld, void* out, int64_t out_ld, void* stream) {
  using namespace b200;
  int rc = check_sizes(T, L, R);
  if (rc != B200_OK) return rc;
  if (num_slices <= 0 || !slice_sizes) return num_slices <= 0 ? B200_ERR_BAD_SHAPE : B200_ERR_NULL_PTR;
  if (num_slices > kMaxSlices) return B200_ERR_TOO_LARGE;
  if (dtype != B200_DT_BF16 && dtype != B200_DT_F16) return B200_ERR_BAD_DTYPE;
  Slices sl = {};
  sl.n = num_slices;
  int64_t N = 0;
  for (int i = 0; i < num_slices; ++i) {
    if (slice_sizes[i] < 0 || slice_sizes[i] % 8 != 0) return B200_ERR_BAD_SHAPE;
    N += slice_sizes[i];
    if (N > (1 << 30)) return B200_ERR_TOO_LARGE;
    sl.first_col[i + 1] = static_cast<int>(N);
    sl.first_block[i + 1] = sl.first_block[i] + static_cast<int>((slice_sizes[i] + 63) / 64);
  }
  if (h_ld < num_slices * static_cast<int64_t>(R) || h_ld % 8 != 0 || out_ld < N || out_ld % 8 != 0 ||
      (base && (base_ld < N || base_ld % 8 != 0)))
    return B200_ERR_BAD_STRIDE;
  if (T == 0 || N == 0) return B200_OK;
  if ((rc = check_plan(plan, plan_bytes, T, L)) != B200_OK) return rc;
  if (!h || !B || !scalings || !out) return B200_ERR_NULL_PTR;
  if (!aligned16(h) || !aligned16(B) || !aligned16(base) || !aligned16(out)) return B200_ERR_MISALIGNED;
  const int64_t tiles = max_tiles(T, L);
  constexpr int kWarps = kExpandThreads / 32;
  const dim3 grid(static_cast<unsigned>((sl.first_block[num_slices] + kWarps - 1) / kWarps), static_cast<unsigned>(tiles));
  const PlanView v = view_plan(plan, T, L);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200_DT_BF16)
    B200_CUDA_TRY(launch_pdl(lora_expand_kernel<__nv_bfloat16>, grid, dim3(kExpandThreads), 0, st, static_cast<const __nv_bfloat16*>(h),
                             h_ld, static_cast<const __nv_bfloat16*>(B), N, R, scalings, v, sl,
                             static_cast<const __nv_bfloat16*>(base), base_ld, static_cast<__nv_bfloat16*>(out), out_ld));
  else
    B200_CUDA_TRY(launch_pdl(lora_expand_kernel<__half>, grid, dim3(kExpandThreads), 0, st, static_cast<const __half*>(h), h_ld,
                             static_cast<const __half*>(B), N, R, scalings, v, sl, static_cast<const __half*>(base), base_ld,
                             static_cast<__half*>(out), out_ld));
  return B200_OK;
}
