// Between the qkv projection and the attention kernel, for sm_100a: RMSNorm of every query and key head, the rotary
// position embedding, keys and values quantised into a paged cache, and the cache read back.  All of it moves data: the
// floor is the bytes read and written once, at the memory's rate.
//
// One head of one token ("row", D elements) belongs to a group of G lanes, G the power of two from D / 8 up, each lane
// holding eight consecutive elements (one 16-byte load).  Everything that a row needs is a shuffle inside its group: the
// sum of squares, the partner of a rotated pair, the largest magnitude.  A warp takes U x (32 / G) neighbouring rows of one
// token, so its cosines and sines are loaded once for all of them, and all rows' loads are in flight before the first is
// used.  All arithmetic is in 32 bits; a query is rounded once, when it is stored, and a key once, to e4m3.
//
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)     neox: b = a + rot / 2; otherwise neighbours a = 2i, b = 2i + 1
//   scale = max(1e-10, max|y|) / 448,  code = e4m3(y / scale)     correctly rounded quotient, as in the group quantiser
#include "common.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 128;

struct HeadRowsParams {
  const void *q, *k, *v;
  void *q_out, *k_out;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;   // element strides: token, head
  const void *q_w, *k_w;
  const void* positions;
  const float* cos_sin;
  const void* slots;
  uint8_t *kc, *vc;
  float *ks, *vs;
  int64_t kc_s[3], vc_s[3], ks_s[3], vs_s[3];   // page, slot inside the page, head
  int64_t T, max_position;
  uint32_t num_slots, page_size;
  int Hq, Hkv, Hv, D, rot, chunks;              // Hv: Hkv with a cache, else 0
  int pos_i64, slots_i64;
  float eps;
};

__device__ __forceinline__ float2 to_f2(uint32_t w, __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 to_f2(uint32_t w, __half*) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ uint32_t from_f2(float a, float b, __nv_bfloat16*) {
  __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t from_f2(float a, float b, __half*) {
  __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = to_f2(w[i], static_cast<T*>(nullptr));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  T* t = nullptr;
  return make_uint4(from_f2(f[0], f[1], t), from_f2(f[2], f[3], t), from_f2(f[4], f[5], t), from_f2(f[6], f[7], t));
}
__device__ __forceinline__ int64_t load_index(const void* p, int i64, int64_t i) {
  return i64 ? __ldg(static_cast<const long long*>(p) + i) : static_cast<int64_t>(__ldg(static_cast<const int*>(p) + i));
}

// The eight codes of one lane.  y / scale correctly rounded from the correctly rounded reciprocal (Markstein: exact for
// every scale whose significand is not all ones); rows with such a scale, a non-finite one or a NaN among the lane's
// elements take the literal fminf(fmaxf(y / scale, -448), 448), in which a NaN becomes -448.
__device__ __forceinline__ uint2 quantise8(const float (&y)[8], float scale) {
  const uint32_t bits = __float_as_uint(scale);
  bool literal = (bits & 0x007fffffu) == 0x007fffffu || (bits & 0x7f800000u) == 0x7f800000u;
  const float r = __frcp_rn(scale);
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q0 = __fmul_rn(y[i], r);
    const float rem = fmaf(q0, scale, -y[i]);
    t[i] = fmaf(-rem, r, q0);
    literal |= !(t[i] == t[i]);
  }
  if (literal) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(__fdiv_rn(y[i], scale), -448.f), 448.f);
  }
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(make_float2(t[2 * i], t[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// ROPE: 0 none, 1 neox, 2 neighbouring pairs.
template <typename T, int G, int U, int ROPE>
__global__ void __launch_bounds__(kThreads) head_rows_kernel(const __grid_constant__ HeadRowsParams p) {
  pdl_start();
  constexpr int RPW = 32 / G;
  const int lane = threadIdx.x & 31;
  const int l = lane % G, sub = lane / G;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = item / p.chunks;
  if (tok >= p.T) return;
  const int h0 = static_cast<int>(item - tok * p.chunks) * (RPW * U) + sub;
  const int H = p.Hq + p.Hkv + p.Hv;
  const bool in_row = l * 8 < p.D;

  int64_t pos = 0;
  if (ROPE != 0) {
    pos = load_index(p.positions, p.pos_i64, tok);
    if (pos < 0) return;                                    // padding: nothing of this token is read or written
  }
  int64_t slot = -1;
  if (p.Hv != 0) slot = load_index(p.slots, p.slots_i64, tok);
  const bool keep = slot >= 0 && slot < p.num_slots;

  uint4 data[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * RPW;
    data[u] = make_uint4(0, 0, 0, 0);
    const T* src = nullptr;
    if (h < p.Hq) src = static_cast<const T*>(p.q) + tok * p.q_st + h * p.q_sh;
    else if (h < p.Hq + p.Hkv) src = static_cast<const T*>(p.k) + tok * p.k_st + (h - p.Hq) * p.k_sh;
    else if (h < H) src = static_cast<const T*>(p.v) + tok * p.v_st + (h - p.Hq - p.Hkv) * p.v_sh;
    if (src != nullptr && in_row) data[u] = *reinterpret_cast<const uint4*>(src + l * 8);
  }
  // cosines and sines of this lane's elements
  float c[8], s[8];
  bool turned = false, second = false;
  int partner = lane;
  float poison = 1.f;
  if (ROPE != 0) {
    if (pos >= p.max_position) {                            // a position that the table lacks: NaN, not a read behind it
      poison = __uint_as_float(0x7fc00000u);
      pos = 0;
    }
    const float* row = p.cos_sin + pos * p.rot;
    const int half = p.rot / 2;
    turned = l * 8 < p.rot;
    if (ROPE == 1) {
      const int hl = half / 8;
      second = l >= hl;
      partner = turned ? lane + (second ? -hl : hl) : lane;
      if (turned) {
        const float4* cp = reinterpret_cast<const float4*>(row + (second ? l - hl : l) * 8);
        const float4* sp = reinterpret_cast<const float4*>(row + half + (second ? l - hl : l) * 8);
        const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
        c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
        s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
      }
    } else if (turned) {
      const float4 c0 = __ldg(reinterpret_cast<const float4*>(row + l * 4));
      const float4 s0 = __ldg(reinterpret_cast<const float4*>(row + half + l * 4));
      c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w;
      s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w;
    }
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * RPW;
    const bool is_q = h < p.Hq, is_k = !is_q && h < p.Hq + p.Hkv, is_v = !is_q && !is_k && h < H;
    float y[8];
    unpack8<T>(data[u], y);
    const void* w = is_q ? p.q_w : is_k ? p.k_w : nullptr;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(y[i], y[i], sq);
#pragma unroll
    for (int off = G / 2; off >= 1; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    if (w != nullptr && in_row) {
      const float rinv = rsqrtf(sq / static_cast<float>(p.D) + p.eps);
      float wf[8];
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + l * 8)), wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * rinv * wf[i];
    }
    if (ROPE == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = __shfl_sync(0xffffffffu, y[i], partner);
        if (turned && !is_v) y[i] = second ? fmaf(y[i], c[i], o * s[i]) : fmaf(y[i], c[i], -(o * s[i]));
      }
    } else if (ROPE == 2) {
      if (turned && !is_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = y[2 * i], b = y[2 * i + 1];
          y[2 * i] = fmaf(a, c[i], -(b * s[i]));
          y[2 * i + 1] = fmaf(b, c[i], a * s[i]);
        }
      }
    }
    if (ROPE != 0 && !is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= poison;
    }
    if (in_row) {
      T* dst = nullptr;
      if (is_q && p.q_out) dst = static_cast<T*>(p.q_out) + tok * p.qo_st + h * p.qo_sh;
      if (is_k && p.k_out) dst = static_cast<T*>(p.k_out) + tok * p.ko_st + (h - p.Hq) * p.ko_sh;
      if (dst != nullptr) *reinterpret_cast<uint4*>(dst + l * 8) = pack8<T>(y);
    }
    if (p.Hv != 0) {
      float amax = 1e-10f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
#pragma unroll
      for (int off = G / 2; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      if ((is_k || is_v) && keep && in_row) {
        const float scale = __fdiv_rn(amax, 448.f);
        const uint32_t page = static_cast<uint32_t>(slot) / p.page_size, at = static_cast<uint32_t>(slot) - page * p.page_size;
        const int hh = is_k ? h - p.Hq : h - p.Hq - p.Hkv;
        const int64_t* cs = is_k ? p.kc_s : p.vc_s;
        const int64_t* ss = is_k ? p.ks_s : p.vs_s;
        uint8_t* cache = (is_k ? p.kc : p.vc) + page * cs[0] + at * cs[1] + hh * cs[2];
        *reinterpret_cast<uint2*>(cache + l * 8) = quantise8(y, scale);
        if (l == 0) (is_k ? p.ks : p.vs)[page * ss[0] + at * ss[1] + hh * ss[2]] = is_k ? scale * poison : scale;
      }
    }
  }
}

template <typename T, int G, int U>
cudaError_t launch_rows(const HeadRowsParams& p, int rope, unsigned grid, cudaStream_t st) {
  switch (rope) {
    case 0: return launch_pdl(head_rows_kernel<T, G, U, 0>, dim3(grid), dim3(kThreads), 0, st, p);
    case 1: return launch_pdl(head_rows_kernel<T, G, U, 1>, dim3(grid), dim3(kThreads), 0, st, p);
    default: return launch_pdl(head_rows_kernel<T, G, U, 2>, dim3(grid), dim3(kThreads), 0, st, p);
  }
}

template <typename T, int G>
int go_rows(HeadRowsParams p, int rope, cudaStream_t st) {
  const int H = p.Hq + p.Hkv + p.Hv, sms = sm_count();
  if (sms <= 0) return B200_ERR_CUDA;
  constexpr int RPW = 32 / G, WPB = kThreads / 32;
  auto chunks = [&](int u) { return (H + RPW * u - 1) / (RPW * u); };
  // four rows a lane group where that still gives every SM sixteen warps; otherwise one, for latency
  const bool wide = p.T * chunks(4) >= 16LL * sms;
  p.chunks = chunks(wide ? 4 : 1);
  const int64_t blocks = (p.T * p.chunks + WPB - 1) / WPB;
  if (blocks > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  B200_CUDA_TRY(wide ? (launch_rows<T, G, 4>(p, rope, static_cast<unsigned>(blocks), st))
                     : (launch_rows<T, G, 1>(p, rope, static_cast<unsigned>(blocks), st)));
  return B200_OK;
}

template <typename T>
int dispatch_rows(const HeadRowsParams& p, int rope, cudaStream_t st) {
  if (p.D <= 32) return go_rows<T, 4>(p, rope, st);
  if (p.D <= 64) return go_rows<T, 8>(p, rope, st);
  if (p.D <= 128) return go_rows<T, 16>(p, rope, st);
  return go_rows<T, 32>(p, rope, st);
}

int take_heads(const b200_heads* h, int64_t T, int H, const void** ptr, int64_t* st, int64_t* sh) {
  if (!h) return B200_OK;
  if (!h->ptr) return B200_ERR_NULL_PTR;
  if (!aligned16(h->ptr) || h->stride_token % 8 != 0 || h->stride_head % 8 != 0) return B200_ERR_MISALIGNED;
  if (h->stride_token < 0 || h->stride_head < 0) return B200_ERR_BAD_STRIDE;
  *ptr = h->ptr;
  *st = h->stride_token;
  *sh = h->stride_head;
  return B200_OK;
}

int check_cache(const b200_kv_cache* c) {
  if (c->num_pages < 0 || c->page_size <= 0) return B200_ERR_BAD_SHAPE;
  if (c->page_size > 0x7fffffffLL || c->num_pages > 0x7fffffffLL / c->page_size) return B200_ERR_TOO_LARGE;
  if (c->num_pages > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return B200_ERR_NULL_PTR;
  if (!aligned16(c->k) || !aligned16(c->v)) return B200_ERR_MISALIGNED;
  for (int i = 0; i < 3; ++i) {
    if (c->k_stride[i] < 0 || c->v_stride[i] < 0 || c->k_scale_stride[i] < 0 || c->v_scale_stride[i] < 0) return B200_ERR_BAD_STRIDE;
    if (c->k_stride[i] % 16 != 0 || c->v_stride[i] % 16 != 0) return B200_ERR_MISALIGNED;
  }
  return B200_OK;
}

// ------------------------------------------------------------------------------------------ the cache read back
struct KvLoadParams {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int64_t kc_s[3], vc_s[3], ks_s[3], vs_s[3];
  const int32_t *page_table, *indptr, *starts;
  int64_t table_stride, tokens;
  void *k_out, *v_out;
  int64_t ko_st, ko_sh, vo_st, vo_sh;
  uint32_t num_pages, page_size, table_cols;
  int batch, Hkv, D;
};

constexpr int kLoadThreads = 256, kLoadTokens = 16, kLoadUnroll = 4;

// out[i] = code * scale for the tokens of all sequences, packed: row i belongs to the sequence b with
// indptr[b] <= i < indptr[b + 1] and holds its token starts[b] + i - indptr[b].  A block takes kLoadTokens rows of keys or of
// values (blockIdx.y).  Its first warp finds the rows' places: the sequence of the first by a 32-way search of indptr, those
// of the others by walking on from there.  Then each thread turns 16 codes (one 16-byte load) into 32 bytes at a time, four
// of them in flight.
template <typename T>
__global__ void __launch_bounds__(kLoadThreads) kv_load_kernel(const __grid_constant__ KvLoadParams p) {
  pdl_start();
  __shared__ int s_page[kLoadTokens], s_at[kLoadTokens];      // page -1: behind the last sequence; -2: no such page
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kLoadTokens;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int lo = 0, n = p.batch;                                  // the answer is lo + (entries of the n from lo on that are <= row0)
    while (n > 0) {
      const int step = (n + 31) / 32;
      const int probe = lo + (lane + 1) * step - 1;           // last of this lane's `step` entries
      const bool le = probe < lo + n && __ldg(p.indptr + 1 + probe) <= row0;
      const int whole = __popc(__ballot_sync(0xffffffffu, le));
      lo += whole * step;
      n = step > 1 ? min(step - 1, n - whole * step) : 0;
    }
    const int64_t row = row0 + lane;
    if (lane < kLoadTokens) {
      int page = -1, at = 0;
      if (row < p.tokens) {
        int b = lo;
        while (b < p.batch && __ldg(p.indptr + 1 + b) <= row) ++b;
        const int first = b < p.batch ? __ldg(p.indptr + b) : 0;
        if (b < p.batch && first <= row) {
          const int64_t t = row - first + (p.starts ? __ldg(p.starts + b) : 0);
          const int64_t col = t >= 0 ? t / p.page_size : -1;
          page = -2;
          if (col >= 0 && col < p.table_cols) {
            const int id = __ldg(p.page_table + b * p.table_stride + col);
            if (id >= 0 && static_cast<uint32_t>(id) < p.num_pages) {
              page = id;
              at = static_cast<int>(t - col * p.page_size);
            }
          }
        }
      }
      s_page[lane] = page;
      s_at[lane] = at;
    }
  }
  __syncthreads();
  const bool keys = blockIdx.y == 0;
  const uint8_t* cache = keys ? p.kc : p.vc;
  const float* scales = keys ? p.ks : p.vs;
  const int64_t* cs = keys ? p.kc_s : p.vc_s;
  const int64_t* ss = keys ? p.ks_s : p.vs_s;
  T* out = static_cast<T*>(keys ? p.k_out : p.v_out);
  const int64_t st = keys ? p.ko_st : p.vo_st, sh = keys ? p.ko_sh : p.vo_sh;
  const int per_head = p.D / 16, vecs = p.Hkv * per_head, total = vecs * kLoadTokens;
  for (int base = threadIdx.x; base < total; base += kLoadThreads * kLoadUnroll) {
    uint4 codes[kLoadUnroll];
    float scale[kLoadUnroll];
    T* dst[kLoadUnroll];
#pragma unroll
    for (int u = 0; u < kLoadUnroll; ++u) {
      const int i = base + u * kLoadThreads;
      dst[u] = nullptr;
      if (i >= total) continue;
      const int r = i / vecs, v = i - r * vecs, h = v / per_head, d = (v - h * per_head) * 16;
      const int page = s_page[r];
      if (page == -1) continue;
      dst[u] = out + (row0 + r) * st + h * sh + d;
      codes[u] = make_uint4(0, 0, 0, 0);
      scale[u] = __uint_as_float(0x7fc00000u);                // a page that does not exist reads as NaN
      if (page >= 0) {
        codes[u] = __ldcs(reinterpret_cast<const uint4*>(cache + page * cs[0] + s_at[r] * cs[1] + h * cs[2] + d));
        scale[u] = __ldg(scales + page * ss[0] + s_at[r] * ss[1] + h * ss[2]);
      }
    }
#pragma unroll
    for (int u = 0; u < kLoadUnroll; ++u) {
      if (dst[u] == nullptr) continue;
      const uint32_t w[4] = {codes[u].x, codes[u].y, codes[u].z, codes[u].w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
        o[i] = from_f2(f.x * scale[u], f.y * scale[u], static_cast<T*>(nullptr));
      }
      reinterpret_cast<uint4*>(dst[u])[0] = make_uint4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<uint4*>(dst[u])[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

int rows_entry(const b200_heads* q, const b200_heads* k, const b200_heads* v, const b200_heads* q_out, const b200_heads* k_out,
               int dtype, const void* positions, int positions_i64, const float* cos_sin, int64_t max_position,
               int rotary_dim, int is_neox, const void* q_weight, const void* k_weight, float norm_eps,
               const b200_kv_cache* cache, const void* slots, int slots_i64, int64_t T, int Hq, int Hkv, int D, void* stream) {
  if (T < 0 || Hq < 0 || Hkv < 0 || D <= 0 || D % 16 != 0) return B200_ERR_BAD_SHAPE;
  if (D > 256 || Hq > (1 << 20) || Hkv > (1 << 20)) return B200_ERR_TOO_LARGE;
  if (dtype != B200_DT_BF16 && dtype != B200_DT_F16) return B200_ERR_BAD_DTYPE;
  if (cos_sin && (rotary_dim <= 0 || rotary_dim > D || rotary_dim % 16 != 0 || max_position < 0)) return B200_ERR_BAD_SHAPE;
  HeadRowsParams p = {};
  if (cache) {
    const int rc = check_cache(cache);
    if (rc != B200_OK) return rc;
  }
  p.Hq = Hq, p.Hkv = Hkv, p.Hv = cache ? Hkv : 0, p.D = D;
  if (T == 0 || Hq + Hkv == 0) return B200_OK;
  if ((Hq > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || (cache ? !v || !slots : !k_out))) || (cos_sin && !positions))
    return B200_ERR_NULL_PTR;
  const void *qo = nullptr, *ko = nullptr;
  int rc;
  if (Hq > 0) {
    if ((rc = take_heads(q, T, Hq, &p.q, &p.q_st, &p.q_sh)) != B200_OK) return rc;
    if ((rc = take_heads(q_out, T, Hq, &qo, &p.qo_st, &p.qo_sh)) != B200_OK) return rc;
  }
  if (Hkv > 0) {
    if ((rc = take_heads(k, T, Hkv, &p.k, &p.k_st, &p.k_sh)) != B200_OK) return rc;
    if ((rc = take_heads(k_out, T, Hkv, &ko, &p.ko_st, &p.ko_sh)) != B200_OK) return rc;
    if (cache && (rc = take_heads(v, T, Hkv, &p.v, &p.v_st, &p.v_sh)) != B200_OK) return rc;
  }
  if ((cos_sin && !aligned16(cos_sin)) || !aligned16(q_weight) || !aligned16(k_weight)) return B200_ERR_MISALIGNED;
  p.q_out = const_cast<void*>(qo);
  p.k_out = const_cast<void*>(ko);
  p.q_w = q_weight, p.k_w = k_weight, p.eps = norm_eps;
  p.positions = positions, p.pos_i64 = positions_i64;
  p.cos_sin = cos_sin, p.max_position = max_position, p.rot = rotary_dim;
  p.T = T, p.page_size = 1;
  if (cache) {
    p.slots = slots, p.slots_i64 = slots_i64;
    p.kc = static_cast<uint8_t*>(cache->k), p.vc = static_cast<uint8_t*>(cache->v);
    p.ks = cache->k_scale, p.vs = cache->v_scale;
    for (int i = 0; i < 3; ++i)
      p.kc_s[i] = cache->k_stride[i], p.vc_s[i] = cache->v_stride[i], p.ks_s[i] = cache->k_scale_stride[i], p.vs_s[i] = cache->v_scale_stride[i];
    p.page_size = static_cast<uint32_t>(cache->page_size);
    p.num_slots = static_cast<uint32_t>(cache->num_pages * cache->page_size);
  }
  const int rope = cos_sin ? (is_neox ? 1 : 2) : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B200_DT_BF16 ? dispatch_rows<__nv_bfloat16>(p, rope, st) : dispatch_rows<__half>(p, rope, st);
}

}  // namespace
}  // namespace b200

extern "C" int b200_qk_norm_rope(const b200_heads* q, const b200_heads* k, const b200_heads* q_out, const b200_heads* k_out,
                                 int dtype, const void* positions, int positions_i64, const float* cos_sin,
                                 int64_t max_position, int rotary_dim, int is_neox, const void* q_weight,
                                 const void* k_weight, float norm_eps, int64_t T, int num_q_heads, int num_kv_heads,
                                 int head_dim, void* stream) {
  return b200::rows_entry(q, k, nullptr, q_out, k_out, dtype, positions, positions_i64, cos_sin, max_position, rotary_dim, is_neox,
                          q_weight, k_weight, norm_eps, nullptr, nullptr, 0, T, num_q_heads, num_kv_heads, head_dim, stream);
}

extern "C" int b200_store_kv_fp8(const b200_heads* k, const b200_heads* v, int dtype, const b200_kv_cache* cache,
                                 const void* slots, int slots_i64, int64_t T, int num_kv_heads, int head_dim, void* stream) {
  if (!cache) return B200_ERR_NULL_PTR;
  return b200::rows_entry(nullptr, k, v, nullptr, nullptr, dtype, nullptr, 0, nullptr, 0, 0, 1, nullptr, nullptr, 0.f, cache, slots,
                          slots_i64, T, 0, num_kv_heads, head_dim, stream);
}

extern "C" int b200_qk_norm_rope_store_kv_fp8(const b200_heads* q, const b200_heads* k, const b200_heads* v,
                                              const b200_heads* q_out, const b200_heads* k_out, int dtype,
                                              const void* positions, int positions_i64, const float* cos_sin,
                                              int64_t max_position, int rotary_dim, int is_neox, const void* q_weight,
                                              const void* k_weight, float norm_eps, const b200_kv_cache* cache,
                                              const void* slots, int slots_i64, int64_t T, int num_q_heads,
                                              int num_kv_heads, int head_dim, void* stream) {
  if (!cache) return B200_ERR_NULL_PTR;
  return b200::rows_entry(q, k, v, q_out, k_out, dtype, positions, positions_i64, cos_sin, max_position, rotary_dim, is_neox, q_weight,
                          k_weight, norm_eps, cache, slots, slots_i64, T, num_q_heads, num_kv_heads, head_dim, stream);
}

extern "C" int b200_load_kv_fp8(const b200_kv_cache* cache, const int32_t* page_table, int64_t page_table_stride,
                                int64_t page_table_cols, const int32_t* indptr, const int32_t* starts, int64_t batch,
                                const b200_heads* k_out, const b200_heads* v_out, int dtype, int64_t tokens,
                                int num_kv_heads, int head_dim, void* stream) {
  using namespace b200;
  if (!cache) return B200_ERR_NULL_PTR;
  if (tokens < 0 || batch < 0 || num_kv_heads < 0 || head_dim <= 0 || head_dim % 16 != 0 || page_table_cols < 0)
    return B200_ERR_BAD_SHAPE;
  if (head_dim > 256 || num_kv_heads > (1 << 16) || batch > (1 << 24) || page_table_cols > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  if (dtype != B200_DT_BF16 && dtype != B200_DT_F16) return B200_ERR_BAD_DTYPE;
  int rc = check_cache(cache);
  if (rc != B200_OK) return rc;
  if (tokens == 0 || batch == 0 || num_kv_heads == 0) return B200_OK;
  if (!page_table || !indptr || !k_out || !v_out) return B200_ERR_NULL_PTR;
  if (page_table_stride < 0) return B200_ERR_BAD_STRIDE;
  KvLoadParams p = {};
  const void *ko = nullptr, *vo = nullptr;
  if ((rc = take_heads(k_out, tokens, num_kv_heads, &ko, &p.ko_st, &p.ko_sh)) != B200_OK) return rc;
  if ((rc = take_heads(v_out, tokens, num_kv_heads, &vo, &p.vo_st, &p.vo_sh)) != B200_OK) return rc;
  p.k_out = const_cast<void*>(ko), p.v_out = const_cast<void*>(vo);
  p.kc = static_cast<const uint8_t*>(cache->k), p.vc = static_cast<const uint8_t*>(cache->v);
  p.ks = cache->k_scale, p.vs = cache->v_scale;
  for (int i = 0; i < 3; ++i)
    p.kc_s[i] = cache->k_stride[i], p.vc_s[i] = cache->v_stride[i], p.ks_s[i] = cache->k_scale_stride[i], p.vs_s[i] = cache->v_scale_stride[i];
  p.page_table = page_table, p.table_stride = page_table_stride, p.table_cols = static_cast<uint32_t>(page_table_cols);
  p.indptr = indptr, p.starts = starts, p.batch = static_cast<int>(batch), p.tokens = tokens;
  p.num_pages = static_cast<uint32_t>(cache->num_pages), p.page_size = static_cast<uint32_t>(cache->page_size);
  p.Hkv = num_kv_heads, p.D = head_dim;
  const int64_t blocks = (tokens + kLoadTokens - 1) / kLoadTokens;
  if (blocks > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  B200_CUDA_TRY(dtype == B200_DT_BF16 ? launch_pdl(kv_load_kernel<__nv_bfloat16>, grid, dim3(kLoadThreads), 0, st, p)
                                      : launch_pdl(kv_load_kernel<__half>, grid, dim3(kLoadThreads), 0, st, p));
  return B200_OK;
}
