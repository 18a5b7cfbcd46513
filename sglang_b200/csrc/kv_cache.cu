// Between the qkv projection and the attention kernel, for sm_100a: RMSNorm of every query and key head, the rotary
// position embedding, keys and values quantised into a paged cache, and the cache read back.  All of it moves data: the
// floor is the bytes read and written once, at the memory's rate.
//
// One head of one token ("row", D elements) belongs to a group of G lanes, G the power of two from D / 16 up, each lane
// holding sixteen elements in two 16-byte loads.  What a row needs beyond its lane is a shuffle inside its group: the sum of
// squares and the largest magnitude.  A warp keeps to one token and to queries, keys or values: weights, cosines and sines
// stay in registers while it walks over its rows, 32 / G at a time, the next ones on their way into shared memory.  All arithmetic is in 32 bits; a
// query is rounded once, when it is stored, and a key once, to e4m3.
//
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)     neox: b = a + rot / 2; otherwise neighbours a = 2i, b = 2i + 1
//   scale = max(1e-10, max|y|) / 448,  code = e4m3(y / scale)     correctly rounded quotient, as in the group quantiser
#include "gemm_common.cuh"

namespace b200 {
namespace {

constexpr int kMaxThreads = 64;

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
  int Hq, Hkv, Hv, D, rot;                      // Hv: Hkv with a cache, else 0
  uint32_t chunks_magic, heads_magic;           // 2^32 / chunks and 2^32 / Hkv, rounded up
  int page_shift;                               // page_size = 1 << page_shift, or -1
  int chunks, chunks_q, chunks_kv;              // warps a token; of them for queries, and for keys (as many for values)
  int heads_q, heads_kv;                        // of one warp
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
// Two fp32 numbers in one 64-bit register pair: one instruction does both.
struct f2 {
  unsigned long long v;
};
__device__ __forceinline__ f2 make_f2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f2 both(float a) { return make_f2(a, a); }
__device__ __forceinline__ float2 split(f2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ f2 mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// The sixteen elements of two vectors as eight pairs: (2e, 2e + 1); or, TURNED, first elements 4e and 4e + 2, then elements 4e + 1
// and 4e + 3, so that neighbours which are rotated with one another lie in the same half of two pairs.
template <typename T, bool TURNED>
__device__ __forceinline__ void unpack16(const uint4& lo, const uint4& hi, f2 (&f)[8]) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 p = to_f2(w[i], static_cast<T*>(nullptr)), q = to_f2(w[i + 1], static_cast<T*>(nullptr));
    f[TURNED ? i / 2 : i] = TURNED ? make_f2(p.x, q.x) : make_f2(p.x, p.y);
    f[TURNED ? i / 2 + 4 : i + 1] = TURNED ? make_f2(p.y, q.y) : make_f2(q.x, q.y);
  }
}
// Back in order: pair i of the elements.
template <bool TURNED>
__device__ __forceinline__ float2 pair_of(const f2 (&f)[8], int i) {
  if (!TURNED) return split(f[i]);
  const float2 a = split(f[i / 2]), b = split(f[i / 2 + 4]);
  return i % 2 == 0 ? make_float2(a.x, b.x) : make_float2(a.y, b.y);
}
template <typename T, bool TURNED>
__device__ __forceinline__ uint4 pack8(const f2 (&f)[8], int half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = pair_of<TURNED>(f, 4 * half + i);
    w[i] = from_f2(p.x, p.y, static_cast<T*>(nullptr));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int64_t load_index(const void* p, int i64, int64_t i) {
  return i64 ? __ldg(static_cast<const long long*>(p) + i) : static_cast<int64_t>(__ldg(static_cast<const int*>(p) + i));
}

// amax / 448, correctly rounded: from the correctly rounded 1 / 448 and the exact remainder (Markstein).
__device__ __forceinline__ float scale_of(float amax) {
  const float r = 1.f / 448.f, q0 = __fmul_rn(amax, r);
  const float q = fmaf(fmaf(-q0, 448.f, amax), r, q0);
  return amax < __uint_as_float(0x7f800000u) ? q : amax;
}

// The sixteen codes of one lane.  y / scale correctly rounded from the correctly rounded reciprocal in the same way, which holds
// for every scale whose significand is not all ones; with such a scale, a non-finite one or a NaN among the lane's elements the
// quotients are taken literally.  Computed as -(y / scale), q0 = y (-r), q0 + (y + q0 scale)(-r), and the codes' signs flipped:
// in this form a zero keeps its sign.
template <bool TURNED>
__device__ __forceinline__ uint4 quantise16(const f2 (&y)[8], float scale) {
  const uint32_t bits = __float_as_uint(scale);
  bool literal = (bits & 0x007fffffu) == 0x007fffffu || (bits & 0x7f800000u) == 0x7f800000u;
  const f2 nr = both(-__frcp_rn(scale)), s = both(scale);
  f2 t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const f2 q0 = mul(y[i], nr);
    t[i] = fma(fma(q0, s, y[i]), nr, q0);
  }
  uint32_t w[4], nan = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(pair_of<TURNED>(t, 2 * i), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(pair_of<TURNED>(t, 2 * i + 1), __NV_SATFINITE, __NV_E4M3);
    w[i] = (lo | (hi << 16)) ^ 0x80808080u;
    nan |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;               // bit 7 of a byte: its code was 0x7f or 0xff
  }
  literal |= (nan & 0x80808080u) != 0;
  if (literal) {                                             // fminf(fmaxf(y / scale, -448), 448): a NaN becomes -448
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[2 * i] = pair_of<TURNED>(y, i).x, v[2 * i + 1] = pair_of<TURNED>(y, i).y;
#pragma unroll 1
    for (int i = 0; i < 16; ++i) v[i] = fminf(fmaxf(__fdiv_rn(v[i], scale), -448.f), 448.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// max(1e-10, the largest magnitude of a row), in all of its lanes.
template <int G>
__device__ __forceinline__ float largest(const f2 (&y)[8]) {
  float amax = 1e-10f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 v = split(y[e]);
    amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
  }
#pragma unroll
  for (int off = G / 2; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  return amax;
}

constexpr int kStages = 4, kStageBytes = 32 * 32;            // row groups in flight for each warp

// The rows of a warp: heads first ... last - 1 of one token's queries, keys or values.
template <typename T>
struct Rows {
  const T* src;              // head 0 of the token
  int64_t src_sh;
  T* dst;                    // or nullptr
  int64_t dst_sh;
  const T* weight;           // or nullptr
  int first, last;
};

// How a row is treated: taken as it is, normalised (if there is a weight) and not rotated, rotated as neox pairs, rotated as
// neighbouring pairs.
enum { kRaw = -1, kNorm = 0, kNeox = 1, kPairs = 2 };

// A lane holds two runs of eight elements, half of the row apart: a group's 16-byte accesses are then neighbours (with sixteen
// elements in one run every access took half of a sector, and 8192 tokens of 36 heads 36.8 us).  With neox pairs the runs are half
// of the rotated part apart, so that a rotation stays inside the lane, and half of the rest in the rest.
// pos: the token's position (none given: 0); slot: its place in the cache (CODES); both were loaded ahead and are looked at only
// when the first rows are under way.
template <typename T, int G, int KIND, bool STORE, bool CODES>
__device__ __forceinline__ void do_rows(const HeadRowsParams& p, const Rows<T>& r, uint32_t ring, int lane, int64_t pos, int64_t slot,
                                        bool keys) {
  constexpr int RPW = 32 / G;
  const int D = p.D, rot = p.rot;
  constexpr bool SPLIT = KIND == kNeox, TURNED = KIND == kPairs, ROPE = SPLIT || TURNED;
  const int l = lane % G, sub = lane / G;
  const bool in_row = l * 16 < D;
  // the lane's two runs of eight, and whether each is rotated
  const bool tail = SPLIT && l * 16 >= rot;
  const int o0 = tail ? rot + 8 * (l - rot / 16) : 8 * l;
  const int o1 = o0 + (SPLIT ? (tail ? D - rot : rot) / 2 : D / 2);
  const bool turn0 = ROPE && (SPLIT ? !tail : o0 < rot), turn1 = ROPE && (SPLIT ? !tail : o1 < rot);
  const float inv_d = 1.f / static_cast<float>(D);
  // ring: this lane's 32 bytes of each of the next kStages row groups; only the lane itself reads them.  A lane behind the end of
  // its rows has zeros there from the start.
  const uint32_t ring_end = ring + kStages * kStageBytes;
  const int heads = in_row ? r.last - r.first - sub : 0;      // of this lane's, counted by RPW
  if (!in_row)
    for (uint32_t at = ring; at != ring_end; at += kStageBytes / 2)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
  const T* src = r.src + (r.first + sub) * r.src_sh + o0;
  const int64_t src_step = RPW * r.src_sh;
  const int run = o1 - o0;
  uint32_t to = ring;
  auto fetch = [&](int i) {                                   // row group i / RPW
    sa::cp_async16_if(to, src, i < heads);
    sa::cp_async16_if(to + kStageBytes / 2, src + run, i < heads);
    src += src_step;
    to = to + kStageBytes == ring_end ? ring : to + kStageBytes;
  };
  const int count = r.last - r.first;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i * RPW < count) fetch(i * RPW);
    sa::cp_async_commit();
  }
  const bool poisoned = ROPE && pos >= p.max_position;         // a position that the table lacks: NaN, not a read behind it
  const bool keep = CODES && slot >= 0 && slot < p.num_slots;
  if (pos < 0 || !(keep || (STORE && r.dst != nullptr))) {     // padding, or nowhere to go: nothing is written
    sa::cp_async_wait<0>();
    return;
  }
  const float* table_row = ROPE ? p.cos_sin + pos * rot : nullptr;
  // A weight times an element is exact in fp32 (both have at most 11 significant bits), so it comes first; rsqrt(...) comes last.  Where
  // the position is not in the table, all factors are NaN.
  const float nan_or_1 = poisoned ? __uint_as_float(0x7fc00000u) : 1.f;
  f2 w[8], cs[4], sn[4], neg_sn[4];
  if (KIND != kRaw) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = both(nan_or_1);
    if (r.weight != nullptr && in_row && !poisoned)
      unpack16<T, TURNED>(__ldg(reinterpret_cast<const uint4*>(r.weight + o0)), __ldg(reinterpret_cast<const uint4*>(r.weight + o1)), w);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float4 c = make_float4(nan_or_1, nan_or_1, nan_or_1, nan_or_1), s = c;
      if (!poisoned && (i == 0 ? turn0 : turn1)) {
        const float* at = table_row + (SPLIT ? 8 * l + 4 * i : (i == 0 ? o0 : o1) / 2);
        c = __ldg(reinterpret_cast<const float4*>(at));
        s = __ldg(reinterpret_cast<const float4*>(at + rot / 2));
      }
      cs[2 * i] = make_f2(c.x, c.y), cs[2 * i + 1] = make_f2(c.z, c.w);
      sn[2 * i] = make_f2(s.x, s.y), sn[2 * i + 1] = make_f2(s.z, s.w);
      neg_sn[2 * i] = make_f2(-s.x, -s.y), neg_sn[2 * i + 1] = make_f2(-s.z, -s.w);
    }
  }
  T* dst = STORE && r.dst != nullptr ? r.dst + (r.first + sub) * r.dst_sh : nullptr;
  const int64_t dst_step = RPW * r.dst_sh;
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  int64_t codes_step = 0, scales_step = 0;
  if (CODES && keep) {
    const uint32_t page = p.page_shift >= 0 ? static_cast<uint32_t>(slot) >> p.page_shift : static_cast<uint32_t>(slot) / p.page_size;
    const uint32_t place = static_cast<uint32_t>(slot) - page * p.page_size;
    const int64_t *cs = keys ? p.kc_s : p.vc_s, *ss = keys ? p.ks_s : p.vs_s;
    codes = (keys ? p.kc : p.vc) + page * cs[0] + place * cs[1] + (r.first + sub) * cs[2];
    scales = (keys ? p.ks : p.vs) + page * ss[0] + place * ss[1] + (r.first + sub) * ss[2];
    codes_step = RPW * cs[2], scales_step = RPW * ss[2];
  }
  uint32_t from = ring;
#pragma unroll 1
  for (int i = 0; i < count; i += RPW) {
    if (i + (kStages - 1) * RPW < count) fetch(i + (kStages - 1) * RPW);
    sa::cp_async_commit();
    sa::cp_async_wait<kStages - 1>();
    const bool live = i < heads;
    f2 y[8];
    unpack16<T, TURNED>(sa::ld_v4(from), sa::ld_v4(from + kStageBytes / 2), y);
    from = from + kStageBytes == ring_end ? ring : from + kStageBytes;
    if (KIND != kRaw) {
      f2 rinv = both(1.f);
      if (r.weight != nullptr) {
        f2 sum = mul(y[0], y[0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) sum = fma(y[e], y[e], sum);
        float sq = split(sum).x + split(sum).y;
#pragma unroll
        for (int off = G / 2; off >= 1; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
        rinv = both(rsqrtf(fmaf(sq, inv_d, p.eps)));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = mul(y[e], w[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {                            // with neighbouring pairs 0 and 1 are the first run's, 2 and 3 the second's
        if (!(e < 2 ? turn0 : turn1)) continue;
        const f2 a = y[e], b = y[e + 4];
        y[e] = fma(a, cs[e], mul(b, neg_sn[e]));
        y[e + 4] = fma(b, cs[e], mul(a, sn[e]));
      }
      if (r.weight != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = mul(y[e], rinv);
      }
    }
    if (STORE && dst != nullptr) {
      if (live) {
        *reinterpret_cast<uint4*>(dst + o0) = pack8<T, TURNED>(y, 0);
        *reinterpret_cast<uint4*>(dst + o1) = pack8<T, TURNED>(y, 1);
      }
      dst += dst_step;
    }
    if (CODES) {
      const float scale = scale_of(largest<G>(y));
      const uint4 q = quantise16<TURNED>(y, scale);
      if (live && keep) {
        *reinterpret_cast<uint2*>(codes + o0) = make_uint2(q.x, q.y);
        *reinterpret_cast<uint2*>(codes + o1) = make_uint2(q.z, q.w);
        if (l == 0) *scales = KIND != kRaw && poisoned ? __uint_as_float(0x7fc00000u) : scale;
      }
      codes += codes_step;
      scales += scales_step;
    }
  }
}

// Keys and values taken as they are, of few heads: rows counted through all tokens and heads, `steps` groups of RPW neighbouring ones
// a warp.  With warps that keep to one token the rate at which blocks start bounds it, whatever the heads.
template <typename T, int G>
__global__ void __launch_bounds__(kMaxThreads, 11) store_rows_kernel(const __grid_constant__ HeadRowsParams p, uint32_t rows, uint32_t warps,
                                                                     int steps) {
  pdl_start();
  constexpr int RPW = 32 / G;
  extern __shared__ __align__(16) uint8_t rings[];
  const int lane = threadIdx.x & 31, l = lane % G, H = p.Hkv;
  const uint32_t item = blockIdx.x * (kMaxThreads / 32) + (threadIdx.x >> 5);
  if (item >= 2 * warps) return;
  const bool keys = item < warps, in_row = l * 16 < p.D;
  const uint32_t row = (keys ? item : item - warps) * (steps * RPW) + lane / G;    // this lane's first
  const int mine = in_row && row < rows ? static_cast<int>((rows - row + RPW - 1) / RPW) : 0;      // and how many it may have
  uint32_t t = H == 1 ? row : __umulhi(row, p.heads_magic);                        // row / H, or one more
  if (t * H > row) --t;
  int head = static_cast<int>(row - t * H);
  const int o0 = 8 * l, run = p.D / 2;
  const uint32_t ring = smem_u32(rings) + (threadIdx.x >> 5) * (kStages * kStageBytes) + lane * 16, ring_end = ring + kStages * kStageBytes;
  if (!in_row)
    for (uint32_t at = ring; at != ring_end; at += kStageBytes / 2)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
  const int64_t st = keys ? p.k_st : p.v_st, sh = keys ? p.k_sh : p.v_sh, step = RPW * sh, wrap = st - H * sh;
  const T* src = static_cast<const T*>(keys ? p.k : p.v) + t * st + head * sh + o0;
  int fetched = head;
  uint32_t to = ring, from = ring;
  auto fetch = [&](int i) {
    sa::cp_async16_if(to, src, i < mine);
    sa::cp_async16_if(to + kStageBytes / 2, src + run, i < mine);
    src += step;
    for (fetched += RPW; fetched >= H; fetched -= H) src += wrap;
    to = to + kStageBytes == ring_end ? ring : to + kStageBytes;
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < steps) fetch(i);
    sa::cp_async_commit();
  }
  auto slot_of = [&](int i) { return i < mine ? load_index(p.slots, p.slots_i64, t) : -1; };
  int64_t slot = slot_of(0);
  uint8_t* const cache = (keys ? p.kc : p.vc) + o0;
  float* const scales = keys ? p.ks : p.vs;
  const int64_t *cs = keys ? p.kc_s : p.vc_s, *ss = keys ? p.ks_s : p.vs_s;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    if (i + kStages - 1 < steps) fetch(i + kStages - 1);
    sa::cp_async_commit();
    const bool keep = slot >= 0 && slot < p.num_slots;
    const uint32_t at = static_cast<uint32_t>(slot), page = p.page_shift >= 0 ? at >> p.page_shift : at / p.page_size, place = at - page * p.page_size;
    const int h = head;
    for (head += RPW; head >= H; head -= H) ++t;
    slot = slot_of(i + 1 < steps ? i + 1 : mine);                    // a step ahead
    sa::cp_async_wait<kStages - 1>();
    f2 y[8];
    unpack16<T, false>(sa::ld_v4(from), sa::ld_v4(from + kStageBytes / 2), y);
    from = from + kStageBytes == ring_end ? ring : from + kStageBytes;
    const float scale = scale_of(largest<G>(y));
    const uint4 q = quantise16<false>(y, scale);
    if (keep) {
      uint8_t* codes = cache + page * cs[0] + place * cs[1] + h * cs[2];
      *reinterpret_cast<uint2*>(codes) = make_uint2(q.x, q.y);
      *reinterpret_cast<uint2*>(codes + run) = make_uint2(q.z, q.w);
      if (l == 0) scales[page * ss[0] + place * ss[1] + h * ss[2]] = scale;
    }
  }
}

// Eleven blocks of two warps: 80 registers, and the rotating kinds spill (up to 96 bytes stored and 52 loaded a thread).
// With ten nothing spills (95 registers) and there are two warps fewer: 54.3 -> 57.7 us for 8192 tokens of 64 + 8 + 8 heads of 128,
// 27.4 -> 29.0 for 8192 of 32 + 4 with pairs rotated, 16.9 -> 17.7 for 2048; only a batch of 64 gains, 2.9 -> 2.7.
template <typename T, int G, int KIND>
__global__ void __launch_bounds__(kMaxThreads, 11) head_rows_kernel(const __grid_constant__ HeadRowsParams p) {
  pdl_start();
  constexpr bool ROPE = KIND == kNeox || KIND == kPairs;
  extern __shared__ __align__(16) uint8_t rings[];
  const int lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(rings) + (threadIdx.x >> 5) * (kStages * kStageBytes) + lane * 16;
  const uint32_t item = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
  uint32_t tok32 = p.chunks == 1 ? item : __umulhi(item, p.chunks_magic);      // item / chunks, or one more
  if (tok32 * p.chunks > item) --tok32;
  if (tok32 >= p.T) return;
  const int64_t tok = tok32;
  int chunk = static_cast<int>(item - tok32 * p.chunks);
  const int64_t pos = ROPE || (KIND == kNorm && p.positions != nullptr) ? load_index(p.positions, p.pos_i64, tok) : 0;
  const int64_t slot = p.Hv != 0 && chunk >= p.chunks_q ? load_index(p.slots, p.slots_i64, tok) : -1;
  Rows<T> r = {};
  if (chunk < p.chunks_q) {
    r.first = chunk * p.heads_q, r.last = min(r.first + p.heads_q, p.Hq);
    r.src = static_cast<const T*>(p.q) + tok * p.q_st, r.src_sh = p.q_sh;
    r.dst = static_cast<T*>(p.q_out) + tok * p.qo_st, r.dst_sh = p.qo_sh;
    r.weight = static_cast<const T*>(p.q_w);
    do_rows<T, G, KIND, true, false>(p, r, ring, lane, pos, -1, false);
    return;
  }
  chunk -= p.chunks_q;
  const bool keys = chunk < p.chunks_kv;
  r.first = (keys ? chunk : chunk - p.chunks_kv) * p.heads_kv, r.last = min(r.first + p.heads_kv, p.Hkv);
  r.src = keys ? static_cast<const T*>(p.k) + tok * p.k_st : static_cast<const T*>(p.v) + tok * p.v_st;
  r.src_sh = keys ? p.k_sh : p.v_sh;
  if constexpr (KIND == kRaw) {
    do_rows<T, G, kRaw, false, true>(p, r, ring, lane, 0, slot, keys);
  } else if (keys) {
    if (p.k_out != nullptr) r.dst = static_cast<T*>(p.k_out) + tok * p.ko_st, r.dst_sh = p.ko_sh;
    r.weight = static_cast<const T*>(p.k_w);
    if (p.Hv != 0) do_rows<T, G, KIND, true, true>(p, r, ring, lane, pos, slot, true);
    else do_rows<T, G, KIND, true, false>(p, r, ring, lane, pos, -1, true);
  } else if (pos >= 0) {
    do_rows<T, G, kRaw, false, true>(p, r, ring, lane, 0, slot, false);
  }
}

template <typename T, int G>
cudaError_t launch_rows(const HeadRowsParams& p, int kind, unsigned grid, int warps, cudaStream_t st) {
  const dim3 block(32 * warps);
  const size_t smem = warps * kStages * kStageBytes;
  switch (kind) {
    case kRaw: return launch_pdl(head_rows_kernel<T, G, kRaw>, dim3(grid), block, smem, st, p);
    case kNorm: return launch_pdl(head_rows_kernel<T, G, kNorm>, dim3(grid), block, smem, st, p);
    case kNeox: return launch_pdl(head_rows_kernel<T, G, kNeox>, dim3(grid), block, smem, st, p);
    default: return launch_pdl(head_rows_kernel<T, G, kPairs>, dim3(grid), block, smem, st, p);
  }
}

template <typename T, int G>
int go_rows(HeadRowsParams p, int kind, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return B200_ERR_CUDA;
  constexpr int RPW = 32 / G;
  // Keys and values alone whose heads fill no more than one step of a warp: counted through all tokens, where warps for each token
  // would be more than sixteen for every SM.  16384 tokens of one head of 128 5.0 us, with warps for each token 18.1; 1500 2.1
  // against 5.4; 33 of 8 heads 1.8 against 1.7; 16384 of 8 heads, two steps a token, 20.9 against 20.4.
  if (kind == kRaw && p.Hkv <= RPW && 2 * p.T > 16LL * sms && p.T <= 0x7fffffffLL / p.Hkv) {
    const int64_t rows = p.T * p.Hkv, most = 2 * rows / (RPW * 16LL * sms);    // steps that leave sixteen warps for every SM
    const int steps = static_cast<int>(most < 1 ? 1 : most < 8 ? most : 8);
    const int64_t warps = (rows + RPW * steps - 1) / (RPW * steps);
    constexpr int kWarps = kMaxThreads / 32;
    p.heads_magic = static_cast<uint32_t>((1ULL << 32) / p.Hkv + 1);
    B200_CUDA_TRY(launch_pdl(store_rows_kernel<T, G>, dim3(static_cast<unsigned>((2 * warps + kWarps - 1) / kWarps)), dim3(kMaxThreads),
                             kWarps * kStages * kStageBytes, st, p, static_cast<uint32_t>(rows), static_cast<uint32_t>(warps), steps));
    return B200_OK;
  }
  auto chunks = [&](int heads, int u) { return (heads + RPW * u - 1) / (RPW * u); };
  // Two rows a lane group at a time, and for queries four rounds of that, where every SM still gets sixteen warps; otherwise one
  // row each, for latency.
  const bool wide = p.T * (chunks(p.Hq, 8) + chunks(p.Hkv, 2)) >= 16LL * sms;
  p.heads_q = RPW * (wide ? 8 : 1), p.heads_kv = RPW * (wide ? 2 : 1);
  p.chunks_q = chunks(p.Hq, wide ? 8 : 1), p.chunks_kv = chunks(p.Hkv, wide ? 2 : 1);
  p.chunks = p.chunks_q + p.chunks_kv + (p.Hv ? p.chunks_kv : 0);
  p.chunks_magic = static_cast<uint32_t>((1ULL << 32) / p.chunks + 1);
  // Blocks of one warp where a warp has four rows a lane group or more on average: warps of a block end at different times (8192
  // tokens of 32 + 4 heads 26.9 us, with two warps 31.1).  With less to do the rate at which blocks start would set the pace (keys
  // and values of 16384 tokens, 16 heads of 64: 34.5 us, with two warps 20.4).
  const int rows = chunks(p.Hq, 1) + chunks(p.Hkv, 1) * (p.Hv ? 2 : 1), warps = rows >= 4 * p.chunks ? 1 : kMaxThreads / 32;
  const int64_t blocks = (p.T * p.chunks + warps - 1) / warps;
  if (blocks * warps > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  B200_CUDA_TRY((launch_rows<T, G>(p, kind, static_cast<unsigned>(blocks), warps, st)));
  return B200_OK;
}

template <typename T>
int dispatch_rows(const HeadRowsParams& p, int kind, cudaStream_t st) {
  if (p.D <= 32) return go_rows<T, 2>(p, kind, st);
  if (p.D <= 64) return go_rows<T, 4>(p, kind, st);
  if (p.D <= 128) return go_rows<T, 8>(p, kind, st);
  return go_rows<T, 16>(p, kind, st);
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
  bool wide;                 // rows of the outputs begin at multiples of 32 bytes
};

constexpr int kLoadThreads = 256, kLoadUnroll = 2;

// out[i] = code * scale for the tokens of all sequences, packed: row i belongs to the sequence b with
// indptr[b] <= i < indptr[b + 1] and holds its token starts[b] + i - indptr[b].  A block takes TOKENS rows of keys or of
// values (blockIdx.y).  Its first warp finds the rows' places: the sequence of the first by a 32-way search of indptr, those
// of the others by walking on from there.  Then each thread turns 16 codes (one 16-byte load) into 32 bytes at a time, two
// of them in flight.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kLoadThreads) kv_load_kernel(const __grid_constant__ KvLoadParams p) {
  pdl_start();
  __shared__ int s_page[TOKENS], s_at[TOKENS];      // page -1: behind the last sequence; -2: no such page
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
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
    if (lane < TOKENS) {
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
  const int per_head = p.D / 16, vecs = p.Hkv * per_head, total = vecs * TOKENS;
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
      if (p.wide) {
        st_global_32(dst[u], o);
      } else {
        reinterpret_cast<uint4*>(dst[u])[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(dst[u])[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
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
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.page_size == 1u << i) p.page_shift = i;
  // only a store alone takes its rows as they are: k_out without a rotation or a weight is a copy, which kNorm makes
  const int kind = cos_sin ? (is_neox ? kNeox : kPairs) : Hq == 0 && !k_weight && !k_out && !positions ? kRaw : kNorm;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B200_DT_BF16 ? dispatch_rows<__nv_bfloat16>(p, kind, st) : dispatch_rows<__half>(p, kind, st);
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
  if ((!page_table && page_table_cols > 0) || !indptr || !k_out || !v_out) return B200_ERR_NULL_PTR;
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
  p.wide = ((p.ko_st | p.ko_sh | p.vo_st | p.vo_sh) % 16 == 0) && ((reinterpret_cast<uintptr_t>(ko) | reinterpret_cast<uintptr_t>(vo)) & 31u) == 0;
  const int sms = sm_count();
  if (sms <= 0) return B200_ERR_CUDA;
  // Rows of a block: 32 from 18944 tokens on (148 SMs; eight blocks for every SM, of which six are resident), else 8; with rows of
  // fewer than 64 vectors, of which eight leave threads idle, from so many fewer tokens on.  8 / 32 rows (us, heads of 128): 8 heads
  // 401 tokens 3.2 / 5.9, 12000 17.0 / 17.4, 16000 21.6 / 22.2, 18000 24.0 / 23.8, 24000 30.8 / 29.1, 80000 93 / 83; 4 heads 8000
  // 8.6 / 9.2, 10000 10.5 / 9.8, 20000 18.8 / 14.5; 2 heads 3000 3.2 / 3.6, 5000 4.7 / 4.1, 20000 13.5 / 8.6; one head 2000
  // 3.0 / 2.7, 20000 11.1 / 6.0; 16 heads 16000 37 / 42, 24000 53 / 54.
  const int64_t vecs = static_cast<int64_t>(num_kv_heads) * (head_dim / 16);
  const int rows = tokens >= 2LL * sms * (vecs < 64 ? vecs : 64) ? 32 : 8;
  const int64_t blocks = (tokens + rows - 1) / rows;
  if (blocks > 0x7fffffffLL) return B200_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_pdl(kern, grid, dim3(kLoadThreads), 0, st, p); };
  if (dtype == B200_DT_BF16)
    B200_CUDA_TRY(rows == 32 ? go(kv_load_kernel<__nv_bfloat16, 32>) : go(kv_load_kernel<__nv_bfloat16, 8>));
  else
    B200_CUDA_TRY(rows == 32 ? go(kv_load_kernel<__half, 32>) : go(kv_load_kernel<__half, 8>));
  return B200_OK;
}
