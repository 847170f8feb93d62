// Paged decode attention over the 4-bit cache (kv_q4.cuh): attentionMultiHead
// (src/paged_attention.zig:108-216) for one query row per lane, as
// glacier_cuda_paged_attention_f32, with K and V read as 4-bit codes.
//
// out[b,h] = sum_p softmax_p(q.K_p / sqrt(hd)) V_p.  Per position and kv head the cache
// holds 18 hd / 16 bytes (144 at hd 128, against 1024 in the float32 pages), and the
// G <= 8 query heads of a group need 4 G hd products on them: on the fp32 pipe that
// is more time than the bytes take, so both products run as mma.sync m16n8k16
// (fp16 in, fp32 sums).  M is the query heads, and eight of them would leave half of the
// sixteen rows idle: rows 0-7 hold the high and rows 8-15 the low fp16 part of the same
// float32 numbers, so q and the weights enter with 22 bits at no extra instruction.  (A
// tcgen05.mma needs 64 or 128 rows and its operands in shared memory as fp16: the codes
// would be unpacked, written and read once more, which is what bounds this kernel.)
//   * K: a code c is used as the fp16 number whose bits are the code: c * 2^-24, or c * 2^-20
//     one nibble higher (q's dims there carry 2^-4).  One shift and four ANDs make four
//     operand registers of eight codes.  The zero point is the accumulator's initial value, -7 sum q
//     of the group, and the group's scale multiplies the fp32 result.
//   * V: the scale belongs to the summed index, so it has to be in the operand: s (c - 7) / 8 =
//     (72 - h) s / 8 for the fp16 number h = 64 + (15 - c), whose bits one LOP3 makes.
//     9 s and the result are fp16 numbers (scales have 7 significant bits), so the half FMA is exact.
// The cache's orders put every operand register's codes in one word of one thread: K's words
// (t, g) and V's 16-bit units by position pair are the fragments of these instructions.
#include "kv_q4.cuh"

namespace glacier {

__device__ int g_attn_q4_error;

namespace {

constexpr int kMaxLanes = 1024;
constexpr int kStagePages = 2;  // pages per pipeline stage of a warp
constexpr int kStagePos = kStagePages * kQ4Page;
constexpr int kWarps = 12;
template <int HD>
constexpr int kStages = HD == 128 ? 3 : 6;  // 166 KB of K/V in flight per SM

struct AttnQ4Params {
  const float* q;
  size_t ldq;
  const uint8_t* pool;
  const int32_t* tables;
  const int32_t* ctx_lens;
  float* out;
  size_t ldo;
  int32_t* meta;   // [grid][2]: the pair that is cut at the end of CTA c's share (or -1), its segments
  float* part_ml;  // [2 grid][G][2] maximum (base 2) and sum of a segment
  float* part_o;   // [2 grid][G][hd]
  size_t page_bytes;
  int lanes, max_pages, num_pages, layer, num_heads, num_kv_heads;
  float scale_log2;
  int* bad;
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// (hi, lo) fp16 pairs of two float32 numbers: x = hi + lo to 22 bits.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2_bits(h);
  lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// fp16 bits of 64 + (15 - c) for the nibbles c at bits 4-7 of both halves of x.
__device__ __forceinline__ uint32_t v_bits(uint32_t x) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xAE;" : "=r"(d) : "r"(x), "r"(0x00F000F0u), "r"(0x54005400u));  // (~x & m) | base
  return d;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> lds(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x; r.w[1] = v.y;
  }
  return r;
}

// The queries of one kv head as mma A fragments, and what undoes their scaling.
template <int HD>
struct QFrag {
  static constexpr int NG = HD / 32;
  uint32_t a[2 * NG][4];  // k-steps (group g, half): rows 0-7 high, 8-15 low parts
  float c[NG][4];         // accumulators' initial values: -7 sum q of the group
  float f;                // raw score -> base-2 score
};

template <int HD>
__device__ __forceinline__ void load_q(const AttnQ4Params& p, int lid, int kvh, int G, int lane, QFrag<HD>& q) {
  constexpr int NG = HD / 32;
  const int h = lane >> 2, t = lane & 3;
  float v[NG][8];
  float top = 0.f;
  if (h < G) {
    const float* src = p.q + (size_t)lid * p.ldq + (size_t)(kvh * G + h) * HD + 8 * t;
#pragma unroll
    for (int g = 0; g < NG; ++g) load8(src + 32 * g, v[g]);
  } else {
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] = 0.f;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[g][i]));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // A power of two that brings the head's largest |q| into [2^14, 2^15), from the exponent bits.
  const int e = top > 0.f && top <= 3.4028235e38f ? min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100), 100) : 0;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  q.f = __uint_as_float((uint32_t)(127 + e) << 23) * 0x1p24f * p.scale_log2;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float sh = 0.f, sl = 0.f;
    // The word's nibbles pair dims (i, i + 4); pairs 1 and 3 are used 2^4 higher.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = (i & 1) ? inv * 0.0625f : inv;
      uint32_t hi, lo;
      split2(v[g][i] * m, v[g][i + 4] * m, hi, lo);
      q.a[2 * g + (i >> 1)][(i & 1) * 2] = hi;
      q.a[2 * g + (i >> 1)][(i & 1) * 2 + 1] = lo;
      const float w = (i & 1) ? 16.f : 1.f;
      const float2 fh = __half22float2(bits_h2(hi)), fl = __half22float2(bits_h2(lo));
      sh += w * (fh.x + fh.y);
      sl += w * (fl.x + fl.y);
    }
    sh += __shfl_xor_sync(0xffffffffu, sh, 1);
    sl += __shfl_xor_sync(0xffffffffu, sl, 1);
    sh += __shfl_xor_sync(0xffffffffu, sh, 2);
    sl += __shfl_xor_sync(0xffffffffu, sl, 2);
    q.c[g][0] = q.c[g][1] = -7.f * 0x1p-24f * sh;
    q.c[g][2] = q.c[g][3] = -7.f * 0x1p-24f * sl;
  }
}

// One stage (two pages) of one warp: scores, online softmax, and the weighted V.  m is the
// running maximum (base 2) of head lane / 4, l this thread's share of its sum; weights carry
// 2^15 so that their low parts stay normal fp16 numbers, o carries 2^15 / 8.
// nvalid: positions of the stage inside the context; pages: bit i set when page i was loaded.
template <int HD, bool MASK>
__device__ __forceinline__ void stage_math(const uint8_t* __restrict__ buf, const QFrag<HD>& q, float& m, float& l,
                                           float (&o)[HD / 8][4], int nvalid, uint32_t pages, int lane) {
  constexpr int NG = HD / 32, NW = HD / 32;  // scale groups; words per thread and position (K) or pair (V)
  constexpr int BLK = 18 * HD;
  const int n = lane >> 2, t = lane & 3;
  float2 sc[kStagePages * 2];
#pragma unroll
  for (int pg = 0; pg < kStagePages; ++pg) {
    const uint8_t* K = buf + pg * BLK;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Words<NW> w = lds<NW>(K + (8 * j + n) * (HD / 2) + t * (4 * NG));
      const Words<NG> s = lds<NG>(K + 16 * HD + (4 * j + t) * (4 * NG));
      float2 r = make_float2(0.f, 0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float d[4];
        const uint32_t x = w.w[g], y = x >> 8;
        mma_f16(d, q.a[2 * g], x & 0x000F000Fu, x & 0x00F000F0u, q.c[g]);
        mma_f16(d, q.a[2 * g + 1], y & 0x000F000Fu, y & 0x00F000F0u, d);
        const float2 f = __half22float2(bits_h2(s.w[g]));
        r = __ffma2_rn(f, make_float2(d[0], d[1]), r);
        r = __ffma2_rn(f, make_float2(d[2], d[3]), r);
      }
      r.x *= q.f;
      r.y *= q.f;
      if constexpr (MASK) {
        const int at = pg * kQ4Page + 8 * j + 2 * t;
        const bool here = (pages >> pg) & 1;
        if (!here || at >= nvalid) r.x = -INFINITY;
        if (!here || at + 1 >= nvalid) r.y = -INFINITY;
      }
      sc[2 * pg + j] = r;
    }
  }
  float mx = fmaxf(sc[0].x, sc[0].y);
#pragma unroll
  for (int i = 1; i < 2 * kStagePages; ++i) mx = fmaxf(mx, fmaxf(sc[i].x, sc[i].y));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  if (__any_sync(0xffffffffu, mx > m)) {
    const float mn = fmaxf(m, mx);
    const float a = m == -INFINITY ? 0.f : ex2(m - mn);
    m = mn;
    l *= a;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] *= a;
  }
  const float base = m == -INFINITY ? 15.f : 15.f - m;
#pragma unroll
  for (int pg = 0; pg < kStagePages; ++pg) {
    uint32_t a[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float x = ex2(sc[2 * pg + j].x + base), y = ex2(sc[2 * pg + j].y + base);
      l += x + y;
      split2(x, y, a[2 * j], a[2 * j + 1]);
    }
    const uint8_t* V = buf + pg * BLK + 8 * HD;
    const uint8_t* S = buf + pg * BLK + 17 * HD + (n / (8 / NG)) * 4;
    __half2 s9[2], s8[2];
    Words<NW> w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[j] = lds<NW>(V + (t + 4 * j) * HD + n * (4 * NW));
      uint32_t sb = *reinterpret_cast<const uint32_t*>(S + (t + 4 * j) * (4 * NG));
      if constexpr (MASK) {  // left-over scales may be anything, and 0 * NaN is NaN
        const int at = pg * kQ4Page + 8 * j + 2 * t;
        const bool here = (pages >> pg) & 1;
        if (!here || at >= nvalid) sb = 0;
        else if (at + 1 >= nvalid) sb &= 0xffffu;
      }
      s9[j] = __hmul2(bits_h2(sb), __float2half2_rn(9.f));
      s8[j] = __hmul2(bits_h2(sb), __float2half2_rn(-0.125f));
    }
#pragma unroll
    for (int k = 0; k < NW; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t x = w[j].w[k];
          const uint32_t y = i == 0 ? x << 4 : i == 1 ? x : i == 2 ? x >> 4 : x >> 8;
          b[j] = h2_bits(__hfma2(bits_h2(v_bits(y)), s8[j], s9[j]));
        }
        mma_f16(o[4 * k + i], a, b[0], b[1], o[4 * k + i]);
      }
    }
  }
}

// The stages (32 positions of one kv head) of all (lane, kv head) pairs laid end to end,
// lane-major; CTA c takes [c Q, (c + 1) Q), so every SM reads the same number of bytes.
// Run by one warp: C[b] = first stage of lane b, ctx[b] its clamped context; returns Q.
__device__ __forceinline__ void stage_plan(const AttnQ4Params& p, long long* C, int* ctx, long long* plan) {
  const int lane = threadIdx.x & 31;
  const long long cap = (long long)p.max_pages * kQ4Page;
  long long total = 0;
  for (int b0 = 0; b0 < p.lanes; b0 += 32) {
    const int b = b0 + lane;
    const int c = b < p.lanes ? (int)min((long long)max(p.ctx_lens[b], 0), cap) : 0;
    const long long mine = (long long)p.num_kv_heads * ((c + (long long)kStagePos - 1) / kStagePos);
    long long incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += u;
    }
    if (b < p.lanes) {
      C[b] = total + incl - mine;
      ctx[b] = c;
    }
    total += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) {
    C[p.lanes] = total;
    plan[0] = total;
    plan[1] = max((long long)kWarps, (total + gridDim.x - 1) / gridDim.x);  // one stage per warp at least
  }
}

// A walk over the pairs of a CTA's share [g0, g1), and this warp's stages [wb, we) of each:
// the pair's segment [sb, se) is cut evenly over the CTA's warps.
struct PairWalk {
  int lid, kvh, ns, sb, se, wb, we;
  long long P;  // the pair's first stage
  __device__ __forceinline__ void set(const int* ctx, long long g0, long long g1, int warp) {
    ns = (int)((ctx[lid] + (long long)kStagePos - 1) / kStagePos);
    sb = (int)max(0ll, g0 - P);
    se = (int)min((long long)ns, g1 - P);
    const int n = se - sb;
    wb = sb + (int)((long long)n * warp / kWarps);
    we = sb + (int)((long long)n * (warp + 1) / kWarps);
  }
  // False when the share is at its end.
  __device__ __forceinline__ bool next(const int* ctx, int lanes, int hkv, long long g0, long long g1, int warp) {
    P += ns;
    if (++kvh == hkv) {
      kvh = 0;
      do ++lid;
      while (lid < lanes && ctx[lid] == 0);
    }
    if (lid >= lanes || P >= g1) return false;
    set(ctx, g0, g1, warp);
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(kWarps * 32, 1) attn_q4_kernel(const AttnQ4Params p) {
  constexpr int BLK = 18 * HD;
  constexpr int NST = kStages<HD>;
  constexpr int ROW = HD + 4;  // floats per (warp, head) of the merge buffer
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kWarps][NST];
  __shared__ float s_ml[kWarps][8][2];
  __shared__ long long C[kMaxLanes + 1];
  __shared__ long long plan[2];
  __shared__ int ctx[kMaxLanes];
  griddep_launch();
  griddep_wait();  // q, the pages, tables and lengths come from earlier kernels
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = p.num_kv_heads, G = p.num_heads / hkv;
  uint8_t* ring = smem + (size_t)warp * NST * kStagePages * BLK;
  float* merge = reinterpret_cast<float*>(smem + (size_t)kWarps * NST * kStagePages * BLK);  // [warps][G][ROW]
  if (warp == 0) stage_plan(p, C, ctx, plan);
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  const long long total = plan[0], Q = plan[1];
  const long long g0 = min(total, blockIdx.x * Q), g1 = min(total, g0 + Q);
  // Lanes of context 0 get zeros.
  for (int b = blockIdx.x; b < p.lanes; b += gridDim.x)
    if (ctx[b] == 0)
      for (int i = threadIdx.x; i < p.num_heads * HD; i += kWarps * 32) p.out[(size_t)b * p.ldo + i] = 0.f;
  if (threadIdx.x == 0) p.meta[2 * blockIdx.x] = -1;
  if (g0 >= g1) return;

  PairWalk use;
  {
    int lo = 0, hi = p.lanes - 1;  // the lane whose stages hold g0: the last with C <= g0 (never an empty one)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (C[mid] <= g0) lo = mid; else hi = mid - 1;
    }
    use.lid = lo;
    use.ns = (int)((ctx[lo] + (long long)kStagePos - 1) / kStagePos);
    use.kvh = (int)((g0 - C[lo]) / use.ns);
    use.P = C[lo] + (long long)use.kvh * use.ns;
    use.set(ctx, g0, g1, warp);
  }
  PairWalk ld = use;
  bool ld_more = true;
  const uint64_t pol = l2_evict_first_policy();
  // ---- loads: the warp's stages in order, NST of them ahead of the arithmetic ----
  int ld_st = ld.wb, ld_at = 0;  // next stage; its place among the 16 stages whose page ids `ids` holds
  int32_t ids = 0;
  auto fetch_ids = [&]() {  // page ids of 16 stages, one per thread
    const long long j = (long long)kStagePages * ld_st + lane;
    ids = j * kQ4Page < ctx[ld.lid] ? p.tables[(size_t)ld.lid * p.max_pages + j] : -2;  // -2: past the context
    ld_at = 0;
  };
  fetch_ids();
  uint32_t issued = 0, loaded = 0;  // loaded: two bits per ring slot, the pages that are there
  int slot_in = 0;
  auto issue = [&]() {
    while (ld_more && ld_st >= ld.we) {
      ld_more = ld.next(ctx, p.lanes, hkv, g0, g1, warp);
      if (!ld_more) break;
      ld_st = ld.wb;
      if (ld_st < ld.we) fetch_ids();
    }
    if (!ld_more) return;
    if (ld_at == 16) fetch_ids();
    const int page = __shfl_sync(0xffffffffu, ids, kStagePages * ld_at + (lane & 1));
    const bool there = (unsigned)page < (unsigned)p.num_pages;
    const uint32_t got = __ballot_sync(0xffffffffu, there) & 3u;
    if (lane < 2 && !there && page != -2) atomicExch(p.bad, 1);
    uint64_t* bar = &full[warp][slot_in];
    if (lane == 0) mbar_arrive_expect_tx(bar, BLK * __popc(got));
    __syncwarp();
    if (lane < kStagePages && there)
      bulk_load(ring + (slot_in * kStagePages + lane) * BLK,
                p.pool + (size_t)page * p.page_bytes + ((size_t)p.layer * hkv + ld.kvh) * BLK, BLK, bar, pol);
    loaded = (loaded & ~(3u << (2 * slot_in))) | got << (2 * slot_in);
    slot_in = slot_in + 1 == NST ? 0 : slot_in + 1;
    ++issued;
    ++ld_st;
    ++ld_at;
  };
#pragma unroll 1
  for (int i = 0; i < NST; ++i) issue();

  uint32_t consumed = 0, phase = 0;
  int slot = 0;
  bool ok = true;
  while (true) {
    QFrag<HD> q;
    load_q<HD>(p, use.lid, use.kvh, G, lane, q);
    float m = -INFINITY, l = 0.f;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    for (int st = use.wb; st < use.we && ok; ++st) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][slot], phase, p.err));
      if (!ok) break;
      const int nvalid = (int)min((long long)kStagePos, ctx[use.lid] - (long long)kStagePos * st);
      const uint32_t pages = (loaded >> (2 * slot)) & 3u;
      const uint8_t* buf = ring + slot * kStagePages * BLK;
      if (nvalid == kStagePos && pages == 3u)
        stage_math<HD, false>(buf, q, m, l, o, nvalid, pages, lane);
      else
        stage_math<HD, true>(buf, q, m, l, o, nvalid, pages, lane);
      ++consumed;
      if (++slot == NST) {
        slot = 0;
        phase ^= 1;
      }
      __syncwarp();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // reads of this slot before the next copy into it
      issue();
    }
    // ---- merge the warps' states, in warp order ----
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int h = lane >> 2, t = lane & 3;
    if (h < G) {
      if (t == 0) {
        s_ml[warp][h][0] = m;
        s_ml[warp][h][1] = l;
      }
      float* d = merge + ((size_t)warp * G + h) * ROW + (HD / 4) * t;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < HD / 32; ++k)
          *reinterpret_cast<float4*>(d + (HD / 8) * c + 4 * k) =
              make_float4(o[4 * k][c] + o[4 * k][c + 2], o[4 * k + 1][c] + o[4 * k + 1][c + 2],
                          o[4 * k + 2][c] + o[4 * k + 2][c + 2], o[4 * k + 3][c] + o[4 * k + 3][c + 2]);
    }
    __syncthreads();
    const bool whole = use.sb == 0 && use.se == use.ns;
    const size_t part = 2 * (size_t)blockIdx.x + (use.sb == 0 ? 1 : 0);
    for (int e = threadIdx.x; e < G * (HD / 4); e += kWarps * 32) {
      const int g = e / (HD / 4), d4 = e % (HD / 4);
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_ml[w][g][0]);
      float L = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = s_ml[w][g][0];
        const float x = mw == -INFINITY ? 0.f : ex2(mw - M);
        L = fmaf(s_ml[w][g][1], x, L);
        const float4 v = *reinterpret_cast<const float4*>(merge + ((size_t)w * G + g) * ROW + 4 * d4);
        a.x = fmaf(v.x, x, a.x);
        a.y = fmaf(v.y, x, a.y);
        a.z = fmaf(v.z, x, a.z);
        a.w = fmaf(v.w, x, a.w);
      }
      if (whole) {
        const float r = L == 0.f ? 0.f : 8.f / L;
        *reinterpret_cast<float4*>(p.out + (size_t)use.lid * p.ldo + (size_t)(use.kvh * G + g) * HD + 4 * d4) =
            make_float4(a.x * r, a.y * r, a.z * r, a.w * r);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part * G + g) * HD + 4 * d4) = a;
        if (d4 == 0) {
          p.part_ml[(part * G + g) * 2] = M;
          p.part_ml[(part * G + g) * 2 + 1] = L;
        }
      }
    }
    if (threadIdx.x == 0 && use.sb == 0 && use.se < use.ns) {
      p.meta[2 * blockIdx.x] = use.lid * hkv + use.kvh;
      p.meta[2 * blockIdx.x + 1] = (int)((use.P + use.ns - 1) / Q - use.P / Q + 1);
    }
    if (!use.next(ctx, p.lanes, hkv, g0, g1, warp)) break;
    __syncthreads();  // the merge buffer is free again
  }
  // Leave no copy in flight (a wait that gave up leaves some outstanding).
  for (uint32_t i = consumed; i < issued; ++i) {
    mbar_wait(&full[warp][slot], phase, p.err);
    if (++slot == NST) {
      slot = 0;
      phase ^= 1;
    }
  }
}

// Pairs that were cut: block c merges the pair whose first segment ends CTA c's share.  Its
// segments are CTA c's last and the first ones of the CTAs behind it, merged in that order.
// 1024 threads: G hd / 4 columns by as many slices of the segments as fit.
__global__ void __launch_bounds__(1024) attn_q4_combine_kernel(const AttnQ4Params p, int hd) {
  __shared__ float4 s_o[1024];
  __shared__ float s_l[1024];
  griddep_launch();
  griddep_wait();
  const int c = blockIdx.x, pair = p.meta[2 * c];
  if (pair < 0) return;
  const int nseg = p.meta[2 * c + 1], G = p.num_heads / p.num_kv_heads;
  const int cols = G * (hd / 4), slices = 1024 / cols;
  const int col = threadIdx.x % cols, slice = threadIdx.x / cols;
  const int g = col / (hd / 4), d = 4 * (col % (hd / 4));
  auto part = [&](int s) { return (s == 0 ? 2 * (size_t)c + 1 : 2 * (size_t)(c + s)) * G + g; };
  float L = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (slice < slices) {
    float M = -INFINITY;
    for (int s = 0; s < nseg; ++s) M = fmaxf(M, p.part_ml[part(s) * 2]);
    const int per = (nseg + slices - 1) / slices;
#pragma unroll 4
    for (int s = slice * per; s < min(nseg, (slice + 1) * per); ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + part(s) * 2);
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + part(s) * hd + d);
      const float x = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      L = fmaf(ml.y, x, L);
      a.x = fmaf(v.x, x, a.x);
      a.y = fmaf(v.y, x, a.y);
      a.z = fmaf(v.z, x, a.z);
      a.w = fmaf(v.w, x, a.w);
    }
  }
  s_o[threadIdx.x] = a;
  s_l[threadIdx.x] = L;
  __syncthreads();
  if (slice != 0) return;
  for (int s = 1; s < slices; ++s) {
    const float4 v = s_o[s * cols + col];
    L += s_l[s * cols + col];
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  const float r = L == 0.f ? 0.f : 8.f / L;
  *reinterpret_cast<float4*>(p.out + (size_t)(pair / p.num_kv_heads) * p.ldo +
                             (size_t)((pair % p.num_kv_heads) * G + g) * hd + d) =
      make_float4(a.x * r, a.y * r, a.z * r, a.w * r);
}

}  // namespace

int attn_q4_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    int z = 0;
    cudaMemcpyToSymbol(g_attn_q4_error, &z, sizeof(int));
  }
  return v;
}

// Two partial segments per CTA (one that begins a pair, one that continues it), and the
// descriptors of cut pairs.
size_t attention_q4_workspace_floats(size_t num_heads, size_t num_kv_heads, size_t head_dim) {
  if (!num_kv_heads) return 0;
  const size_t ctas = (size_t)sm_count();
  return ceil_div(2 * ctas, (size_t)4) * 4 + 2 * ctas * (num_heads / num_kv_heads) * (head_dim + 2);
}

int paged_attention_q4(const float* q, size_t ldq, const void* pool, size_t num_pages, size_t num_layers,
                       const int32_t* block_tables, size_t max_pages, const int32_t* ctx_lens, size_t lanes,
                       size_t layer, size_t num_heads, size_t num_kv_heads, size_t head_dim, float* out, size_t ldo,
                       float* workspace, size_t workspace_floats, cudaStream_t stream) {
  GLC_REQUIRE(q && block_tables && ctx_lens && out && workspace, "paged_attention_q4: null argument");
  int rc = q4_check_pool("paged_attention_q4", pool, num_pages, num_layers, layer, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  GLC_REQUIRE(lanes > 0 && lanes <= (size_t)kMaxLanes, "paged_attention_q4: %zu lanes (1 to %d)", lanes, kMaxLanes);
  GLC_REQUIRE(max_pages > 0 && max_pages <= ((size_t)1 << 26), "paged_attention_q4: %zu pages per lane", max_pages);
  GLC_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0 && ldq % 4 == 0 &&
                  ldo % 4 == 0,
              "paged_attention_q4: q, out and workspace must be 16-byte aligned");
  const size_t need = attention_q4_workspace_floats(num_heads, num_kv_heads, head_dim);
  GLC_REQUIRE(workspace_floats >= need, "paged_attention_q4: workspace of %zu floats needed", need);
  const int grid = sm_count();
  const size_t G = num_heads / num_kv_heads;
  AttnQ4Params p;
  p.q = q;
  p.ldq = ldq;
  p.pool = static_cast<const uint8_t*>(pool);
  p.tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.out = out;
  p.ldo = ldo;
  p.meta = reinterpret_cast<int32_t*>(workspace);
  p.part_o = workspace + ceil_div(2 * (size_t)grid, (size_t)4) * 4;
  p.part_ml = p.part_o + 2 * (size_t)grid * G * head_dim;
  p.page_bytes = num_layers * num_kv_heads * q4_block_bytes(head_dim);
  p.lanes = (int)lanes;
  p.max_pages = (int)max_pages;
  p.num_pages = (int)num_pages;
  p.layer = (int)layer;
  p.num_heads = (int)num_heads;
  p.num_kv_heads = (int)num_kv_heads;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  p.bad = ops_error_word();
  p.err = device_symbol_address(g_attn_q4_error);
  GLC_REQUIRE(p.bad && p.err, "paged_attention_q4: device status word unavailable");
  auto kern = head_dim == 128 ? attn_q4_kernel<128> : attn_q4_kernel<64>;
  const size_t stages = head_dim == 128 ? kStages<128> : kStages<64>;
  const size_t smem = kWarps * (stages * kStagePages * q4_block_bytes(head_dim) + G * (head_dim + 4) * sizeof(float));
  if ((rc = allow_dynamic_smem((const void*)kern, (int)smem))) return rc;
  if ((rc = launch_pdl(kern, dim3((unsigned)grid), dim3(kWarps * 32), smem, stream, 1, p))) return rc;
  return launch_pdl(attn_q4_combine_kernel, dim3((unsigned)grid), dim3(1024), 0, stream, 1, p, (int)head_dim);
}

}  // namespace glacier
