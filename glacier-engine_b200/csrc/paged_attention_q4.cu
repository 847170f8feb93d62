// Paged decode attention over the 4-bit cache (kv_q4.cuh): attentionMultiHead
// (src/paged_attention.zig:108-216) for one query row per lane, as
// glacier_cuda_paged_attention_f32, with K and V read as 4-bit codes.
//
// out[b,h] = sum_p softmax_p(q.K_p / sqrt(hd)) V_p.  Per position and kv head the cache
// holds 18 hd / 16 bytes (144 at hd 128, against 1024 in the float32 pages), and the
// G <= 8 query heads of a group need 4 G hd products on them: on the fp32 pipe that
// is more time than the bytes take, so both products run as mma.sync m16n8k16
// (fp16 in, fp32 sums).  q and the softmax weights go in as a high and a low fp16 part, 22
// bits together; the held values are exact.  (tcgen05.mma would take the unpacked codes as its A operand
// in tensor memory, 128 positions or dims a tile, with q or the weights as sixteen columns in shared
// memory.  Every operand register would go there by tcgen05.st first, and the accumulators would leave the
// register file; this form has not been built or measured.)
//   * q K^T: M is the query heads, and eight of them would leave half of the sixteen rows
//     idle: rows 0-7 hold q's high and rows 8-15 its low parts.  A code c at bits 4-7 is used as
//     the subnormal fp16 number that these bits are, c * 2^-20: three shifts and four ANDs make
//     four operand registers of eight codes.  (At bits 0-3, c * 2^-24, one shift would do, but the
//     tensor core aligns a subnormal's products as if it had the smallest normal exponent, and
//     its sums were 2^-20 off; at bits 4-7 they are within 2^-25.)  The zero point is the
//     accumulator's initial value, -7 sum q of the group, and the group's scale multiplies the
//     fp32 result.
//   * (P V)^T = V^T P^T: M is sixteen dims, N the heads, so that no accumulator is idle, and the
//     score accumulators are the weights' operand as they stand.  The scale belongs to the summed
//     index, so it has to be in the operand: (c - 7) s / 8 = (72 - h) s / 8 for the fp16 number
//     h = 64 + (15 - c), whose bits one LOP3 makes from a code at bits 4-7.  9 s and the result
//     are fp16 numbers (scales have 7 significant bits), so one half FMA is exact.
//     With four heads at most (PACK) the weights' high and low parts share the eight columns: score
//     rows 4-7 repeat heads 0-3, columns 4-7 take the low parts, and one instruction does both.
// The cache's orders put every operand register's codes in one word of one thread: K's words
// (t, g) and V's 16-bit units by position pair are the fragments of these instructions.
//
// What bounds it (B200, 7B heads, graph replay): 64 lanes of 2048 positions take 30.1 us, their 77 MB
// at the measured copy rate 12.0; from there on 8.5 us for every 1000 positions more, against 5.7. The
// slope is arithmetic and its dependences (with all pages in L2 it is the same, and the loads alone run
// at the copy rate): some 600 instructions per warp and 32 positions, 64 of them mma.sync of 8 cycles, with
// two warps per SM partition take 1250 cycles, twice what their issue does. The rest, some 10 us (7 when no
// pair is cut between CTAs), is fixed: launch, three dependent loads to the first stage, the merges. Of
// that much is fetching code that runs once, so the stage and the loads stand in the kernel once (two
// copies of each: 1 to 3 % slower). Few short contexts are all fixed costs (one lane of 40: 4.7 us, of
// 1000: 6.1). The FP32 cache's kernel takes 98 us on the layer whose 64 lanes (256 to 4096 positions) take
// 30 here.
#include <algorithm>
#include <atomic>
#include <chrono>

#include "kv_q4.cuh"

namespace glacier {

namespace {

constexpr int kMaxLanes = 1024;
// Warps per CTA (one CTA per SM).  Three warps per SM partition cover each other's latencies better than
// two, but at hd 128 they have to spill at 168 registers: with stages of 32 positions the 64-lane 7B
// layer takes 32.3 us with eight warps and 33.3 with twelve (one lane of 1000 positions 6.1 and 7.4), 128
// lanes of 1 to 1999 positions at hd 64 31.4 and 29.8.
template <int HD>
constexpr int kWarps = HD == 128 ? 8 : 12;
// Pages per stage: 64 positions, which spread the softmax's chain and the loop over twice the products
// of 32 (the 64-lane 7B layer 30.1 and 32.2 us; 64 lanes of 512 13.7 and 13.0).  The cluster form at hd 128
// takes 32: one lane of 1000 positions 6.1 us, with 64 6.7; of 2000 7.6 and 7.1, of 6000 10.3 and 11.9.
template <int HD, bool CLUSTER>
constexpr int kStagePages = HD == 128 && CLUSTER ? 2 : 4;
// Stages in a warp's ring: 147 and 166 KB of K/V per SM.
template <int HD, bool CLUSTER>
constexpr int kStages = HD == 64 ? 3 : CLUSTER ? 4 : 2;
constexpr int kClusterCtas = 4;
constexpr int kPart = 4;  // heads that a warp merges at once, at most
struct AttnQ4Params {
  const float* q;
  size_t ldq;
  const uint8_t* pool;
  const int32_t* tables;
  const int32_t* ctx_lens;
  float* out;
  size_t ldo;
  unsigned long long* tickets;  // [grid][8]: segments written of the pair that CTA c began and left open, per head
  unsigned long long nonce;     // marks this launch's tickets: whatever else a ticket holds counts as none
  float* part_ml;  // [2 grid][G][2] maximum (base 2) and sum of a segment
  float* part_o;   // [2 grid][G][hd]
  uint32_t page_bytes;
  int lanes, max_pages, num_pages, layer, num_heads, num_kv_heads;
  int clusters;  // cluster form: clusters per pair
  float scale_log2;
  int* bad;
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
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  const float2 r = __ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x);
  hi = h2_bits(h);
  lo = h2_bits(__floats2half2_rn(r.x, r.y));
}

// fp16 bits of 64 + (15 - c) for the nibbles c at bits 4-7 of both halves of x.
__device__ __forceinline__ uint32_t v_bits(uint32_t x) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xAE;" : "=r"(d) : "r"(x), "r"(0x00F000F0u), "r"(0x54005400u));  // (~x & m) | base
  return d;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// This thread's dims of head lane / 4 (PACK: lane / 4 % 4): v[2g][..], v[2g + 1][..] are dims 8 t .. 8 t + 7
// of group g (zeros past the last head).
template <int HD, bool PACK>
__device__ __forceinline__ void load_q(const AttnQ4Params& p, int lid, int kvh, int G, int lane,
                                       float (&v)[HD / 16][4]) {
  const int h = PACK ? lane >> 2 & 3 : lane >> 2, t = lane & 3;
#pragma unroll
  for (int g = 0; g < HD / 32; ++g) {
    float x[8];
    if (h < G) {
      load8(p.q + (size_t)lid * p.ldq + (size_t)(kvh * G + h) * HD + 8 * t + 32 * g, x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[2 * g + i / 4][i % 4] = x[i];
  }
}

template <int HD>
__device__ __forceinline__ void split_q(const AttnQ4Params& p, const float (&v)[HD / 16][4], QFrag<HD>& q) {
  constexpr int NG = HD / 32;
  float top = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[2 * g + i / 4][i % 4]));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // A power of two that brings the head's largest |q| into [2^14, 2^15), from the exponent bits: up to
  // 2^125, where q.f is still a float32 number.
  const int top_e = (int)(__float_as_uint(top) >> 23) - 127 - 14;
  const int e = top > 0.f && top <= 3.4028235e38f ? min(max(top_e, -100), 110) : 0;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  q.f = __uint_as_float((uint32_t)(127 + e) << 23) * (0x1p20f * p.scale_log2);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    // High and low parts keep sums of their own: the high row then adds numbers of few bits, which the
    // tensor core's sums hold whole.
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the word's nibbles pair dims (i, i + 4)
      uint32_t hi, lo;
      split2(make_float2(v[2 * g][i] * inv, v[2 * g + 1][i] * inv), hi, lo);
      q.a[2 * g + (i >> 1)][(i & 1) * 2] = hi;
      q.a[2 * g + (i >> 1)][(i & 1) * 2 + 1] = lo;
      const float2 h = __half22float2(bits_h2(hi)), l = __half22float2(bits_h2(lo));
      sum = __fadd2_rn(sum, make_float2(h.x + h.y, l.x + l.y));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
      sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
    }
    q.c[g][0] = q.c[g][1] = -7.f * 0x1p-20f * sum.x;
    q.c[g][2] = q.c[g][3] = -7.f * 0x1p-20f * sum.y;
  }
}

// Raw scores of one stage: sc[2 page + half] = the scores of head lane / 4 with the positions
// 8 half + 2 (lane % 4) + {0, 1} of the page.
template <int HD, int SP>
__device__ __forceinline__ void stage_scores(const uint8_t* __restrict__ buf, const QFrag<HD>& q,
                                             float2 (&sc)[2 * SP], int lane) {
  constexpr int NG = HD / 32;  // scale groups = words per thread and position
  constexpr int BLK = 18 * HD;
  const int n = lane >> 2, t = lane & 3;
#pragma unroll
  for (int pg = 0; pg < SP; ++pg) {
    const uint8_t* K = buf + pg * BLK;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Words<NG> w = lds<NG>(K + (8 * j + n) * (HD / 2) + t * (4 * NG));
      const Words<NG> s = lds<NG>(K + 16 * HD + (4 * j + t) * (4 * NG));
      float2 r = make_float2(0.f, 0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float d[4];
        const uint32_t x = w.w[g], y = x >> 8;
        mma_f16(d, q.a[2 * g], x * 16u & 0x00F000F0u, x & 0x00F000F0u, q.c[g]);
        mma_f16(d, q.a[2 * g + 1], y * 16u & 0x00F000F0u, y & 0x00F000F0u, d);
        const float2 f = __half22float2(bits_h2(s.w[g]));
        r = __ffma2_rn(f, make_float2(d[0], d[1]), r);
        r = __ffma2_rn(f, make_float2(d[2], d[3]), r);
      }
      sc[2 * pg + j] = r;
    }
  }
}

// The online softmax of one stage's scores and its weighted V.  Weights are 2^13 2^(s - m) in
// base-2 scores s: m is a reference near the running maximum of head lane / 4, moved
// (and everything rescaled) only when a score passes it by more than 2^2, so the weights stay
// below 2^15.  Their two fp16 parts hold them to 22 bits above 2^-3, and to 2^-25 below: n positions
// lose up to n 2^-38 of max |v| (with 2^7 and 2^8 in these places it was n 2^-32, 2.8e-7 where 64 lanes of
// 4000 positions have one 22 nats above the others; the time is the same).  l: this thread's share of their
// sum; o: sums of weight * v / 8.
// keep: masks of the V scales, one per eight positions (two positions a word).
template <int HD, int SP, bool PACK>
__device__ __forceinline__ void stage_values(const uint8_t* __restrict__ buf, const QFrag<HD>& q,
                                             float2 (&sc)[2 * SP], const uint32_t (&keep)[2 * SP],
                                             float& m, float2& l, float (&o)[HD / 16][4], int lane) {
  constexpr int NG = HD / 32, NW = HD / 32;  // scale groups; words per thread and position pair
  constexpr int BLK = 18 * HD;
  const int n = lane >> 2, t = lane & 3;
  float mx = fmaxf(sc[0].x, sc[0].y);
#pragma unroll
  for (int i = 1; i < 2 * SP; ++i) mx = fmaxf(mx, fmaxf(sc[i].x, sc[i].y));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const bool move = (mx - m) * q.f > 2.f;  // false for NaN: no score yet
  if (__any_sync(0xffffffffu, move)) {
    const float mn = move ? mx : m;
    const float a = m == -INFINITY ? 0.f : ex2((m - mn) * q.f);
    m = mn;
    l.x *= a;
    l.y *= a;
    const float a0 = __shfl_sync(0xffffffffu, a, 8 * t), a1 = __shfl_sync(0xffffffffu, a, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      o[i][0] *= a0;
      o[i][1] *= a1;
      o[i][2] *= a0;
      o[i][3] *= a1;
    }
  }
  // The state's maximum is the rounded m q.f, so the weights refer to it and its error cancels.  Beyond
  // base-2 scores of 2^18 that error could move a weight out of fp16's range, and is taken back.  (Weights
  // from q.f (s - m) need no such step, but each has the difference's rounding then: errors up to a quarter larger,
  // and the same time.)
  const float m0 = m == -INFINITY ? 0.f : m, top = m0 * q.f, err = fmaf(m0, q.f, -top);
  const float back = fabsf(err) > 0x1p-6f ? -err : 0.f;
  // The stage's sums start from zero and are added with rounding: a tensor core's sums cut, always
  // towards zero, and over ten stages that was 1e-6 of the result (with this, 3e-7; 1.5 % of the time).
  uint32_t hi[2 * SP], lo[2 * SP];
  __half2 s9[2 * SP], s8[2 * SP];
  Words<NW> w[2 * SP];
#pragma unroll
  for (int pj = 0; pj < 2 * SP; ++pj) {
    float2 e = __ffma2_rn(sc[pj], make_float2(q.f, q.f), make_float2(-top, -top));
    e = __fadd2_rn(e, make_float2(back, back));
    e.x = ex2(e.x);
    e.y = ex2(e.y);
    e = __fmul2_rn(e, make_float2(8192.f, 8192.f));
    l = __fadd2_rn(l, e);
    split2(e, hi[pj], lo[pj]);
    if (PACK && n >= 4) hi[pj] = lo[pj];
    const uint8_t* V = buf + pj / 2 * BLK + 8 * HD;
    const uint8_t* S = buf + pj / 2 * BLK + 17 * HD + (n / (8 / NG)) * 4;
    w[pj] = lds<NW>(V + (t + 4 * (pj & 1)) * HD + n * (4 * NW));
    // Left-over scales may be anything, and 0 * NaN is NaN.
    const uint32_t sb = *reinterpret_cast<const uint32_t*>(S + (t + 4 * (pj & 1)) * (4 * NG)) & keep[pj];
    s9[pj] = __hmul2(bits_h2(sb), __float2half2_rn(9.f));
    s8[pj] = __hmul2(bits_h2(sb), __float2half2_rn(-0.125f));
  }
  constexpr int KC = 2;  // words at a time: four tiles, whose instructions do not wait for one another
#pragma unroll
  for (int k0 = 0; k0 < NW; k0 += KC) {
    float sum[2 * KC][4];
#pragma unroll
    for (int i = 0; i < 2 * KC; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[i][c] = 0.f;
#pragma unroll
    for (int pg = 0; pg < SP; ++pg) {
      // A tile's rows g and g + 8 are dims 4k + i and 4k + i + 1 of this thread's sixteen (eight at hd 64).
#pragma unroll
      for (int k = 0; k < KC; ++k) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          uint32_t a[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int pj = 2 * pg + j;
            const uint32_t x = w[pj].w[k0 + k];
            a[2 * j] = h2_bits(__hfma2(bits_h2(v_bits(i == 0 ? x * 16u : x >> 4)), s8[pj], s9[pj]));
            a[2 * j + 1] = h2_bits(__hfma2(bits_h2(v_bits(i == 0 ? x : x >> 8)), s8[pj], s9[pj]));
          }
          float(&d)[4] = sum[2 * k + i / 2];
          mma_f16(d, a, hi[2 * pg], hi[2 * pg + 1], d);
          if constexpr (!PACK) mma_f16(d, a, lo[2 * pg], lo[2 * pg + 1], d);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * KC; ++i)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        float(&d)[4] = o[2 * k0 + i];
        const float2 r = __fadd2_rn(make_float2(d[c], d[c + 1]), make_float2(sum[i][c], sum[i][c + 1]));
        d[c] = r.x;
        d[c + 1] = r.y;
      }
  }
}

// A walk over the pairs of a warp's share [g0, g1) and its segment [sb, se) of each.  All (lane,
// kv head) pairs are laid end to end, lane-major, each with a unit for every stage and one in front
// for the change of pair (it takes about a stage's time), and warp w of the grid takes units
// [w Q, (w + 1) Q): every warp does the same work.
template <int SP>
struct PairWalk {
  int lid, kvh, ns, sb, se;
  int P;  // the pair's first unit
  __device__ __forceinline__ static int stages(int ctx) { return (ctx + SP * kQ4Page - 1) / (SP * kQ4Page); }
  __device__ __forceinline__ static int units(int ctx) { return ctx > 0 ? stages(ctx) + 1 : 0; }
  __device__ __forceinline__ void set(const int* ctx, int g0, int g1) {
    ns = stages(ctx[lid]);
    sb = max(0, g0 - P - 1);
    se = min(ns, g1 - P - 1);
  }
  // False when the share holds no further stage.
  __device__ __forceinline__ bool next(const int* ctx, int hkv, int g0, int g1) {
    P += ns + 1;
    if (P + 1 >= g1) return false;
    if (++kvh == hkv) {
      kvh = 0;
      do ++lid;
      while (ctx[lid] == 0);  // a unit before g1 is some lane's
    }
    set(ctx, g0, g1);
    return true;
  }
};

// Shares of the warps, found by every warp for itself: the sum of all units, then the lane that
// holds the share's first one.  ctx: clamped contexts, for the block.  Returns Q; start.lid = -1 when
// the share is empty.  A chunk of 128 lanes is four consecutive ones per thread; the first chunk
// stays in registers.
template <int HD, int SP>
__device__ __forceinline__ int find_share(const AttnQ4Params& p, int gw, int* ctx, PairWalk<SP>& start, int& g0,
                                          int& g1) {
  const int lane = threadIdx.x & 31;
  const int cap = p.max_pages * kQ4Page;
  int ns[4], incl = 0;
  auto chunk = [&](int b0) {  // units of lanes b0 + 4 lane ..; incl: running sum over the threads
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + 4 * lane + i;
      const int c = b < p.lanes ? min(max(p.ctx_lens[b], 0), cap) : 0;
      if (b < p.lanes) ctx[b] = c;  // every warp writes the same values, and reads its own
      ns[i] = PairWalk<SP>::units(c);
    }
    __syncwarp();
    incl = ns[0] + ns[1] + ns[2] + ns[3];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += u;
    }
  };
  int total = 0;
  for (int b0 = (p.lanes - 1) / 128 * 128; b0 >= 0; b0 -= 128) {
    chunk(b0);
    total += __shfl_sync(0xffffffffu, incl, 31);
  }
  total *= p.num_kv_heads;
  const int warps = gridDim.x * kWarps<HD>;
  const int Q = max(1, (int)(((unsigned)total + warps - 1) / (unsigned)warps));
  start.lid = -1;
  // Whole pairs to every CTA, if that is a unit per warp more at most: then no pair is cut between CTAs,
  // and there is no merge over memory (7B heads, 64 lanes of 100 positions: 10.6 us with cuts, 7.6
  // without; of 1200 22.0 and 21.0). Two units more are too many (20 lanes of 1200 13.0 and 13.5).
  const unsigned ctas = gridDim.x, hkv = p.num_kv_heads, pairs = p.lanes * hkv;
  const int longest = __reduce_max_sync(0xffffffffu, max(max(ns[0], ns[1]), max(ns[2], ns[3])));
  if (p.lanes <= 128 && (unsigned long long)((pairs + ctas - 1) / ctas) * longest <= (Q + 1ull) * kWarps<HD>) {
    const int e = incl - (ns[0] + ns[1] + ns[2] + ns[3]);
    auto first_unit = [&](unsigned pair) {
      const unsigned b = pair / hkv, i = b & 3;
      const int before = e + (i > 0 ? ns[0] : 0) + (i > 1 ? ns[1] : 0) + (i > 2 ? ns[2] : 0);
      const int n = i == 0 ? ns[0] : i == 1 ? ns[1] : i == 2 ? ns[2] : ns[3];
      const int lane_first = __shfl_sync(0xffffffffu, before, b >> 2) * hkv;
      const int first = lane_first + (pair - b * hkv) * __shfl_sync(0xffffffffu, n, b >> 2);
      return pair == pairs ? total : first;  // c * pairs < 2^32: 128 lanes of 1024 heads
    };
    const unsigned c = blockIdx.x;
    const int w = gw - c * kWarps<HD>, from = first_unit(c * pairs / ctas), to = first_unit((c + 1) * pairs / ctas);
    const int each = (to - from + kWarps<HD> - 1) / kWarps<HD>;
    g0 = min(from + w * each, to);
    g1 = min(g0 + each, to);
  } else {
    g0 = (int)min((long long)gw * Q, (long long)total);
    g1 = min(total - g0, Q) + g0;
  }
  if (g0 >= g1) return Q;
  const int at = (unsigned)g0 / (unsigned)p.num_kv_heads;  // lane b holds g0 when its sums straddle `at`
  int before = 0;
  for (int b0 = 0;; b0 += 128) {
    const uint32_t hit = __ballot_sync(0xffffffffu, before + incl > at);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int first = before + incl - (ns[0] + ns[1] + ns[2] + ns[3]), i = 0, n = ns[0];
#pragma unroll
      for (int k = 1; k < 4; ++k)
        if (i == k - 1 && first + n <= at) {
          first += n;
          i = k;
          n = ns[k];
        }
      first = __shfl_sync(0xffffffffu, first, src) * p.num_kv_heads;
      start.lid = b0 + 4 * src + __shfl_sync(0xffffffffu, i, src);
      n = __shfl_sync(0xffffffffu, n, src);
      start.kvh = (unsigned)(g0 - first) / (unsigned)n;
      start.P = first + start.kvh * n;
      start.set(ctx, g0, g1);
      if (start.se <= start.sb) start.lid = -1;  // the change of pair alone: the next warp begins it
      return Q;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
    chunk(b0 + 128);
  }
}

// Tickets count the arrivals of a pair's segments; the last arrival clears its ticket.  A launch
// marks its tickets with a number of its own, so whatever else one holds (any contents of a new
// workspace) counts as none: 48 bits tell them apart.  open_ticket() is called early by whoever owns the
// ticket, so that an arrival is one atomic addition as a rule; it does not rely on it.
__device__ __forceinline__ void open_ticket(unsigned long long* ticket, unsigned long long nonce) {
  unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(ticket);
  while (old >> 16 != nonce) {
    const unsigned long long was = atomicCAS(ticket, old, nonce << 16);
    if (was == old) return;
    old = was;
  }
}

// One of `n` arrivals; true for the last.
__device__ __forceinline__ bool last_of(unsigned long long* ticket, unsigned long long nonce, int n) {
  unsigned long long old = atomicAdd(ticket, 1ull);
  if (old >> 16 != nonce) {  // not open yet: the addition went to something that does not count
    open_ticket(ticket, nonce);
    old = atomicAdd(ticket, 1ull);
  }
  if ((int)(old & 0xffffu) + 1 != n) return false;
  atomicExch(ticket, 0ull);
  return true;
}

// One head of a pair from its n partial segments in order: rows at(s) of part_o and part_ml.
template <int HD, typename At>
__device__ __forceinline__ void merge_segments(const AttnQ4Params& p, int pair, int g, int n, int lane, int G, At at) {
  const int d = 4 * (lane % (HD / 4));
  float M = -INFINITY, L = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = lane; s < n; s += 32) M = fmaxf(M, __ldcg(p.part_ml + at(s) * 2));
  M = warp_max(M);
#pragma unroll 8
  for (int s = 0; s < n; ++s) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + at(s) * HD + d));
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at(s) * 2));
    const float x = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
    L = fmaf(ml.y, x, L);
    a.x = fmaf(v.x, x, a.x);
    a.y = fmaf(v.y, x, a.y);
    a.z = fmaf(v.z, x, a.z);
    a.w = fmaf(v.w, x, a.w);
  }
  const float r = L == 0.f ? 0.f : 8.f / L;
  if (lane < HD / 4)
    *reinterpret_cast<float4*>(p.out + (size_t)(pair / p.num_kv_heads) * p.ldo +
                               (size_t)((pair % p.num_kv_heads) * G + g) * HD + d) =
        make_float4(a.x * r, a.y * r, a.z * r, a.w * r);
}

// Position of the k-th set bit.
__device__ __forceinline__ int nth_bit(uint32_t bits, int k) {
  for (; k > 0; --k) bits &= bits - 1;
  return __ffs(bits) - 1;
}

// Clusters that a pair of `ns` stages is cut into: two stages per warp at least.
template <int HD>
__device__ __forceinline__ int pair_clusters(int ns, int most) {
  return min(most, max(1, (ns + 2 * kClusterCtas * kWarps<HD> - 1) / (2 * kClusterCtas * kWarps<HD>)));
}

// The states of a cluster's warps to the pair's output: warp g merges head g over the CTA's
// warps, then one rank merges it over the CTAs, and the last of the pair's clusters to come to
// head g's ticket merges it over the clusters.  A pair of context 0 has no state and gets zeros.
template <int HD>
__device__ __forceinline__ void merge_cluster(const AttnQ4Params& p, uint8_t* smem, const float* state_a,
                                              const float (*ml)[8][2], const int* s_state, int warp, int lane, int G,
                                              int pair, int nclusters) {
  constexpr int ROW = HD + 4;
  static_assert(kWarps<HD> >= 8, "a warp per query head");
  __syncthreads();  // every state is written, every ring idle
  float* part = reinterpret_cast<float*>(smem);  // [G][ROW]: o, maximum, sum
  const int g = warp, d = 4 * (lane % (HD / 4));
  if (g < G) {
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps<HD>; ++w)
      if (s_state[w]) M = fmaxf(M, ml[w][g][0]);
#pragma unroll
    for (int w = 0; w < kWarps<HD>; ++w) {
      if (!s_state[w]) continue;
      const float x = ml[w][g][0] == -INFINITY ? 0.f : ex2(ml[w][g][0] - M);
      const float4 y = *reinterpret_cast<const float4*>(state_a + ((size_t)w * G + g) * ROW + d);
      L = fmaf(ml[w][g][1], x, L);
      a.x = fmaf(y.x, x, a.x);
      a.y = fmaf(y.y, x, a.y);
      a.z = fmaf(y.z, x, a.z);
      a.w = fmaf(y.w, x, a.w);
    }
    if (lane < HD / 4) *reinterpret_cast<float4*>(part + g * ROW + d) = a;
    if (lane == 0) *reinterpret_cast<float2*>(part + g * ROW + HD) = make_float2(M, L);
  }
  cluster_sync_all();  // every CTA's states are visible to the cluster
  const int rank = (int)cluster_ctarank();
  const int head = warp * kClusterCtas + rank;  // heads go to the ranks in turn
  if (head < G) {
    const uint32_t local = smem_u32(part + head * ROW);
    float m[kClusterCtas], M = -INFINITY, L = 0.f;
    float4 y[kClusterCtas], a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kClusterCtas; ++c) {
      const uint32_t at = mapa_shared(local, c);
      m[c] = ld_dsmem_f32(at + 4 * HD);
      y[c] = make_float4(ld_dsmem_f32(at + 4 * d), ld_dsmem_f32(at + 4 * d + 4), ld_dsmem_f32(at + 4 * d + 8),
                         ld_dsmem_f32(at + 4 * d + 12));
      M = fmaxf(M, m[c]);
    }
#pragma unroll
    for (int c = 0; c < kClusterCtas; ++c) {
      const float x = m[c] == -INFINITY ? 0.f : ex2(m[c] - M);
      L = fmaf(ld_dsmem_f32(mapa_shared(local, c) + 4 * HD + 4), x, L);
      a.x = fmaf(y[c].x, x, a.x);
      a.y = fmaf(y[c].y, x, a.y);
      a.z = fmaf(y[c].z, x, a.z);
      a.w = fmaf(y[c].w, x, a.w);
    }
    const bool whole = nclusters == 1;
    const int hkv = p.num_kv_heads;
    const size_t at = (size_t)(blockIdx.x / kClusterCtas) * G + head;
    const float r = !whole ? 1.f : L == 0.f ? 0.f : 8.f / L;
    float* dst = whole ? p.out + (size_t)(pair / hkv) * p.ldo + (size_t)((pair % hkv) * G + head) * HD
                       : p.part_o + at * HD;
    if (lane < HD / 4) *reinterpret_cast<float4*>(dst + d) = make_float4(a.x * r, a.y * r, a.z * r, a.w * r);
    if (!whole && lane == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
  }
  cluster_sync_all();  // keep every CTA's shared memory until the ranks have read it
  if (nclusters > 1 && head < G) {
    __syncwarp();
    bool last = false;
    if (lane == 0) {
      __threadfence();
      last = last_of(p.tickets + pair * G + head, p.nonce, nclusters);
      __threadfence();
    }
    if (__shfl_sync(0xffffffffu, last, 0))
      merge_segments<HD>(p, pair, head, nclusters, lane, G,
                         [&](int s) { return ((size_t)pair * p.clusters + s) * G + head; });
  }
}

// A warp's share is one run of stages: whole pairs, which it finishes by itself, and at most
// two pieces of pairs: one that continues a pair begun before it (state A), then one that
// begins a pair which goes on behind it (state B).  At the end of the CTA the pieces
// merge in shared memory in stage order.  What is cut at the CTA's own ends is written out, at
// most two partial segments per CTA, and the CTA that finds itself to be the last of a pair's takes
// them all together, in order: no second launch, and the result does not depend on which it was.
//
// CLUSTER, for few pairs: clusters of four CTAs per pair instead, as many as its context wants and
// the SMs hold, whose warps take even pieces.  Every piece is a state, and the CTAs' states merge over
// distributed shared memory in rank order.
template <int HD, bool CLUSTER, bool PACK>
__global__ void __launch_bounds__(kWarps<HD> * 32, 1) attn_q4_kernel(const AttnQ4Params p) {
  constexpr int BLK = 18 * HD, SP = kStagePages<HD, CLUSTER>, SPOS = SP * kQ4Page;
  constexpr int NST = kStages<HD, CLUSTER>, IDS = 32 / SP;
  constexpr uint32_t ALL = (1u << SP) - 1;
  constexpr int ROW = HD + 4;  // floats per head of a state
  constexpr int RING = NST * SP * BLK;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) float s_ml[2][kWarps<HD>][8][2];
  __shared__ int s_state[kWarps<HD>];  // 1: state A, 2: and it ends its pair, 4: state B
  __shared__ int s_pair[2][kWarps<HD>], s_first[2][kWarps<HD>];  // of the states; the unit of the pair's first stage
  __shared__ int ctx[kMaxLanes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = p.num_kv_heads, G = p.num_heads / hkv;
  griddep_launch();
  griddep_wait();  // q, the pages, tables and lengths come from earlier kernels
  uint8_t* ring = smem + (size_t)warp * RING;
  float* state_a = reinterpret_cast<float*>(smem + (size_t)kWarps<HD> * RING);  // [warps][G][ROW]
  PairWalk<SP> use;
  int g0 = 0, g1 = 0;
  int Q = 0, pair = 0, nclusters = 1;  // cluster form: the CTA's pair and its clusters
  if constexpr (CLUSTER) {
    const int cluster = blockIdx.x / kClusterCtas;
    pair = cluster / p.clusters;
    use.lid = pair / hkv;
    use.kvh = pair - use.lid * hkv;
    const int c = min(max(p.ctx_lens[use.lid], 0), p.max_pages * kQ4Page);
    ctx[use.lid] = c;  // every warp writes the same value
    use.ns = PairWalk<SP>::stages(c);
    use.P = 0;
    nclusters = pair_clusters<HD>(use.ns, p.clusters);
    const int part = cluster - pair * p.clusters;
    if (part >= nclusters) return;  // the whole cluster
    if (part == 0 && nclusters > 1 && cluster_ctarank() == 0 && threadIdx.x < G)
      open_ticket(p.tickets + pair * G + threadIdx.x, p.nonce);
    // [ns w / all, ns (w + 1) / all), in 32 bits (a 64-bit division takes 0.1 us here).
    constexpr unsigned W = kClusterCtas * kWarps<HD>;
    const unsigned w = part * W + cluster_ctarank() * kWarps<HD> + warp, all = nclusters * W;
    const unsigned each = use.ns / all, rest = use.ns - each * all;
    use.sb = g0 = (int)(each * w + rest * w / all);
    use.se = g1 = (int)(each * (w + 1) + rest * (w + 1) / all);
    if (use.sb == use.se) use.lid = -1;
  } else {
    if (threadIdx.x < G) open_ticket(p.tickets + 8 * blockIdx.x + threadIdx.x, p.nonce);
    Q = find_share<HD, SP>(p, blockIdx.x * kWarps<HD> + warp, ctx, use, g0, g1);
  }
  if (lane == 0) s_state[warp] = 0;
  __syncwarp();  // ctx and the state word are this warp's own writes

  if (use.lid >= 0) {
    float o[HD / 16][4];  // between pairs it holds the next one's q, which costs no registers then
    load_q<HD, PACK>(p, use.lid, use.kvh, G, lane, o);
    // ---- loads: the warp's stages in order, the ring kept full ----
    PairWalk<SP> ld = use;
    const uint64_t pol = l2_evict_first_policy();
    int ld_st = 0, ld_at = 0;  // next stage; its place among the stages whose page ids `ids` holds
    int32_t ids = 0;
    uint32_t ids_ok = 0;             // bit i: page id i is one of the pool's
    const uint8_t* src0 = nullptr;   // this thread's 16 bytes of the head's block in page 0
    auto fetch_ids = [&]() {         // page ids of the next 32 pages, one per thread
      const int j = SP * ld_st + lane;
      const bool inside = j * kQ4Page < ctx[ld.lid];
      ids = inside ? p.tables[(size_t)ld.lid * p.max_pages + j] : 0;
      const bool ok = inside && (unsigned)ids < (unsigned)p.num_pages;
      ids_ok = __ballot_sync(0xffffffffu, ok);
      if (inside && !ok) atomicExch(p.bad, 1);
      if (!ok) ids = 0;
      ld_at = 0;
    };
    auto enter = [&]() {
      ld_st = ld.sb;
      src0 = p.pool + ((size_t)p.layer * hkv + ld.kvh) * BLK + 16 * lane;
      fetch_ids();
    };
    enter();
    const uint32_t ring_at = smem_u32(ring) + 16 * lane;
    uint32_t loaded = 0;  // SP bits per ring slot: the pages that are there
    int slot_in = 0;
    bool ld_more = true;
    auto issue = [&]() {
      if (ld_more && ld_st >= ld.se) {
        ld_more = ld.next(ctx, hkv, g0, g1);
        if (ld_more) enter();
      }
      if (ld_more) {
        if (ld_at == IDS) fetch_ids();
        const uint32_t got = (ids_ok >> (SP * ld_at)) & ALL;
        const uint8_t* src[SP];
#pragma unroll
        for (int i = 0; i < SP; ++i)
          src[i] = src0 + (uint64_t)(uint32_t)__shfl_sync(0xffffffffu, ids, SP * ld_at + i) * p.page_bytes - i * BLK;
        const uint32_t dst = ring_at + slot_in * (SP * BLK);
        // A stage's pages follow one another in the ring: chunks of 16 bytes, one per thread and step.
        // A page that is not there reads page 0 in its place (one path, and no traffic to speak of).
#pragma unroll
        for (int i = 0; i < SP * BLK / 512; ++i) {
          const int lo = 512 * i / BLK, cut = ((lo + 1) * BLK - 512 * i) / 16;  // threads from `cut` on: the next page
          const uint8_t* s = cut < 32 && lane >= cut ? src[lo + 1 < SP ? lo + 1 : lo] : src[lo];
          cp_async16(dst + 512 * i, s + 512 * i, pol);
        }
        loaded = (loaded & ~(ALL << (SP * slot_in))) | got << (SP * slot_in);
        ++ld_st;
        ++ld_at;
      }
      cp_async_commit();
      slot_in = slot_in + 1 == NST ? 0 : slot_in + 1;
    };
    int ahead = 0;  // stages in the ring, this one included

    // ---- arithmetic ----
    int slot = 0;
    bool fresh = true;  // a pair begins
    const int h = lane >> 2, t = lane & 3;
    QFrag<HD> q;
    float m = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    int st = 0, left = 0;
#pragma unroll 1
    for (;;) {
      __syncwarp();  // nobody reads the slot of the stage before any more
#pragma unroll 1
      for (; ahead < NST; ++ahead) issue();
      --ahead;
      if (fresh) {
        split_q<HD>(p, o, q);
        m = -INFINITY;
        l2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
        st = use.sb;
        left = ctx[use.lid] - SPOS * st;  // positions from this stage on
        fresh = false;
      }
      cp_async_wait<NST - 1>();
      __syncwarp();  // this stage is there for every thread
      const uint32_t pages = (loaded >> (SP * slot)) & ALL;
      const uint8_t* buf = ring + slot * (SP * BLK);
      float2 sc[2 * SP];
      stage_scores<HD, SP>(buf, q, sc, lane);
      uint32_t keep[2 * SP];
#pragma unroll
      for (int i = 0; i < 2 * SP; ++i) keep[i] = 0xffffffffu;
      if (left < SPOS || pages != ALL) {
        // Positions past the context, and of pages that are not there.
#pragma unroll
        for (int i = 0; i < 2 * SP; ++i) {
          const int in = (pages >> (i / 2) & 1) ? left - 8 * i - 2 * t : 0;  // this thread's two positions
          if (in < 1) sc[i].x = -INFINITY;
          if (in < 2) sc[i].y = -INFINITY;
          keep[i] = in < 1 ? 0u : in < 2 ? 0xffffu : 0xffffffffu;
        }
      }
      stage_values<HD, SP, PACK>(buf, q, sc, keep, m, l2, o, lane);
      slot = slot + 1 == NST ? 0 : slot + 1;
      left -= SPOS;
      if (++st < use.se) continue;
      __syncwarp();  // the last stage is read
      const PairWalk<SP> done = use;
      float l = l2.x + l2.y;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if constexpr (PACK) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][c] += __shfl_xor_sync(0xffffffffu, o[i][c], 2);
      }
      const bool begins = !CLUSTER && done.sb == 0, ends = done.se == done.ns;
      const int which = begins ? 1 : 0;
      // A whole pair goes out; a piece to its state (B only at the share's end, over the idle ring).
      float* d = begins && ends ? p.out + (size_t)done.lid * p.ldo + (size_t)done.kvh * G * HD
                 : begins       ? reinterpret_cast<float*>(ring)
                                : state_a + (size_t)warp * G * ROW;
      const int row = begins && ends ? HD : ROW;
      const float r = begins && ends ? (l == 0.f ? 0.f : 8.f / l) : 1.f;
      // This thread holds dims h hd/8 .. + hd/8 - 1 of heads 2t and 2t + 1.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float rc = __shfl_sync(0xffffffffu, r, 8 * t + 4 * c);
        if (2 * t + c < G) {
          float* dc = d + (2 * t + c) * row + (HD / 8) * h;
#pragma unroll
          for (int k = 0; k < HD / 32; ++k)
            *reinterpret_cast<float4*>(dc + 4 * k) = make_float4(o[2 * k][c] * rc, o[2 * k][c + 2] * rc,
                                                                 o[2 * k + 1][c] * rc, o[2 * k + 1][c + 2] * rc);
        }
      }
      if (h < G && t == 0 && !(begins && ends)) {
        s_ml[which][warp][h][0] = m * q.f;
        s_ml[which][warp][h][1] = l;
      }
      if (lane == 0 && !(begins && ends)) {
        s_state[warp] |= begins ? 4 : ends ? 3 : 1;
        if (begins || warp == 0) s_first[which][warp] = done.P + 1;
        s_pair[which][warp] = done.lid * hkv + done.kvh;
      }
      if (!use.next(ctx, hkv, g0, g1)) break;
      load_q<HD, PACK>(p, use.lid, use.kvh, G, lane, o);
      fresh = true;
    }
  }
  if constexpr (CLUSTER) {
    merge_cluster<HD>(p, smem, state_a, s_ml[0], s_state, warp, lane, G, pair, nclusters);
  } else {
    // Lanes of context 0 get zeros.
    for (int b = blockIdx.x; b < p.lanes; b += gridDim.x)
      if (ctx[b] == 0)
        for (int i = threadIdx.x; i < p.num_heads * HD; i += kWarps<HD> * 32) p.out[(size_t)b * p.ldo + i] = 0.f;
    __syncthreads();

    // ---- pieces.  Chain 0 starts with A of warp 0, chain 1 + w with B of warp w; each goes on with
    // the A's behind it until one ends its pair.  A warp takes one head of a chain when there are warps
    // enough, up to four otherwise; its threads take the dims.  The first chain and the last come
    // first: theirs are the pairs that are cut. ----
    constexpr uint32_t WARPS = (1u << kWarps<HD>) - 1;
    const int st = lane < kWarps<HD> ? s_state[lane] : 0;
    const uint32_t is_b = __ballot_sync(0xffffffffu, st & 4) & WARPS,
                   is_1 = __ballot_sync(0xffffffffu, (st & 3) == 1) & WARPS,
                   is_3 = __ballot_sync(0xffffffffu, (st & 3) == 3) & WARPS;
    const uint32_t chains = is_b << 1 | ((is_1 | is_3) & 1u);
    const int d = 4 * (lane % (HD / 4)), num_chains = __popc(chains);
    int per = 1;  // heads per task
    while (per < kPart && num_chains * ((G + per - 1) / per) > kWarps<HD>) ++per;
    const int parts = (G + per - 1) / per;
#pragma unroll 1
    for (int task = warp; task < num_chains * parts; task += kWarps<HD>) {
      const int k = task / parts, h0 = (task - k * parts) * per, heads = min(per, G - h0);
      const int chain = k == 1 ? 31 - __clz(chains) : nth_bit(chains, max(k - 1, 0));
      const int first = chain ? chain - 1 : 0;           // warp of the chain's first state
      const int from = chain ? first + 1 : 0;            // its first A
      const int stop = __ffs(~is_1 >> from) - 1 + from;  // the first warp from there whose A does not go on
      const bool ended = is_3 >> stop & 1;
      const int end = ended ? stop + 1 : stop;  // states of warps [first, end), the first as B unless chain 0
      float M[kPart], L[kPart];
      float4 a[kPart];
#pragma unroll
      for (int g = 0; g < kPart; ++g) {
        M[g] = -INFINITY;
        L[g] = 0.f;
        a[g] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      // One more state of head g.
      auto add = [&](int g, float2 ml, float4 y) {
        const float Mn = fmaxf(M[g], ml.x);
        const float x = M[g] == -INFINITY ? 0.f : ex2(M[g] - Mn), z = ml.x == -INFINITY ? 0.f : ex2(ml.x - Mn);
        M[g] = Mn;
        L[g] = L[g] * x + ml.y * z;
        a[g].x = a[g].x * x + y.x * z;
        a[g].y = a[g].y * x + y.y * z;
        a[g].z = a[g].z * x + y.z * z;
        a[g].w = a[g].w * x + y.w * z;
      };
#pragma unroll 1
      for (int w = first; w < end; ++w) {
        const bool b = chain && w == first;
        const float(*ml)[2] = s_ml[b ? 1 : 0][w] + h0;
        const float* src = b ? reinterpret_cast<const float*>(smem + (size_t)w * RING) : state_a + (size_t)w * G * ROW;
        src += h0 * ROW + d;
#pragma unroll
        for (int g = 0; g < kPart; ++g)
          if (g < heads)
            add(g, *reinterpret_cast<const float2*>(ml[g]), *reinterpret_cast<const float4*>(src + g * ROW));
      }
      const int pair = s_pair[chain ? 1 : 0][first];
      float* out = p.out + (size_t)(pair / hkv) * p.ldo + (size_t)((pair % hkv) * G + h0) * HD + d;
      uint32_t write = (1u << heads) - 1;  // a whole pair's heads
      if (!(chain && ended)) {
        // A segment of a pair that is cut at the CTA's front or end.
        const size_t part = (2 * (size_t)blockIdx.x + (chain ? 1 : 0)) * G + h0;
        float2 mine = make_float2(0.f, 0.f);
#pragma unroll
        for (int g = 0; g < kPart; ++g) {
          if (g < heads && lane < HD / 4) *reinterpret_cast<float4*>(p.part_o + (part + g) * HD + d) = a[g];
          if (lane == g) mine = make_float2(M[g], L[g]);
        }
        if (lane < heads) *reinterpret_cast<float2*>(p.part_ml + (part + lane) * 2) = mine;
        const int units = Q * kWarps<HD>, begin = s_first[chain ? 1 : 0][first];
        const int ns = PairWalk<SP>::stages(ctx[pair / hkv]);
        const int c0 = begin / units, n = (begin + ns - 1) / units - c0 + 1;  // its first CTA, its CTAs
        __syncwarp();
        bool last = false;
        if (lane < heads) {
          __threadfence();
          last = last_of(p.tickets + 8 * c0 + h0 + lane, p.nonce, n);
          __threadfence();
        }
        write = __ballot_sync(0xffffffffu, last);
        __syncwarp();
        if (write) {
          // All are there: CTA c0's last segment, then the first ones of the CTAs behind it.
#pragma unroll
          for (int g = 0; g < kPart; ++g) {
            M[g] = -INFINITY;
            L[g] = 0.f;
            a[g] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll 1
          for (int s = 0; s < n; ++s) {
            const size_t at = (s == 0 ? 2 * (size_t)c0 + 1 : 2 * (size_t)(c0 + s)) * G + h0;
            float2 ml[kPart];
            float4 y[kPart];
#pragma unroll
            for (int g = 0; g < kPart; ++g) {
              if (write >> g & 1) {
                ml[g] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (at + g) * 2));
                y[g] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (at + g) * HD + d));
              }
            }
#pragma unroll
            for (int g = 0; g < kPart; ++g)
              if (write >> g & 1) add(g, ml[g], y[g]);
          }
        }
      }
      if (write) {
#pragma unroll
        for (int g = 0; g < kPart; ++g) {
          const float r = L[g] == 0.f ? 0.f : 8.f / L[g];
          if ((write >> g & 1) && lane < HD / 4)
            *reinterpret_cast<float4*>(out + g * HD) = make_float4(a[g].x * r, a[g].y * r, a[g].z * r, a[g].w * r);
        }
      }
    }
  }
}

// The cluster form: about as many clusters of four CTAs as fit on the SMs at once (33 of eight GPCs,
// while clusters of eight leave 28 of the 148 SMs out).
constexpr size_t kClusters = 32;

}  // namespace

// Tickets: one per head and CTA, or pair of the cluster form.
static size_t ticket_floats() { return 2 * 8 * std::max((size_t)sm_count(), kClusters); }

// The tickets and two partial segments per CTA (one that begins a pair, one that continues it).
size_t attention_q4_workspace_floats(size_t num_heads, size_t num_kv_heads, size_t head_dim) {
  if (!num_kv_heads) return 0;
  const size_t ctas = (size_t)sm_count();
  return ticket_floats() + 2 * ctas * (num_heads / num_kv_heads) * (head_dim + 2);
}

int paged_attention_q4(const float* q, size_t ldq, const void* pool, size_t num_pages, size_t num_layers,
                       const int32_t* block_tables, size_t max_pages, const int32_t* ctx_lens, size_t lanes,
                       size_t layer, size_t num_heads, size_t num_kv_heads, size_t head_dim, float* out, size_t ldo,
                       float* workspace, size_t workspace_floats, cudaStream_t stream) {
  GLC_REQUIRE(q && block_tables && ctx_lens && out && workspace, "paged_attention_q4: null argument");
  int rc = q4_check_pool("paged_attention_q4", pool, num_pages, num_layers, layer, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  GLC_REQUIRE(lanes > 0 && lanes <= (size_t)kMaxLanes, "paged_attention_q4: %zu lanes (1 to %d)", lanes, kMaxLanes);
  GLC_REQUIRE(max_pages > 0 && max_pages <= ((size_t)1 << 26) &&
                  lanes * num_kv_heads * max_pages < ((size_t)1 << 31),
              "paged_attention_q4: %zu pages per lane (at most 2^26, and 2^31 with lanes * kv heads)", max_pages);
  GLC_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0 && ldq % 4 == 0 &&
                  ldo % 4 == 0,
              "paged_attention_q4: q, out and workspace must be 16-byte aligned");
  const size_t need = attention_q4_workspace_floats(num_heads, num_kv_heads, head_dim);
  GLC_REQUIRE(workspace_floats >= need, "paged_attention_q4: workspace of %zu floats needed", need);
  const size_t page_bytes = num_layers * num_kv_heads * q4_block_bytes(head_dim);
  GLC_REQUIRE(page_bytes < ((size_t)1 << 32), "paged_attention_q4: pages of %zu bytes", page_bytes);
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
  // Every launch marks its tickets with a number of its own; a captured one keeps its, and finds the
  // tickets cleared by the replay before.
  static std::atomic<unsigned long long> launches{
      (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
  do p.nonce = launches.fetch_add(1, std::memory_order_relaxed) & 0xffffffffffffull;
  while (p.nonce == 0);
  p.tickets = reinterpret_cast<unsigned long long*>(workspace);
  p.part_o = workspace + ticket_floats();
  p.part_ml = p.part_o + 2 * (size_t)grid * G * head_dim;
  p.page_bytes = (uint32_t)page_bytes;
  p.lanes = (int)lanes;
  p.max_pages = (int)max_pages;
  p.num_pages = (int)num_pages;
  p.layer = (int)layer;
  p.num_heads = (int)num_heads;
  p.num_kv_heads = (int)num_kv_heads;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  p.bad = ops_error_word();
  GLC_REQUIRE(p.bad, "paged_attention_q4: device status word unavailable");
  const size_t pairs = lanes * num_kv_heads;
  const bool cluster = pairs <= kClusters;
  p.clusters = cluster ? (int)(kClusters / pairs) : 0;
  using Kern = void (*)(AttnQ4Params);
  static const Kern kerns[8] = {attn_q4_kernel<64, false, false>, attn_q4_kernel<64, false, true>,
                                attn_q4_kernel<64, true, false>,  attn_q4_kernel<64, true, true>,
                                attn_q4_kernel<128, false, false>, attn_q4_kernel<128, false, true>,
                                attn_q4_kernel<128, true, false>,  attn_q4_kernel<128, true, true>};
  const Kern kern = kerns[(head_dim == 128 ? 4 : 0) + (cluster ? 2 : 0) + (G <= 4 ? 1 : 0)];
  const size_t warps = head_dim == 128 ? kWarps<128> : kWarps<64>;
  const size_t pages = head_dim == 128 ? (cluster ? kStagePages<128, true> * kStages<128, true>
                                                  : kStagePages<128, false> * kStages<128, false>)
                                       : kStagePages<64, true> * kStages<64, true>;  // of a warp's ring
  static_assert(kStagePages<64, true> * kStages<64, true> == kStagePages<64, false> * kStages<64, false>);
  const size_t smem = warps * (pages * q4_block_bytes(head_dim) + G * (head_dim + 4) * sizeof(float));
  if ((rc = allow_dynamic_smem((const void*)kern, (int)smem))) return rc;
  if (cluster)
    return launch_pdl(kern, dim3((unsigned)(pairs * p.clusters * kClusterCtas)), dim3((unsigned)warps * 32), smem,
                      stream, kClusterCtas, p);
  return launch_pdl(kern, dim3((unsigned)grid), dim3((unsigned)warps * 32), smem, stream, 1, p);
}

}  // namespace glacier
