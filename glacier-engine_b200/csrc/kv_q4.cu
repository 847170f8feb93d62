// Writing and reading the 4-bit paged KV cache (kv_q4.cuh): RoPE + quantise + append,
// and rows back as float32.
#include <float.h>

#include "kv_q4.cuh"

namespace glacier {

int q4_check_pool(const char* who, const void* pool, size_t num_pages, size_t num_layers, size_t layer,
                  size_t num_heads, size_t num_kv_heads, size_t head_dim) {
  GLC_REQUIRE(pool && (uintptr_t)pool % 16 == 0, "%s: the pool is null or not 16-byte aligned", who);
  GLC_REQUIRE(num_pages > 0 && num_pages < ((size_t)1 << 31) && layer < num_layers && num_layers < ((size_t)1 << 16),
              "%s: %zu pages, layer %zu of %zu", who, num_pages, layer, num_layers);
  GLC_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %zu (64 or 128)", who, head_dim);
  GLC_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 1024 && num_heads % num_kv_heads == 0 && num_heads > 0 &&
                  num_heads / num_kv_heads <= 8,
              "%s: %zu heads over %zu kv heads (a multiple, at most 8 times)", who, num_heads, num_kv_heads);
  return GLACIER_CUDA_OK;
}

namespace {

// The scale of a group whose largest magnitude is `top`: the smallest multiple of
// 2^-21 with 7 significant bits and 7 s >= top, at most 7168.  top / 7 rounds to
// nearest, so its rounded-up grid value can only be one unit short, and 7 s is exact.
__device__ __forceinline__ float q4_scale_of(float top) {
  const float t = __fdiv_rn(top, 7.f);
  const int e = max((int)(__float_as_uint(t) >> 23) - 127 - 6, -21);
  const float unit = __uint_as_float((uint32_t)(e + 127) << 23);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  if (!(t < kQ4MaxScale)) return kQ4MaxScale;
  float s = ceilf(t * inv) * unit;
  if (7.f * s < top) s += unit;
  return fminf(s, kQ4MaxScale);
}

// 7 + x / s to the nearest integer, ties to even, within [0, 15]: exact, because the
// remainder x - r s of the rounded quotient is (11 bits times a power of two below x).
__device__ __forceinline__ uint32_t q4_code(float x, float s, float inv) {
  float r = fminf(fmaxf(rintf(x * inv), -7.f), 8.f);
  const float d = fmaf(-r, s, x), h = 0.5f * s;
  const bool odd = ((int)r & 1) != 0;
  if (d > h || (d == h && odd)) r += 1.f;
  if (d < -h || (d == -h && odd)) r -= 1.f;
  return (uint32_t)((int)fminf(fmaxf(r, -7.f), 8.f) + 7);
}

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p) {
  if constexpr (VEC) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}

// RopeTable.apply (src/generate.zig:816-831) + appendRowTxn (paged_kv_cache.zig:1074)
// into the 4-bit cache.  head_dim / 4 threads hold one head's row, four dims each: the
// rotation's partner (dim + head_dim/2) is a shuffle away, a scale group is eight
// threads, and each thread's four codes are the 16-bit unit that both layouts keep
// together, so no two threads and no two positions share a byte.  Bias, products
// and their sum are each rounded to float32 (no contraction): the codes are those of
// the row that the float32 cache would hold.
// Launch and one dependent chain of loads (slot and position, row, angles) bound it: 1.9 us for one row of
// 14/2 heads of 64, 2.9 for 128 rows of 28/4 heads of 128 (4.3 MB, 0.7 us at the copy rate), in a CUDA graph.
template <int HD, bool VEC>
__global__ void __launch_bounds__(256)
    qkv_rope_append_q4_kernel(const float* __restrict__ qkv, size_t ld, size_t split_stride, int nsplit,
                              const float* __restrict__ bias, const float* __restrict__ cos_t,
                              const float* __restrict__ sin_t, int positions, const int32_t* __restrict__ pos,
                              const int64_t* __restrict__ slots, int num_heads, int num_kv_heads,
                              float* __restrict__ q_out, size_t ldq, uint8_t* __restrict__ pool, int64_t num_slots,
                              size_t page_bytes, int layer, int* __restrict__ bad) {
  constexpr int T = HD / 4;  // threads per head row
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.x;
  const int r = blockIdx.y * (256 / T) + threadIdx.x / T;  // head row: q heads, k heads, v heads
  const int l = threadIdx.x % T;
  const int nrows = num_heads + 2 * num_kv_heads;
  const int64_t slot = slots[b];
  const int p = pos[b];
  // A padding row (slot -1) writes a zero q and no K/V; a slot outside the pool or a
  // position outside the RoPE table does the same and raises the bad-input word.
  const bool live = slot >= 0 && slot < num_slots && p >= 0 && p < positions;
  if (!live) {
    if (threadIdx.x == 0 && blockIdx.y == 0 && slot != -1) atomicExch(bad, 1);
    if (r < num_heads) {
      float* dst = q_out + (size_t)b * ldq + (size_t)r * HD + 4 * l;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = 0.f;
    }
    return;
  }
  const bool on = r < nrows;
  const int row = on ? r : nrows - 1;  // idle threads of the last block follow a real row
  const size_t col = (size_t)row * HD + 4 * l;
  const float* src = qkv + (size_t)b * ld + col;
  float4 x4 = load4<VEC>(src);
#pragma unroll 4
  for (int s = 1; s < nsplit; ++s) {  // split-K partials in split order
    const float4 u = load4<VEC>(src + (size_t)s * split_stride);
    x4.x += u.x; x4.y += u.y; x4.z += u.z; x4.w += u.w;
  }
  if (bias) {
    const float4 c = load4<VEC>(bias + col);
    x4.x += c.x; x4.y += c.y; x4.z += c.z; x4.w += c.w;
  }
  float x[4] = {x4.x, x4.y, x4.z, x4.w};
  if (__any_sync(0xffffffffu, row < num_heads + num_kv_heads)) {
    const int j = (4 * l) % (HD / 2);
    const float4 c4 = load4<VEC>(cos_t + (size_t)p * (HD / 2) + j), s4 = load4<VEC>(sin_t + (size_t)p * (HD / 2) + j);
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
    const bool upper = l >= T / 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o = __shfl_xor_sync(0xffffffffu, x[i], T / 2);
      const float xc = __fmul_rn(x[i], c[i]), os = __fmul_rn(o, s[i]);
      const float y = upper ? __fadd_rn(os, xc) : __fsub_rn(xc, os);
      if (row < num_heads + num_kv_heads) x[i] = y;
    }
  }
  if (row < num_heads) {
    if (!on) return;
    float* dst = q_out + (size_t)b * ldq + col;
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = x[i];
    }
    return;
  }
  // ---- quantise: one scale per 32 dims (8 threads) ----
  const unsigned group_mask = 0xffu << (threadIdx.x & 24);
  float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  bool fin = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) fin = fin && fabsf(x[i]) <= FLT_MAX;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(group_mask, top, o));
  fin = __all_sync(group_mask, fin);
  const float s = fin ? q4_scale_of(top) : 0.f;
  const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  uint32_t u = 0x7777u;
  if (s > 0.f) {
    u = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) u |= q4_code(x[i], s, inv) << (4 * i);
  }
  if (!on) return;
  const int kind = row >= num_heads + num_kv_heads ? 1 : 0;
  const int head = row - num_heads - kind * num_kv_heads;
  uint8_t* blk = pool + (size_t)(slot >> 4) * page_bytes +
                 ((size_t)layer * num_kv_heads + head) * q4_block_bytes(HD);
  const int pr = (int)(slot & 15);
  *reinterpret_cast<uint16_t*>(blk + (kind ? q4_v_quad(HD, pr, l) : q4_k_quad(HD, pr, l))) = (uint16_t)u;
  if (l % 8 == 0)  // a NaN scale poisons a group that held a NaN or an infinity
    *reinterpret_cast<uint16_t*>(blk + q4_scale(HD, kind, pr, l / 8)) =
        fin ? __half_as_ushort(__float2half_rn(s)) : (uint16_t)0x7E00;
}

// The held values of K and V rows at `slots`, one head row per HD/4 threads (1.0 us for one row, 1.4 for 128).
template <int HD>
__global__ void __launch_bounds__(256)
    kv_q4_read_kernel(const uint8_t* __restrict__ pool, int64_t num_slots, size_t page_bytes, int layer,
                      const int64_t* __restrict__ slots, int num_kv_heads, float* __restrict__ k_out,
                      float* __restrict__ v_out, int* __restrict__ bad) {
  constexpr int T = HD / 4;
  griddep_launch();
  griddep_wait();
  const size_t b = blockIdx.x;
  const int r = blockIdx.y * (256 / T) + threadIdx.x / T, l = threadIdx.x % T;
  if (r >= 2 * num_kv_heads) return;
  const int kind = r >= num_kv_heads ? 1 : 0, head = r - kind * num_kv_heads;
  const int64_t slot = slots[b];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (slot >= 0 && slot < num_slots) {
    const uint8_t* blk = pool + (size_t)(slot >> 4) * page_bytes +
                         ((size_t)layer * num_kv_heads + head) * q4_block_bytes(HD);
    const int pr = (int)(slot & 15);
    const uint32_t u = *reinterpret_cast<const uint16_t*>(blk + (kind ? q4_v_quad(HD, pr, l) : q4_k_quad(HD, pr, l)));
    const float s = __half2float(*reinterpret_cast<const __half*>(blk + q4_scale(HD, kind, pr, l / 8)));
    v = make_float4(s * (float)((int)(u & 15) - 7), s * (float)((int)(u >> 4 & 15) - 7),
                    s * (float)((int)(u >> 8 & 15) - 7), s * (float)((int)(u >> 12) - 7));
  } else if (slot != -1 && threadIdx.x == 0 && blockIdx.y == 0) {
    atomicExch(bad, 1);
  }
  float* dst = (kind ? v_out : k_out) + (b * num_kv_heads + head) * HD + 4 * l;
  *reinterpret_cast<float4*>(dst) = v;
}

}  // namespace

int qkv_rope_append_q4(const float* qkv, size_t ld, size_t split_stride, int nsplit, const float* bias,
                       const float* cos_t, const float* sin_t, size_t positions, const int32_t* pos,
                       const int64_t* slots, size_t batch, size_t num_heads, size_t num_kv_heads, size_t head_dim,
                       float* q_out, size_t ldq, void* pool, size_t num_pages, size_t num_layers, size_t layer,
                       cudaStream_t stream) {
  GLC_REQUIRE(cos_t && sin_t && ((qkv && pos && slots && q_out) || batch == 0), "qkv_rope_append_q4: null argument");
  int rc = q4_check_pool("qkv_rope_append_q4", pool, num_pages, num_layers, layer, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  const size_t nrows = num_heads + 2 * num_kv_heads;
  GLC_REQUIRE(ld >= nrows * head_dim && ldq >= num_heads * head_dim, "qkv_rope_append_q4: row strides %zu / %zu", ld,
              ldq);
  GLC_REQUIRE(positions > 0 && positions < ((size_t)1 << 31) && batch < ((size_t)1 << 31),
              "qkv_rope_append_q4: %zu positions, %zu rows", positions, batch);
  if (batch == 0) return GLACIER_CUDA_OK;
  auto a16 = [](const void* p) { return (uintptr_t)p % 16 == 0; };
  const bool vec = ld % 4 == 0 && split_stride % 4 == 0 && ldq % 4 == 0 && a16(qkv) && a16(bias) && a16(cos_t) &&
                   a16(sin_t) && a16(q_out);
  const size_t page_bytes = num_layers * num_kv_heads * q4_block_bytes(head_dim);
  const dim3 grid((unsigned)batch, (unsigned)ceil_div(nrows, 256 / (head_dim / 4)));
  auto kern = head_dim == 128 ? (vec ? qkv_rope_append_q4_kernel<128, true> : qkv_rope_append_q4_kernel<128, false>)
                              : (vec ? qkv_rope_append_q4_kernel<64, true> : qkv_rope_append_q4_kernel<64, false>);
  int* bad = ops_error_word();
  GLC_REQUIRE(bad, "qkv_rope_append_q4: device status word unavailable");
  return launch_pdl(kern, grid, dim3(256), 0, stream, 1, qkv, ld, split_stride, nsplit, bias, cos_t, sin_t,
                    (int)positions, pos, slots, (int)num_heads, (int)num_kv_heads, q_out, ldq, (uint8_t*)pool,
                    (int64_t)num_pages * kQ4Page, page_bytes, (int)layer, bad);
}

int kv_q4_read(const void* pool, size_t num_pages, size_t num_layers, size_t layer, size_t num_kv_heads,
               size_t head_dim, const int64_t* slots, size_t rows, float* k_out, float* v_out, cudaStream_t stream) {
  GLC_REQUIRE(((slots && k_out && v_out) || rows == 0) && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
              "kv_q4_read: null or unaligned argument");
  int rc = q4_check_pool("kv_q4_read", pool, num_pages, num_layers, layer, num_kv_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  GLC_REQUIRE(rows < ((size_t)1 << 31), "kv_q4_read: %zu rows", rows);
  if (rows == 0) return GLACIER_CUDA_OK;
  const size_t page_bytes = num_layers * num_kv_heads * q4_block_bytes(head_dim);
  const dim3 grid((unsigned)rows, (unsigned)ceil_div(2 * num_kv_heads, 256 / (head_dim / 4)));
  auto kern = head_dim == 128 ? kv_q4_read_kernel<128> : kv_q4_read_kernel<64>;
  int* bad = ops_error_word();
  GLC_REQUIRE(bad, "kv_q4_read: device status word unavailable");
  return launch_pdl(kern, grid, dim3(256), 0, stream, 1, (const uint8_t*)pool, (int64_t)num_pages * kQ4Page,
                    page_bytes, (int)layer, slots, (int)num_kv_heads, k_out, v_out, bad);
}

}  // namespace glacier
