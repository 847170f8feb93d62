// Paged decode attention over the 4-bit cache (kv_q4.cuh): attentionMultiHead
// (src/paged_attention.zig:108-216) for one query row per lane, as
// glacier_cuda_paged_attention_f32, with K and V read as 4-bit codes.
#include "kv_q4.cuh"

namespace glacier {

namespace {

constexpr int kWarps = 8;

struct AttnQ4Params {
  const float* q;
  const uint8_t* pool;
  const int32_t* tables;
  const int32_t* ctx_lens;
  float* out;
  size_t page_bytes;
  int max_pages, num_pages, layer, num_heads, num_kv_heads;
  float scale_log2;
  int* bad;
};

// One CTA per (kv head, lane), its warps taking positions in turn: each lane of a warp
// holds HD/32 dims of q for the G heads, keeps a running maximum, sum and output, and
// the warps' states merge in shared memory in warp order.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) attn_q4_kernel(const AttnQ4Params p) {
  constexpr int VD = HD / 32;
  __shared__ float s_m[kWarps][8], s_l[kWarps][8], s_o[kWarps][8][HD];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int G = p.num_heads / p.num_kv_heads;
  const int ctx = min(max(p.ctx_lens[b], 0), p.max_pages * kQ4Page);
  float q[8][VD], m[8], l[8], acc[8][VD];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < VD; ++i) {
      acc[g][i] = 0.f;
      q[g][i] = g < G ? p.q[((size_t)b * p.num_heads + kvh * G + g) * HD + VD * lane + i] * p.scale_log2 : 0.f;
    }
  }
  for (int pos = warp; pos < ctx; pos += kWarps) {
    const int page = p.tables[(size_t)b * p.max_pages + pos / kQ4Page];
    if ((unsigned)page >= (unsigned)p.num_pages) {
      if (lane == 0) atomicExch(p.bad, 1);
      continue;
    }
    const uint8_t* blk = p.pool + (size_t)page * p.page_bytes +
                         ((size_t)p.layer * p.num_kv_heads + kvh) * q4_block_bytes(HD);
    const int row = pos % kQ4Page;
    float k[VD], v[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) {
      const int d = VD * lane + i, sh = 4 * (d & 3);
      const int g = d / kQ4Group;
      const float ks = __half2float(*reinterpret_cast<const __half*>(blk + q4_scale(HD, 0, row, g)));
      const float vs = __half2float(*reinterpret_cast<const __half*>(blk + q4_scale(HD, 1, row, g)));
      k[i] = ks * (float)(int)(((*reinterpret_cast<const uint16_t*>(blk + q4_k_quad(HD, row, d / 4)) >> sh) & 15) - 7);
      v[i] = vs * (float)(int)(((*reinterpret_cast<const uint16_t*>(blk + q4_v_quad(HD, row, d / 4)) >> sh) & 15) - 7);
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < VD; ++i) s = fmaf(q[g][i], k[i], s);
      s = warp_sum(s);
      const float mn = fmaxf(m[g], s);
      const float a = exp2f(m[g] - mn), e = exp2f(s - mn);
      m[g] = mn;
      l[g] = l[g] * a + e;
#pragma unroll
      for (int i = 0; i < VD; ++i) acc[g][i] = acc[g][i] * a + e * v[i];
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if (lane == 0) {
      s_m[warp][g] = m[g];
      s_l[warp][g] = l[g];
    }
#pragma unroll
    for (int i = 0; i < VD; ++i) s_o[warp][g][VD * lane + i] = acc[g][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * HD; e += blockDim.x) {
    const int g = e / HD, d = e % HD;
    float M = -INFINITY, L = 0.f, o = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][g]);
    for (int w = 0; w < kWarps; ++w) {
      const float a = s_l[w][g] == 0.f ? 0.f : exp2f(s_m[w][g] - M);
      L += s_l[w][g] * a;
      o += s_o[w][g][d] * a;
    }
    p.out[((size_t)b * p.num_heads + kvh * G + g) * HD + d] = L == 0.f ? 0.f : o / L;
  }
}

}  // namespace

size_t attention_q4_workspace_floats(size_t num_heads, size_t num_kv_heads, size_t head_dim) {
  if (!num_kv_heads) return 0;
  return 4 + 2 * (size_t)sm_count() * (num_heads / num_kv_heads) * (head_dim + 2);
}

int paged_attention_q4(const float* q, size_t ldq, const void* pool, size_t num_pages, size_t num_layers,
                       const int32_t* block_tables, size_t max_pages, const int32_t* ctx_lens, size_t lanes,
                       size_t layer, size_t num_heads, size_t num_kv_heads, size_t head_dim, float* out, size_t ldo,
                       float* workspace, size_t workspace_floats, cudaStream_t stream) {
  GLC_REQUIRE(q && block_tables && ctx_lens && out && workspace, "paged_attention_q4: null argument");
  int rc = q4_check_pool("paged_attention_q4", pool, num_pages, num_layers, layer, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  GLC_REQUIRE(lanes > 0 && lanes <= 1024, "paged_attention_q4: %zu lanes (1 to 1024)", lanes);
  GLC_REQUIRE(max_pages > 0 && max_pages <= ((size_t)1 << 26), "paged_attention_q4: %zu pages per lane", max_pages);
  GLC_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)workspace % 16 == 0,
              "paged_attention_q4: q, out and workspace must be 16-byte aligned");
  GLC_REQUIRE(workspace_floats >= attention_q4_workspace_floats(num_heads, num_kv_heads, head_dim),
              "paged_attention_q4: workspace of %zu floats needed",
              attention_q4_workspace_floats(num_heads, num_kv_heads, head_dim));
  AttnQ4Params p;
  p.q = q;
  p.pool = static_cast<const uint8_t*>(pool);
  p.tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.out = out;
  p.page_bytes = num_layers * num_kv_heads * q4_block_bytes(head_dim);
  p.max_pages = (int)max_pages;
  p.num_pages = (int)num_pages;
  p.layer = (int)layer;
  p.num_heads = (int)num_heads;
  p.num_kv_heads = (int)num_kv_heads;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  p.bad = ops_error_word();
  GLC_REQUIRE(p.bad, "paged_attention_q4: device status word unavailable");
  const dim3 grid((unsigned)num_kv_heads, (unsigned)lanes);
  return launch_pdl(head_dim == 128 ? attn_q4_kernel<128> : attn_q4_kernel<64>, grid, dim3(kWarps * 32), 0, stream, 1,
                    p);
}

}  // namespace glacier
