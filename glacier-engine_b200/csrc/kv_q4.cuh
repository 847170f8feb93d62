// The 4-bit paged KV cache: its byte layout and the numbers it holds.
//
// A page holds 16 positions of every layer (PagedKVCache's page,
// src/paged_kv_cache.zig:16).  The block of one (page, layer, kv head) is
// 18 * head_dim contiguous bytes, K and V with their scales, a multiple of 16: the
// attention kernel copies them in 16-byte chunks, the pages of a stage end to end:
//
//   K codes   [16 positions][4 t][head_dim/32 g]  u32: dims 32g+8t .. 32g+8t+7
//   V codes   [8 position pairs][head_dim/4 w][2] u16: dims 4w .. 4w+3
//   K scales  [8 position pairs][head_dim/32 g][2] fp16
//   V scales  the same
//
// Codes are low nibble first with zero point 7, as the weights' (quant.zig:164-177):
// value = s * (u - 7).  The orders are the ones a warp's mma.sync fragments want
// (paged_attention_q4.cu): no shuffle lies between shared memory and the tensor core.
//
// Scales are fp16 numbers of at most 7 significant bits and multiples of 2^-21, at
// most 7168.  Then s * (u - 7) / 8 is an fp16 number (3 or 4 bits times 7), and so is
// 9 * s: the attention kernel makes values from codes in one exact half-precision
// FMA.  Seven bits instead of eleven cost nothing that matters next to 4-bit codes:
// the codes are rounded against the scale that is stored.
#pragma once

#include "common.cuh"

namespace glacier {

constexpr int kQ4Page = 16;             // positions per page
constexpr int kQ4Group = 32;            // dims per scale
constexpr float kQ4MaxScale = 7168.f;   // 9 * 7168 is below fp16's largest number

__host__ __device__ constexpr size_t q4_block_bytes(size_t head_dim) { return 18 * head_dim; }

// Byte offsets inside a block.  q = dim / 4 (a quad of codes is one u16).
__host__ __device__ constexpr int q4_k_quad(int hd, int row, int q) {
  return row * (hd / 2) + (((q % 8) / 2) * (hd / kQ4Group) + q / 8) * 4 + (q & 1) * 2;
}
__host__ __device__ constexpr int q4_v_quad(int hd, int row, int q) {
  return 8 * hd + (row / 2) * hd + q * 4 + (row & 1) * 2;
}
__host__ __device__ constexpr int q4_scale(int hd, int kind, int row, int g) {
  return (16 + kind) * hd + 2 * ((row / 2) * 2 * (hd / kQ4Group) + 2 * g + (row & 1));
}

// Geometry checks that every entry over a 4-bit pool shares.
int q4_check_pool(const char* who, const void* pool, size_t num_pages, size_t num_layers, size_t layer,
                  size_t num_heads, size_t num_kv_heads, size_t head_dim);

}  // namespace glacier
