// Layout of the 4-bit cache, shared by the kernels that write and read it.
//
// A page holds `page` tokens of every kv head; the block of one (page, head) is
// page / 16 slabs of 16 tokens, each contiguous, so that one bulk copy brings a
// slab into shared memory:
//   K1 codes [16][D/2 B] | K2 codes | V codes | K1 scales [16][D/32 bf16] | K2 scales | V scales
// A code is the nibble round(7 x / amax) + 8 of a group of 32 elements along
// the head dimension, its scale bf16(amax / 7).  A zeroed block reads as zeros.
//
// Nibbles are permuted so that a warp feeds matrix products straight from
// 16-byte shared-memory loads at lane * 16: in an m16n8k16 A fragment, lane
// (g, t) = (lane / 4, lane % 4) holds rows g and g + 8 and columns 2t, 2t+1,
// 2t+8, 2t+9.  Of a word w, w & 0x000f000f gives two nibbles as they are and
// w & 0x00f000f0 two more times 16 (nibbles i and i + 4 share a register).
//   K (A row = token, columns = dims): row r is D/2 bytes, lane t owns the D/8
//     at t D/8; word w covers dims 32w + 4t.. and 32w + 16 + 4t.., nibble
//     2 h + i / 2 + 4 (i % 2) = element i of half h.
//   V (A row = dim, columns = tokens): lane (g, t) owns 4 tokens (2t, 2t+1,
//     2t+8, 2t+9) of dims 64u + 4g.. (nibbles 0-3 of word u) and 64u + 32 +
//     4g.. (nibbles 4-7): 16 bytes hold the words of 2 tokens at D = 128 and of
//     all 4 at D = 64.
#pragma once

#include <cstddef>
#include <cstdint>

namespace tda {

constexpr int kGroup4 = 32;
constexpr int kSlab4 = 16;

__host__ __device__ constexpr int cache4_row_bytes(int D) { return D / 2; }
__host__ __device__ constexpr int cache4_scale_bytes(int D) { return D / kGroup4 * 2; }
__host__ __device__ constexpr int cache4_slab_bytes(int D) { return 3 * kSlab4 * (cache4_row_bytes(D) + cache4_scale_bytes(D)); }
__host__ __device__ constexpr size_t cache4_block_bytes(int page, int D) {
  return static_cast<size_t>(page / kSlab4) * cache4_slab_bytes(D);
}
// byte offset in a slab of tensor x's (0 K1, 1 K2, 2 V) codes / scales
__host__ __device__ constexpr int cache4_codes_at(int x, int D) { return x * kSlab4 * cache4_row_bytes(D); }
__host__ __device__ constexpr int cache4_scales_at(int x, int D) {
  return 3 * kSlab4 * cache4_row_bytes(D) + x * kSlab4 * cache4_scale_bytes(D);
}
// byte offset of K word w of lane t in token row r / of V word u of lane g
__host__ __device__ constexpr int cache4_k_word(int r, int t, int w, int D) { return r * (D / 2) + t * (D / 8) + 4 * w; }
__host__ __device__ constexpr int cache4_v_word(int r, int g, int u, int D) {
  const int t = (r & 7) >> 1, i = (r & 1) + 2 * (r >> 3);
  return D == 128 ? (i >> 1) * 512 + (4 * g + t) * 16 + (i & 1) * 8 + u * 4 : (4 * g + t) * 16 + i * 4;
}

}  // namespace tda
