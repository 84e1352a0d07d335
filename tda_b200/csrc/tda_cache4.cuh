// Layout of the 4-bit cache, shared by the kernels that write and read it.
//
// A page holds `page` tokens of every kv head; the block of one (page, head)
// is contiguous:
//   K1 codes [page][D/2 B] | K2 codes | V codes | K1 scales [page][D/32 bf16] | K2 scales | V scales
// A code is the nibble round(7 x / amax) + 8 of a group of 32 elements along
// the head dimension, its scale bf16(amax / 7).  A zeroed block reads as zeros.
//
// The nibbles of a row are permuted so that a warp feeds matrix products
// straight from global memory: in an m16n8k16 A fragment, lane (g, t) =
// (lane / 4, lane % 4) holds rows g and g + 8 and columns 2t, 2t+1, 2t+8, 2t+9.
//   K row (A row = token, columns = dims): lane t owns the D/8 bytes at t D/8;
//     its word w covers the 4 dims 32w + 4t.. and the 4 dims 32w + 16 + 4t..,
//     nibble i + 4 e = element 2 (i % 2) + e of half i / 2 (i < 4, e < 2), so
//     (word >> 4i) & 0x000f000f is one register of the fragment.
//   V row (A row = dim, columns = tokens): lane g owns the D/16 bytes at
//     g D/16; word u = 4 dims 64u + 4g.. (nibbles 0-3) and 64u + 32 + 4g.. (4-7).
#pragma once

#include <cstddef>
#include <cstdint>

namespace tda {

constexpr int kGroup4 = 32;

__host__ __device__ constexpr size_t cache4_row_bytes(int D) { return D / 2; }
__host__ __device__ constexpr size_t cache4_scale_bytes(int D) { return D / kGroup4 * 2; }
__host__ __device__ constexpr size_t cache4_block_bytes(int page, int D) {
  return 3 * static_cast<size_t>(page) * (cache4_row_bytes(D) + cache4_scale_bytes(D));
}
// byte offset of tensor x's (0 K1, 1 K2, 2 V) codes / scales in a block
__host__ __device__ constexpr size_t cache4_codes_at(int x, int page, int D) { return x * page * cache4_row_bytes(D); }
__host__ __device__ constexpr size_t cache4_scales_at(int x, int page, int D) {
  return page * (3 * cache4_row_bytes(D) + x * cache4_scale_bytes(D));
}

}  // namespace tda
