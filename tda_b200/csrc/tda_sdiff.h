// Softmax differential attention: parameters shared by its kernels.
//
//   P_m = softmax(scale q_m k_m^T) over the keys row i sees: j < key_lengths[b]
//         and, when causal, j <= i + Sk - Sq;  a row that sees none gives zeros
//   out = P_1 v - lambda P_2 v
//   L_m(i) = log2 of the row's sum of 2^(scale log2(e) s_ij): P_ij = 2^(c s_ij - L_m(i));
//            +infinity where the row sees no key; NaN where its keys have no softmax
//            (a NaN or +infinity among the scores, or -infinity alone)
// Backward, with O_m = P_m v, dP = dout v^T, D_m = rowsum(dout O_m):
//   dS_1 = P_1 (dP - D_1), dS_2 = -lambda P_2 (dP - D_2)
//   dq_m = scale dS_m k_m, dk_m = scale dS_m^T q_m, dv = (P_1 - lambda P_2)^T dout
//   dlambda = -sum_i D_2(i)
// With a single key the weight is 1 whatever its score: dS is exactly zero, and
// set so where it is a number, since dP and D are sums in different orders.
// Shared heads: query head h reads kv head h / (H / Hkv); dk and dv sum over the group.
#pragma once

#include "tda_host.h"

namespace tda {

constexpr int kAuxTileBytes = 128 * 16 * 2;
// The units of the product tables' columns, three columns a unit.  bf16 has the
// exponents of fp32 and needs one.  fp16 holds numbers from 1 to 65504 to 33 bits in three
// values, and D is as small as the gradient that comes in: a number takes the columns
// of the largest unit that it is not below (the last one below 2^-14 too, to 2^-38).
constexpr int aux_units(bool f16) { return f16 ? 3 : 1; }
constexpr float aux_unit(bool f16, int g) { return !f16 || g == 1 ? 1.0f : g == 0 ? 0x1p15f : 0x1p-14f; }

struct SdView {  // (batch, head, seq, dim) view: element strides, dim contiguous
  const void* p;
  long long sb, sh, ss;
};

struct SdParams {
  SdView q[2], k[2], v;
  void* out;       // contiguous (B, H, Sq, D), of the inputs' type
  // Kept for the backward, or null: O_1 and O_2 in fp32 [2][B][H][Sq][D], since
  // D_m is subtracted from a dP it nearly equals where one weight is near 1
  // (rounded to bf16 they cost 2^-8 of dq there), and L_1, L_2 [2][B][H][Sq].
  float* o12;
  float* lse;
  const int* key_lengths;
  LambdaRef lam;
  int B, H, Hkv, group, Sq, Sk, causal;
  float scale;     // of the scores
  float c;         // scale log2(e)
  int q_together, k_together;  // heads side by side (heads_together) by query tiles, kv heads by key tiles
  // backward
  SdView dout;
  float* table;    // [2][B][H][pad / 128][2][128]: -L_m, then -D_m of each row; -inf, 0 past Sq
  // The same numbers as products read them (16-bit types): per tile of 128 rows
  // [128][16] for -L / c, then for -D, three values a row that add up to it over
  // their columns' aux_unit and zeros, in core-matrix order.
  void* aux;
  int pad;         // Sq rounded up to a tile of 128
  void* dq[2];     // contiguous, of the inputs' type
  void* dk[2];
  void* dv;
  float* dlam;     // [B][H], or null
};

#ifdef __CUDACC__
// fp16: the largest finite |dout| of a kv head's query heads and the largest finite
// |v| of its keys, two words that hold an fp16 number each.  They lie in the last
// four columns of the first row of the head's D tables, whose unit is zero.
__device__ __forceinline__ uint32_t* sizes_of(const SdParams& p, int b, int kvh) {
  const long long tile = (static_cast<long long>(b) * p.H + kvh * p.group) * (p.pad / kTile);
  return reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.aux) + (tile * 2 + 1) * kAuxTileBytes + 128 + 8);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// The e with x <= 2^e for 0 <= x, within +-60
__device__ __forceinline__ int exponent_above(float x) {
  return min(max(static_cast<int>(__float_as_uint(x) >> 23) - 126, -60), 60);
}
// fp16: dS enters its products times 2^e.  |dP - D| <= 2 |dout| |v| <= 2 head_dim max|dout|
// max|v|, so with this e no dS passes 2^15, and one 2^29 below the largest possible is
// still a normal number: gradients of any size keep their bits.
__device__ __forceinline__ int ds_exponent(const SdParams& p, int b, int kvh, int D, float largest_weight) {
  const uint32_t* s = sizes_of(p, b, kvh);
  float g, v;
  asm("cvt.f32.f16 %0, %1;" : "=f"(g) : "h"(static_cast<unsigned short>(s[0])));
  asm("cvt.f32.f16 %0, %1;" : "=f"(v) : "h"(static_cast<unsigned short>(s[1])));
  return min(15 - exponent_above(2.0f * D * g * v * largest_weight), 60);
}
#endif

cudaError_t launch_sdiff_simt_fwd(const SdParams& p, int dtype, int D, cudaStream_t s);
cudaError_t launch_sdiff_simt_bwd(const SdParams& p, int dtype, int D, cudaStream_t s);
// D_1, D_2 from dout and o12, and dlambda where asked for
cudaError_t launch_sdiff_delta(const SdParams& p, int dtype, int D, cudaStream_t s);

// rows of a tile of the CUDA-core kernels
constexpr int simt_tile_rows(int D) { return D <= 128 ? 64 : 32; }

// How many of `heads` heads (a divisor) run side by side, each tile of all of them
// before the next tile.  A causal call's tiles differ in length: taken head by
// head, the last head's longest one starts when the other SMs are nearly done.
// Measured on B200 against that order: dkv at (4, 32 on 8, 4096, 128) 1990 -> 1820
// us, a backward of (1, 8, 8192, 128) 960 -> 805, a fp32 step of (2, 16 on 8, 1024,
// 64) 2010 -> 1670; the same bits.  So heads go together until they make 512 tiles,
// a few for each SM, and no further, so that long sequences keep few heads' keys
// in L2; heads that share keys (`side`) stay together.  Uncausal tiles are equal:
// side by side they only lose L2 hits (a ragged fp16 backward of (6, 16, 1999, 64) 705 -> 728 us).
inline int heads_together(bool causal, int heads, long long tiles, int side) {
  if (!causal) return side;
  for (int n = side; n < heads && n <= 2048; n += side)
    if (heads % n == 0 && n * tiles >= 512) return n;
  return heads;
}

// tile (in the caller's order, longest first) and head of a block
__device__ __forceinline__ void tile_of_block(int block, int tiles, int together, int& head, int& tile) {
  const int per = together * tiles, g = block / per, r = block % per;
  tile = r / together;
  head = g * together + r % together;
}

}  // namespace tda
