// Device code shared by the tensor-core kernels of softmax differential
// attention: tile geometry, product issue, row masks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tda_internal.h"
#include "tda_ptx.cuh"
#include "tda_sdiff.h"
#include "tda_transform.cuh"

namespace tda {
namespace sd {

using tc::drain_wait;
using tc::f2u;
using tc::max3f;

constexpr int kSmemBudget = 232448;

// A [128 rows][D] operand tile: D / 64 boxes of 128 rows x 128 B, 128-byte swizzle.
template <int D, bool F16>
struct Geo {
  static constexpr int kBoxes = D / 64;
  static constexpr int kBoxBytes = kTile * 128;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr uint32_t kIdescScore = idesc_f16(128, 128, !F16, false);
  static constexpr uint32_t kIdescMn = idesc_f16(128, D, !F16, true);
};

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// D[dcol] = A B^T over D: A and B K-major tiles in shared memory
template <int D, bool F16>
__device__ __forceinline__ void mma_score(uint32_t dcol, uint32_t a, uint32_t b) {
  using G = Geo<D, F16>;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = (kk >> 2) * G::kBoxBytes + (kk & 3) * 32;
    mma_ss(dcol, smem_desc_sw128(a + off, 16, 1024), smem_desc_sw128(b + off, 16, 1024), G::kIdescScore, kk > 0 ? 1u : 0u);
  }
}

// D[dcol] (+)= W X: W [128][128] 16-bit in TMEM, X an MN-major tile of 128 rows.  W fills 64
// columns, or (HALVES) 32 at wcol and 32 at wcol + 64: each half over the scores it came
// from, so that the two warps that share a row's scores need not wait for one another.
template <int D, bool F16, bool HALVES = false>
__device__ __forceinline__ void mma_weights(uint32_t dcol, uint32_t wcol, uint32_t x, bool accumulate) {
  using G = Geo<D, F16>;
#pragma unroll
  for (int m = 0; m < kTile / 16; ++m)
    mma_ts(dcol, wcol + (HALVES ? 64 * (m >> 2) + 8 * (m & 3) : 8 * m), smem_desc_sw128(x + m * 2048, G::kBoxBytes, 1024), G::kIdescMn, (accumulate || m > 0) ? 1u : 0u);
}

template <int D, bool F16>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int h, int b) {
  using G = Geo<D, F16>;
#pragma unroll
  for (int x = 0; x < G::kBoxes; ++x) tma_load_4d(dst + x * G::kBoxBytes, map, bar, x * 64, row, h, b);
}

// Row r of a tile set to zero: what lies past a sequence's length may be NaN,
// and a weight of 0 does not hide that from a product.
template <int D>
__device__ __forceinline__ void zero_row(uint8_t* tile, int r) {
#pragma unroll
  for (int x = 0; x < D / 64; ++x)
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + x * (kTile * 128) + r * 128 + 16 * c) = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ int keys_of(const SdParams& p, int b) {
  return p.key_lengths ? max(0, min(p.key_lengths[b], p.Sk)) : p.Sk;
}

// stores 32 fp32 columns [col, col + 32) of row r into 128-byte-swizzled boxes of 32 columns
__device__ __forceinline__ void stage_f32(uint8_t* boxes, int r, int col, const float (&x)[32]) {
  uint8_t* row = boxes + (col >> 5) * (kTile * 128) + r * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(row + ((c ^ (r & 7)) << 4)) = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
}
// the same as 16-bit values in boxes of 64 columns
template <bool F16>
__device__ __forceinline__ void stage_16(uint8_t* boxes, int r, int col, const float (&x)[32]) {
  uint8_t* row = boxes + (col >> 6) * (kTile * 128) + r * 128;
  const int c0 = (col & 63) >> 3;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2<F16>(x[8 * c + 2 * i], x[8 * c + 2 * i + 1]);
    *reinterpret_cast<uint4*>(row + (((c0 + c) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace sd

// Tensor maps of the kernels: inputs as 4-D {D, S, heads, batches} with boxes
// of 64 columns x 128 rows, contiguous outputs as 3-D {D, S, batch * head}.
struct SdMaps {
  CUtensorMap q[2], k[2], v, dout;
  CUtensorMap out;   // 16-bit, boxes of 64 x 128
  CUtensorMap o12;   // fp32, {D, Sq, 2 B H}, boxes of 32 x 128
  CUtensorMap dq[2], dk[2], dv;
};

struct SdTcParams {
  SdMaps m;
  SdParams p;
  int* status;
  unsigned long long timeout_ns;
  int n_qt, n_kt;
};

}  // namespace tda
