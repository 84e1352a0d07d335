// Device code shared by the tensor-core kernels of softmax differential
// attention: tile geometry, product issue, row masks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tda_internal.h"
#include "tda_ptx.cuh"
#include "tda_sdiff.h"
#include "tda_transform.cuh"
#include "tda_wait.cuh"

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

// The issuing warp stays converged: every lane runs the waits and the address
// arithmetic, so that descriptors and TMEM addresses live in uniform registers,
// and one elected lane (the same every time) issues.  With a branch on the lane
// index instead, each product's operands are moved there one by one, about 60-100
// cycles a product against 64 of tensor work.
__device__ __forceinline__ bool elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (elected()) tc_commit(bar);
  __syncwarp();
}

// Operand descriptors differ in their address field alone (bytes / 16, and all of
// shared memory fits the field): one 32-bit addition an operand keeps the single
// issuing thread ahead of the tensor cores.
__device__ __forceinline__ uint64_t desc_at(uint32_t lo, uint32_t hi, uint32_t bytes) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo + (bytes >> 4)), "r"(hi));
  return d;
}

// D[dcol] = A B^T over D: A and B K-major tiles in shared memory
template <int D, bool F16>
__device__ __forceinline__ void mma_score(uint32_t dcol, uint32_t a, uint32_t b) {
  using G = Geo<D, F16>;
  const uint64_t da = smem_desc_sw128(a, 16, 1024), db = smem_desc_sw128(b, 16, 1024);
  const uint32_t hi = static_cast<uint32_t>(da >> 32), la = static_cast<uint32_t>(da), lb = static_cast<uint32_t>(db);
  if (elected()) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t off = (kk >> 2) * G::kBoxBytes + (kk & 3) * 32;
      mma_ss(dcol, desc_at(la, hi, off), desc_at(lb, hi, off), G::kIdescScore, kk > 0 ? 1u : 0u);
    }
  }
  __syncwarp();
}

// D[dcol] (+)= W X: W [128][128] 16-bit in TMEM, X an MN-major tile of 128 rows.  W fills 64
// columns, or (QUARTERS) 16 of each 32: each quarter over the scores it came from, so that
// the four warps that share a row's scores need not wait for one another.
// Rows [16 M0, 16 M1) of X alone: a part of the product, once a part of W is there.
template <int D, bool F16, bool QUARTERS = false, int M0 = 0, int M1 = kTile / 16>
__device__ __forceinline__ void mma_weights(uint32_t dcol, uint32_t wcol, uint32_t x, bool accumulate) {
  using G = Geo<D, F16>;
  const uint64_t dx = smem_desc_sw128(x, G::kBoxBytes, 1024);
  const uint32_t hi = static_cast<uint32_t>(dx >> 32), lo = static_cast<uint32_t>(dx);
  if (elected()) {
#pragma unroll
    for (int m = M0; m < M1; ++m)
      mma_ts(dcol, wcol + (QUARTERS ? 32 * (m >> 1) + 8 * (m & 1) : 8 * m), desc_at(lo, hi, m * 2048), G::kIdescMn,
             (accumulate || m > 0) ? 1u : 0u);
  }
  __syncwarp();
}

// One more step of 16 along the contracted dimension: D[dcol] += ones aux^T, with
// `aux` a [128][16] table in shared memory (unswizzled: 8 x 16-byte core matrices,
// 128 bytes apart along the columns, 256 along the rows) whose columns times their
// units add up to a number a row, and `ones` the units, of the same form.  It subtracts L or D of
// the query from a column of scores without a load in the threads that use them:
// 16 shared-memory loads a thread and step cost more than the product.
template <bool F16>
__device__ __forceinline__ void mma_offsets(uint32_t dcol, uint32_t ones, uint32_t aux) {
  constexpr uint64_t kForm = (static_cast<uint64_t>(128 >> 4) << 16) | (static_cast<uint64_t>(256 >> 4) << 32) | (1ull << 46);
  if (elected())
    mma_ss(dcol, kForm | ((ones >> 4) & 0x3FFFu), kForm | ((aux >> 4) & 0x3FFFu), idesc_f16(128, 128, !F16, false), 1u);
  __syncwarp();
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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where an operand is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair for -125 <= x <= 126 on the FMA pipe (below: 2^-125): 2^n by the
// exponent field, 2^f, |f| <= 1/2, by the polynomial of least relative error,
// 7.5e-5 (degree 3, bf16 weights) or 2.6e-6 (degree 4, fp16 weights).  Of a NaN it
// gives the largest finite number: r and p are then the NaN 0x7fffffff, the only
// one that fp32 arithmetic makes, and their bits add up to 0x7f7fffff.  With
// KEEP_NAN a multiplication by 2^n takes the addition's place, the same bits for
// numbers, and a NaN stays one.
template <bool F16, bool KEEP_NAN = false>
__device__ __forceinline__ float2 poly_ex2(float2 x) {
  x.x = max_nan(x.x, -125.0f);
  x.y = max_nan(x.y, -125.0f);
  const float2 r = __fadd2_rn(x, make_float2(12582912.0f, 12582912.0f));  // 1.5 2^23: the last bits are n
  const float2 n = __fadd2_rn(r, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
  float2 p;
  if constexpr (F16) {
    p = __ffma2_rn(f, make_float2(0.009570102207362652f, 0.009570102207362652f), make_float2(0.05591786280274391f, 0.05591786280274391f));
    p = __ffma2_rn(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
    p = __ffma2_rn(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
    p = __ffma2_rn(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  } else {
    p = __ffma2_rn(f, make_float2(0.0551716685295105f, 0.0551716685295105f), make_float2(0.2426111251115799f, 0.2426111251115799f));
    p = __ffma2_rn(p, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
    p = __ffma2_rn(p, f, make_float2(0.9999280571937561f, 0.9999280571937561f));
  }
  if constexpr (KEEP_NAN)
    return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(r.x) << 23) + 0x3f800000u),
                                     __uint_as_float((__float_as_uint(r.y) << 23) + 0x3f800000u)));
  return make_float2(__uint_as_float((__float_as_uint(r.x) << 23) + __float_as_uint(p.x)),
                     __uint_as_float((__float_as_uint(r.y) << 23) + __float_as_uint(p.y)));
}

template <int kRegs>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
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
