// Softmax differential attention: parameters shared by its kernels.
//
//   P_m = softmax(scale q_m k_m^T) over the keys row i sees: j < key_lengths[b]
//         and, when causal, j <= i + Sk - Sq;  a row that sees none gives zeros
//   out = P_1 v - lambda P_2 v
//   L_m(i) = log2 of the row's sum of 2^(scale log2(e) s_ij): P_ij = 2^(c s_ij - L_m(i));
//            +infinity where the row sees no key
// Backward, with O_m = P_m v, dP = dout v^T, D_m = rowsum(dout O_m):
//   dS_1 = P_1 (dP - D_1), dS_2 = -lambda P_2 (dP - D_2)
//   dq_m = scale dS_m k_m, dk_m = scale dS_m^T q_m, dv = (P_1 - lambda P_2)^T dout
//   dlambda = -sum_i D_2(i)
// With a single key the weight is 1 whatever its score: dS is exactly zero, and
// set so, since dP and D are sums in different orders.
// Shared heads: query head h reads kv head h / (H / Hkv); dk and dv sum over the group.
#pragma once

#include "tda_host.h"

namespace tda {

constexpr int kAuxTileBytes = 128 * 16 * 2;
// fp16 holds -L / c up to 2^24 as a multiple of this
constexpr float aux_unit(bool f16) { return f16 ? 256.0f : 1.0f; }

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
  // backward
  SdView dout;
  float* table;    // [2][B][H][pad / 128][2][128]: -L_m, then -D_m of each row; -inf, 0 past Sq
  // The same numbers as products read them (16-bit types): per tile of 128 rows
  // [128][16] for -L / c, then for -D, three values a row that add up to it over
  // aux_unit, in core-matrix order.
  void* aux;
  int pad;         // Sq rounded up to a tile of 128
  void* dq[2];     // contiguous, of the inputs' type
  void* dk[2];
  void* dv;
  float* dlam;     // [B][H], or null
};

cudaError_t launch_sdiff_simt_fwd(const SdParams& p, int dtype, int D, cudaStream_t s);
cudaError_t launch_sdiff_simt_bwd(const SdParams& p, int dtype, int D, cudaStream_t s);
// D_1, D_2 from dout and o12, and dlambda where asked for
cudaError_t launch_sdiff_delta(const SdParams& p, int dtype, int D, cudaStream_t s);

}  // namespace tda
