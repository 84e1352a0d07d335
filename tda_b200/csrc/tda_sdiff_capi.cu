// C entry points of softmax differential attention: argument checks and the
// choice between the tensor-core and the CUDA-core kernels.
#include <cmath>
#include <cstring>

#include "tda_sdiff.h"

using namespace tda;

namespace {

int fill(SdParams& p, const void* q1, const void* q2, const void* k1, const void* k2, const void* v,
         const int64_t* strides, int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
         float scale, int causal, const int32_t* key_lengths, const void* lambda, int lambda_dtype, int64_t lsb,
         int64_t lsh, float lambda_value) {
  if (dtype != TDA_F32 && dtype != TDA_BF16 && dtype != TDA_F16)
    return fail(TDA_ERR_INVALID, "dtype must be TDA_F32, TDA_BF16 or TDA_F16");
  if (B < 1 || H < 1 || Sq < 1 || Sk < 1) return fail(TDA_ERR_INVALID, "batch, heads and lengths must be >= 1");
  if (Hkv < 1 || H % Hkv != 0) return fail(TDA_ERR_INVALID, "kv heads (%lld) must divide the query heads (%lld)",
                                           static_cast<long long>(Hkv), static_cast<long long>(H));
  if (D < 16 || D > 256 || (D & (D - 1)) != 0)
    return fail(TDA_ERR_INVALID, "head_dim must be a power of two in [16, 256] (got %lld)", static_cast<long long>(D));
  if (Sq > (1ll << 30) || Sk > (1ll << 30)) return fail(TDA_ERR_INVALID, "sequence too long");
  if (B > 0x7fffffffll / H || B * H > 0x7fffffffll / ceil_div(Sq > Sk ? Sq : Sk, 32))
    return fail(TDA_ERR_INVALID, "batch * heads * tiles exceed the grid limit");
  if (!(std::isfinite(scale) && scale > 0.f)) return fail(TDA_ERR_INVALID, "scale must be finite and positive");
  if (key_lengths && !aligned(key_lengths, 4)) return fail(TDA_ERR_INVALID, "key_lengths must be int32");
  const void* in[5] = {q1, q2, k1, k2, v};
  SdView* out[5] = {&p.q[0], &p.q[1], &p.k[0], &p.k[1], &p.v};
  for (int i = 0; i < 5; ++i) {
    if (!in[i] || !aligned(in[i], 16)) return fail(TDA_ERR_INVALID, "inputs must be non-NULL and 16-byte aligned");
    const int64_t h = i < 2 ? H : Hkv, s = i < 2 ? Sq : Sk;
    *out[i] = strides ? SdView{in[i], strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}
                      : SdView{in[i], h * s * D, s * D, D};
    if (out[i]->sb <= 0 || out[i]->sh <= 0 || out[i]->ss <= 0 || (out[i]->sb | out[i]->sh | out[i]->ss) % 8 != 0)
      return fail(TDA_ERR_INVALID, "input strides must be positive multiples of 8 elements");
  }
  p.key_lengths = key_lengths;
  p.lam = LambdaRef{lambda, lambda_dtype, lsb, lsh, lambda_value};
  if (int e = check_lambda(p.lam)) return e;
  p.B = static_cast<int>(B);
  p.H = static_cast<int>(H);
  p.Hkv = static_cast<int>(Hkv);
  p.group = static_cast<int>(H / Hkv);
  p.Sq = static_cast<int>(Sq);
  p.Sk = static_cast<int>(Sk);
  p.causal = causal != 0;
  p.scale = scale;
  p.c = scale * 1.4426950408889634f;
  return TDA_OK;
}

}  // namespace

extern "C" {

int tda_sdiff_fwd(const void* q1, const void* q2, const void* k1, const void* k2, const void* v,
                  const int64_t* strides, void* out, float* o12, float* lse, int dtype, int64_t batch, int64_t heads,
                  int64_t kv_heads, int64_t q_len, int64_t k_len, int64_t head_dim, float scale, int causal,
                  const int32_t* key_lengths, const void* lambda, int lambda_dtype, int64_t lambda_stride_b,
                  int64_t lambda_stride_h, float lambda_value, int* status, void* stream) {
  SdParams p;
  std::memset(&p, 0, sizeof(p));
  if (int e = fill(p, q1, q2, k1, k2, v, strides, dtype, batch, heads, kv_heads, q_len, k_len, head_dim, scale, causal,
                   key_lengths, lambda, lambda_dtype, lambda_stride_b, lambda_stride_h, lambda_value))
    return e;
  if (!out || !aligned(out, 16)) return fail(TDA_ERR_INVALID, "out must be non-NULL and 16-byte aligned");
  if (!o12 != !lse || !aligned(o12, 16) || !aligned(lse, 4))
    return fail(TDA_ERR_INVALID, "o12 (16-byte aligned) and lse come together or not at all");
  if (!status) return fail(TDA_ERR_INVALID, "status must point to a device int32");
  p.out = out;
  p.o12 = o12;
  p.lse = lse;
  cudaError_t e = launch_sdiff_simt_fwd(p, dtype, static_cast<int>(head_dim), static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "softmax differential forward launch");
}

size_t tda_sdiff_bwd_workspace_size(int64_t batch, int64_t heads, int64_t q_len) {
  if (batch < 1 || heads < 1 || q_len < 1) return 0;
  return 2 * static_cast<size_t>(batch) * heads * q_len * sizeof(float);
}

int tda_sdiff_bwd(const void* q1, const void* q2, const void* k1, const void* k2, const void* v,
                  const int64_t* strides, const void* dout, const int64_t* dout_strides,
                  const float* o12, const float* lse, void* dq1, void* dq2, void* dk1, void* dk2, void* dv, float* dlam,
                  int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len, int64_t k_len,
                  int64_t head_dim, float scale, int causal, const int32_t* key_lengths, const void* lambda,
                  int lambda_dtype, int64_t lambda_stride_b, int64_t lambda_stride_h, float lambda_value,
                  void* workspace, size_t workspace_bytes, int* status, void* stream) {
  SdParams p;
  std::memset(&p, 0, sizeof(p));
  if (int e = fill(p, q1, q2, k1, k2, v, strides, dtype, batch, heads, kv_heads, q_len, k_len, head_dim, scale, causal,
                   key_lengths, lambda, lambda_dtype, lambda_stride_b, lambda_stride_h, lambda_value))
    return e;
  const void* need[] = {dout, o12, dq1, dq2, dk1, dk2, dv};
  for (const void* x : need)
    if (!x || !aligned(x, 16)) return fail(TDA_ERR_INVALID, "dout, o12 and the gradients must be non-NULL and 16-byte aligned");
  if (!lse || !aligned(lse, 4)) return fail(TDA_ERR_INVALID, "lse must be a non-NULL fp32 array");
  if (!status) return fail(TDA_ERR_INVALID, "status must point to a device int32");
  p.dout = dout_strides ? SdView{dout, dout_strides[0], dout_strides[1], dout_strides[2]}
                        : SdView{dout, heads * q_len * head_dim, q_len * head_dim, head_dim};
  if (p.dout.sb <= 0 || p.dout.sh <= 0 || p.dout.ss <= 0 || (p.dout.sb | p.dout.sh | p.dout.ss) % 8 != 0)
    return fail(TDA_ERR_INVALID, "dout strides must be positive multiples of 8 elements");
  const size_t bytes = tda_sdiff_bwd_workspace_size(batch, heads, q_len);
  if (!workspace || workspace_bytes < bytes || !aligned(workspace, 16))
    return fail(TDA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed", bytes);
  p.o12 = const_cast<float*>(o12);
  p.lse = const_cast<float*>(lse);
  p.delta = static_cast<float*>(workspace);
  p.dq[0] = dq1;
  p.dq[1] = dq2;
  p.dk[0] = dk1;
  p.dk[1] = dk2;
  p.dv = dv;
  p.dlam = dlam;
  const int D = static_cast<int>(head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_sdiff_delta(p, dtype, D, s);
  if (e == cudaSuccess) e = launch_sdiff_simt_bwd(p, dtype, D, s);
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "softmax differential backward launch");
}

}  // extern "C"
