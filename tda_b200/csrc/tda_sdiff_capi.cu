// C entry points of softmax differential attention: argument checks and the
// choice between the tensor-core and the CUDA-core kernels.
#include <cmath>
#include <cstring>

#include <cudaTypedefs.h>

#include <mutex>

#include "tda_sdiff_tc.cuh"

using namespace tda;

namespace tda {
cudaError_t launch_sdiff_tc_fwd(const SdTcParams& tp, int dtype, int D, cudaStream_t s);
cudaError_t launch_sdiff_tc_bwd(const SdTcParams& tp, int dtype, int D, cudaStream_t s);
}

namespace {

// bf16 and fp16 at these head dims fit the tensor-core kernels' tiles; fp32 needs
// its own arithmetic and other head dims do not fill a 128-byte box
bool on_tensor_cores(int dtype, int64_t D) { return dtype != TDA_F32 && (D == 64 || D == 128); }

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
  const int rows = on_tensor_cores(dtype, D) ? 128 : simt_tile_rows(static_cast<int>(D));
  p.q_together = heads_together(causal != 0, static_cast<int>(B * H), ceil_div(Sq, rows), p.group);
  p.k_together = heads_together(causal != 0, static_cast<int>(B * Hkv), ceil_div(Sk, rows), 1);
  p.Sq = static_cast<int>(Sq);
  p.Sk = static_cast<int>(Sk);
  p.causal = causal != 0;
  p.scale = scale;
  p.c = scale * 1.4426950408889634f;
  return TDA_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// {D, S, heads, batches} with boxes of 128 bytes x 128 rows, 128-byte swizzle, zeros out of bounds
int map4(CUtensorMap* m, int dtype, const SdView& x, int64_t B, int64_t H, int64_t S, int64_t D) {
  auto enc = encoder();
  if (!enc) return fail(TDA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const int es = dtype == TDA_F32 ? 4 : 2;
  const CUtensorMapDataType dt = dtype == TDA_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == TDA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(B)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(x.ss) * es, static_cast<cuuint64_t>(x.sh) * es, static_cast<cuuint64_t>(x.sb) * es};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / es), static_cast<cuuint32_t>(kTile), 1, 1};
  cuuint32_t one[4] = {1, 1, 1, 1};
  CUresult r = enc(m, dt, 4, const_cast<void*>(x.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TDA_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
  return TDA_OK;
}

// a contiguous (n, S, D) output as {D, S, n}, same boxes
int map3(CUtensorMap* m, int dtype, const void* x, int64_t n, int64_t S, int64_t D) {
  auto enc = encoder();
  if (!enc) return fail(TDA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const int es = dtype == TDA_F32 ? 4 : 2;
  const CUtensorMapDataType dt = dtype == TDA_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == TDA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(n)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D * es), static_cast<cuuint64_t>(S * D * es)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / es), static_cast<cuuint32_t>(kTile), 1};
  cuuint32_t one[3] = {1, 1, 1};
  CUresult r = enc(m, dt, 3, const_cast<void*>(x), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TDA_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
  return TDA_OK;
}

int input_maps(SdTcParams& tp, int dtype, int64_t D) {
  const SdParams& p = tp.p;
  for (int i = 0; i < 2; ++i) {
    if (int e = map4(&tp.m.q[i], dtype, p.q[i], p.B, p.H, p.Sq, D)) return e;
    if (int e = map4(&tp.m.k[i], dtype, p.k[i], p.B, p.Hkv, p.Sk, D)) return e;
  }
  if (int e = map4(&tp.m.v, dtype, p.v, p.B, p.Hkv, p.Sk, D)) return e;
  tp.n_qt = static_cast<int>(ceil_div(p.Sq, kTile));
  tp.n_kt = static_cast<int>(ceil_div(p.Sk, kTile));
  tp.timeout_ns = wait_timeout_ns();
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (on_tensor_cores(dtype, head_dim)) {
    SdTcParams tp;
    std::memset(&tp, 0, sizeof(tp));
    tp.p = p;
    tp.status = status;
    if (int r = input_maps(tp, dtype, head_dim)) return r;
    if (int r = map3(&tp.m.out, dtype, out, batch * heads, q_len, head_dim)) return r;
    if (o12)
      if (int r = map3(&tp.m.o12, TDA_F32, o12, 2 * batch * heads, q_len, head_dim)) return r;
    e = launch_sdiff_tc_fwd(tp, dtype, static_cast<int>(head_dim), s);
  } else {
    e = launch_sdiff_simt_fwd(p, dtype, static_cast<int>(head_dim), s);
  }
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "softmax differential forward launch");
}

size_t tda_sdiff_bwd_workspace_size(int64_t batch, int64_t heads, int64_t q_len) {
  if (batch < 1 || heads < 1 || q_len < 1) return 0;
  // per map, head and padded row: two floats and two rows of 16 16-bit values
  return 2 * static_cast<size_t>(batch) * heads * padded_seq(q_len) * (2 * sizeof(float) + 64);
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
  p.table = static_cast<float*>(workspace);
  p.pad = static_cast<int>(padded_seq(q_len));
  if (on_tensor_cores(dtype, head_dim)) p.aux = p.table + 4 * batch * heads * padded_seq(q_len);
  p.dq[0] = dq1;
  p.dq[1] = dq2;
  p.dk[0] = dk1;
  p.dk[1] = dk2;
  p.dv = dv;
  p.dlam = dlam;
  const int D = static_cast<int>(head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_sdiff_delta(p, dtype, D, s);
  if (e == cudaSuccess && on_tensor_cores(dtype, head_dim)) {
    SdTcParams tp;
    std::memset(&tp, 0, sizeof(tp));
    tp.p = p;
    tp.status = status;
    if (int r = input_maps(tp, dtype, head_dim)) return r;
    if (int r = map4(&tp.m.dout, dtype, p.dout, batch, heads, q_len, head_dim)) return r;
    for (int i = 0; i < 2; ++i) {
      if (int r = map3(&tp.m.dq[i], dtype, p.dq[i], batch * heads, q_len, head_dim)) return r;
      if (int r = map3(&tp.m.dk[i], dtype, p.dk[i], batch * kv_heads, k_len, head_dim)) return r;
    }
    if (int r = map3(&tp.m.dv, dtype, dv, batch * kv_heads, k_len, head_dim)) return r;
    e = launch_sdiff_tc_bwd(tp, dtype, D, s);
  } else if (e == cudaSuccess) {
    e = launch_sdiff_simt_bwd(p, dtype, D, s);
  }
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "softmax differential backward launch");
}

}  // extern "C"
