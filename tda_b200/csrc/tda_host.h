// Host-side helpers of the C-ABI translation units: error text, argument
// checks and the wait settings shared by every entry point.
#pragma once

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

#include "../../include/tda_b200.h"
#include "tda_internal.h"

namespace tda {

// Records the message tda_last_error() returns and passes `code` through.
__attribute__((format(printf, 2, 3))) inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

inline int cuda_fail(cudaError_t e, const char* what) {
  return fail(TDA_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Lets a kernel use `bytes` of dynamic shared memory, once a device.
template <auto kKernel>
cudaError_t allow_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  done.fetch_or(bit, std::memory_order_relaxed);
  return cudaSuccess;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// lambda of the softmax differential forms and of the cache operators: one
// value a (batch, head), read on the device in its own type, or a host scalar
// (ptr == nullptr).
struct LambdaRef {
  const void* ptr;
  int dtype;  // TDA_F32, TDA_BF16 or TDA_F16
  long long sb;
  long long sh;
  float scalar;
};

#ifdef __CUDACC__
__device__ __forceinline__ float lambda_at(const LambdaRef& l, int b, int h) {
  if (l.ptr == nullptr) return l.scalar;
  const long long i = b * l.sb + h * l.sh;
  if (l.dtype == TDA_F32) return static_cast<const float*>(l.ptr)[i];
  const unsigned short u = static_cast<const unsigned short*>(l.ptr)[i];
  if (l.dtype == TDA_BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  float f;
  asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(u));
  return f;
}
#endif

inline int check_lambda(const LambdaRef& l) {
  if (l.ptr == nullptr) return TDA_OK;
  if (l.dtype != TDA_F32 && l.dtype != TDA_BF16 && l.dtype != TDA_F16)
    return fail(TDA_ERR_INVALID, "lambda must be TDA_F32, TDA_BF16 or TDA_F16");
  if (l.sb < 0 || l.sh < 0) return fail(TDA_ERR_INVALID, "lambda strides must be >= 0");
  if (!aligned(l.ptr, l.dtype == TDA_F32 ? 4 : 2)) return fail(TDA_ERR_INVALID, "lambda is misaligned");
  return TDA_OK;
}

}  // namespace tda
