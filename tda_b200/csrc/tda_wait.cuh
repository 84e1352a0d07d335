// Bounded barrier waits without a function call.
#pragma once

#include "tda_ptx.cuh"

namespace tda {

// mbar_wait in line: a warp whose register count changes (setmaxnreg) may not call
// a function, and a call in an inner loop costs the registers it may overwrite.
__device__ __forceinline__ bool wait_inline(uint64_t* bar, uint32_t parity, const WaitCtl& ctl, int code) {
  const uint32_t a = smem_u32(bar);
  if (mbar_try_wait(a, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(a, parity)) {
    if (*ctl.abort_flag) return false;
    const uint64_t waited = global_timer_ns() - t0;
    const bool other = waited > 1000000ull && *reinterpret_cast<volatile int*>(ctl.status) != ctl.status0;
    if (other || waited > ctl.timeout_ns) {
      *ctl.abort_flag = 1;
      if (!other) atomicCAS(ctl.status, 0, code);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_inline_warp(uint64_t* bar, uint32_t parity, const WaitCtl& ctl, int code) {
  const bool ok = wait_inline(bar, parity, ctl, code);
  return __all_sync(0xffffffffu, ok);
}

}  // namespace tda
