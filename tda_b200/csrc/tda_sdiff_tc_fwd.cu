// Forward of softmax differential attention on the tensor cores (tcgen05,
// TMEM, TMA): bf16 or fp16, head_dim 64 / 128.
//
// One CTA takes 128 query rows of one head and both maps, so V is loaded once
// for the two products with it.  Two warpgroups, a map each, one thread a row:
//   warps 0-3 map 1, warps 4-7 map 2, warp 8 TMA producer, warp 9 issues products
// TMEM columns: S1 0, S2 128, O1 256, O2 384.  P_m (16 bit, 64 columns)
// replaces S_m.  The issuing thread alternates
//   O1 += P1(j) V(j), S1(j+1) = Q1 K1(j+1)^T, O2 += P2(j) V(j), S2(j+1) = Q2 K2(j+1)^T
// so the tensor cores work on one map while the other map's warpgroup
// exponentiates.  Products of one thread run in order, hence S_m(j+1) may
// overwrite P_m(j), and whoever saw S_m(j+1) complete knows that O_m holds
// tiles 0..j and is not being written: the rescaling of O needs no barrier of
// its own.  It is rare: the row maximum m moves only when a score passes it by
// 2^8 in the weight (weights stay below 2^8, sums and O in fp32, so nothing is
// lost), which after the first tiles almost never happens.
//
// A key tile has four products of 128^3 (2048 cycles at the tensor peak) and 2 x
// 128 x 128 exponentials (2048 at 16 a cycle and SM, so 3 of 8 pairs go to the FMA
// pipe as a polynomial).  What bounds it is the hand-over: scores ready, 500
// cycles to the row maximum, 1400 for the weights, 1300 until the products that
// need them are done, for two maps in turn, 3200 a tile.  Measured on B200, bf16
// (1,16,32768,128): 7.7 to 8.2 ms by the card, 1080-1140 TFLOP/s of executed
// products; (8 heads, 8192): 254 us, tensor pipe 59% active, exponential unit 38%.
// Polynomials for 0 to 4 of 8 pairs differ by 3%.
//
// P_m enters its product as one 16-bit value, which leaves out with 1.4 to 1.6 times
// the error of a single rounding (the most where rows see many keys and the maps'
// common mean cancels).  A second product with the rounding rest brings that to 1.0 and
// costs more than it is worth: 7.95 -> 12.6 ms at (1,16,32768,128), 374 -> 506 us at
// (6,16,1999,64) fp16.
#include <cstring>

#include "tda_sdiff_tc.cuh"

namespace tda {
namespace {

using namespace sd;

constexpr int kThreads = 384;  // warps 10 and 11 fill the third warpgroup
// registers: 168 a thread at launch (64512); 128 x 72 + 256 x 216 = 64512
constexpr int kFewRegs = 72, kManyRegs = 216;
constexpr int kSoftmaxThreads = 256;
constexpr int ST_PROD = 0x801, ST_MMA = 0x802, ST_SM = 0x803;
constexpr float kLazy = 8.0f;
constexpr int kPolyPairs = 3;  // of 8

template <int D, bool F16>
struct FC : Geo<D, F16> {
  using G = Geo<D, F16>;
  static constexpr int kBarBytes = 1024 + 2 * kTile * 4;
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kOffRing = 2 * G::kTileBytes;
  static constexpr int kOffBar = kOffRing + kSlots * G::kTileBytes;
  static constexpr int kSmem = kOffBar + kBarBytes + 1024;
  static_assert(kSmem <= kSmemBudget, "shared memory");
  static_assert(kSlots * G::kTileBytes >= kTile * D * 10, "the ring holds the staged out, O1 and O2");
  static __device__ __forceinline__ constexpr uint32_t s_col(int m) { return 128u * m; }
  static __device__ __forceinline__ constexpr uint32_t o_col(int m) { return 256u + 128u * m; }
};

struct FBars {
  uint64_t q_full, o_full, drain;
  uint64_t s_full[2], p_half[2], p_full[2];
  uint64_t slot_full[8], slot_empty[8];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(FBars) <= 1024, "barriers");

// tile idx of the ring: K1, K2, V of key tile idx / 3
template <int D, bool F16>
__device__ __forceinline__ void fetch(const SdTcParams& tp, uint8_t* smem, FBars* bars, int b, int kvh, int idx) {
  using C = FC<D, F16>;
  const int slot = idx % C::kSlots, x = idx % 3;
  mbar_arrive_expect_tx(&bars->slot_full[slot], C::kTileBytes);
  load_tile<D, F16>(smem + C::kOffRing + slot * C::kTileBytes, x == 2 ? &tp.m.v : &tp.m.k[x], &bars->slot_full[slot], idx / 3 * kTile,
                    kvh, b);
}

// The loads that wait for nothing, issued by the thread that set the barriers up
// while the others still allocate and synchronise (1500 cycles of a CTA's start).
template <int D, bool F16>
__device__ int prime(const SdTcParams& tp, uint8_t* smem, FBars* bars, int b, int h, int kvh, int qt, int n) {
  using C = FC<D, F16>;
  mbar_arrive_expect_tx(&bars->q_full, 2 * C::kTileBytes);
  load_tile<D, F16>(smem, &tp.m.q[0], &bars->q_full, qt * kTile, h, b);
  fetch<D, F16>(tp, smem, bars, b, kvh, 0);
  load_tile<D, F16>(smem + C::kTileBytes, &tp.m.q[1], &bars->q_full, qt * kTile, h, b);
  const int primed = min(3 * n, C::kSlots);
  for (int idx = 1; idx < primed; ++idx) fetch<D, F16>(tp, smem, bars, b, kvh, idx);
  return primed;
}

template <int D, bool F16>
__device__ void produce(const SdTcParams& tp, uint8_t* smem, FBars* bars, const WaitCtl& ctl, int b, int kvh, int n, int idx) {
  using C = FC<D, F16>;
  bool ok = true;
  for (; idx < 3 * n; ++idx) {
    ok = wait_inline(&bars->slot_empty[idx % C::kSlots], ((idx / C::kSlots) & 1) ^ 1, ctl, ST_PROD);
    if (!ok) break;
    fetch<D, F16>(tp, smem, bars, b, kvh, idx);
  }
  if (!ok) {
    drain_wait(&bars->q_full, 0, ctl);
    for (int i = idx > C::kSlots ? idx - C::kSlots : 0; i < idx; ++i)
      drain_wait(&bars->slot_full[i % C::kSlots], (i / C::kSlots) & 1, ctl);
  }
}

template <int D, bool F16>
__device__ void issue(uint8_t* smem, FBars* bars, const WaitCtl& ctl, uint32_t tmem, int n) {
  using C = FC<D, F16>;
  const uint32_t q = smem_u32(smem), ring = smem_u32(smem + C::kOffRing);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = wait_inline_warp(bar, parity, ctl, ST_MMA);
    if (ok) tc_fence_after();
  };
  auto acquire = [&](int idx) {
    wait(&bars->slot_full[idx % C::kSlots], (idx / C::kSlots) & 1);
    return ring + (idx % C::kSlots) * C::kTileBytes;
  };
  auto score = [&](int m, int j) {
    const uint32_t k = acquire(3 * j + m);
    if (!ok) return;
    mma_score<D, F16>(tmem + C::s_col(m), q + m * C::kTileBytes, k);
    commit(&bars->slot_empty[(3 * j + m) % C::kSlots]);
    commit(&bars->s_full[m]);
  };
  wait(&bars->q_full, 0);
  score(0, 0);
  score(1, 0);
  for (int j = 0; j < n && ok; ++j) {
    const uint32_t v = acquire(3 * j + 2);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      wait(&bars->p_half[m], j & 1);
      if (!ok) break;
      mma_weights<D, F16, false, 0, 4>(tmem + C::o_col(m), tmem + C::s_col(m), v, j > 0);
      wait(&bars->p_full[m], j & 1);
      if (!ok) break;
      mma_weights<D, F16, false, 4, 8>(tmem + C::o_col(m), tmem + C::s_col(m), v, true);
      if (m == 1) commit(&bars->slot_empty[(3 * j + 2) % C::kSlots]);
      if (j + 1 < n) score(m, j + 1);
    }
  }
  if (ok) {
    commit(&bars->o_full);
  } else {
    commit(&bars->drain);
    drain_wait(&bars->drain, 0, ctl);
  }
}

// 32 scores of a row to weights 2^(c s + base), written as 16 bits to TMEM; of
// every 8 pairs, POLY go to the FMA pipe instead of the exponential unit.
template <bool F16, int POLY>
__device__ __forceinline__ void exponentials(const uint32_t (&s)[32], float c, float base, float2 (&sum)[2], uint32_t col) {
  uint32_t w[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const float2 e = __ffma2_rn(f2u(s[2 * x], s[2 * x + 1]), make_float2(c, c), make_float2(base, base));
    const float2 pr = (x * POLY) % 8 < POLY ? poly_ex2<F16>(e) : make_float2(fast_ex2(e.x), fast_ex2(e.y));
    sum[x & 1] = __fadd2_rn(sum[x & 1], pr);
    w[x] = pack2<F16>(pr.x, pr.y);
  }
  tmem_st16(col, w);
}

// The polynomial exponential is finite whatever the score, so that rows which have no
// softmax are found by their sum and their maximum, off the common path: a sum
// of weights (2^30 of 2^8 at most) is larger than 2^100 if a score was NaN
// (poly_ex2), and after a score of +infinity the maximum is.  Both rows become NaN, as the
// definition has it, and so does a row whose scores are all -infinity: its maximum is,
// and the polynomial's 2^-125 are no weights.
__device__ __forceinline__ float checked(float sum, float top) {
  return sum < 0x1p100f && top < __builtin_huge_valf() ? sum : __uint_as_float(0x7fffffffu);
}

template <int D, bool F16>
__device__ void softmax(const SdTcParams& tp, uint8_t* smem, FBars* bars, const WaitCtl& ctl, uint32_t tmem, int b, int h, int qt,
                        int n, int len, int warp, int lane) {
  using C = FC<D, F16>;
  const SdParams& p = tp.p;
  const int m = warp >> 2, row = (warp & 3) * 32 + lane, grow = qt * kTile + row;
  const int off = p.Sk - p.Sq;
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t s_col = tmem + lane_off + C::s_col(m), o_col = tmem + lane_off + C::o_col(m);
  const int last = p.causal ? min(len - 1, grow + off) : len - 1;  // last key the row sees
  const float c = p.c;
  float top = -__builtin_huge_valf();  // running maximum of c s
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  bool ok = true;
  for (int j = 0; j < n; ++j) {
    ok = wait_inline_warp(&bars->s_full[m], j & 1, ctl, ST_SM);
    if (!ok) break;
    tc_fence_after();
    uint32_t s[4][32];
#pragma unroll
    for (int i = 0; i < 4; ++i) tmem_ld32(s_col + 32 * i, s[i]);
    tmem_wait_ld();
    const bool masked = (j + 1) * kTile > len || (p.causal && (j + 1) * kTile - 1 > qt * kTile + off);
    if (masked) {
      const int lim = last - j * kTile;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 32; ++x) s[i][x] = 32 * i + x <= lim ? s[i][x] : 0xff800000u;
    }
    float mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mx[i] = __uint_as_float(s[i][0]);
#pragma unroll
      for (int x = 1; x < 31; x += 2) mx[i] = max3f(mx[i], __uint_as_float(s[i][x]), __uint_as_float(s[i][x + 1]));
      mx[i] = fmaxf(mx[i], __uint_as_float(s[i][31]));
    }
    const float now = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
    const bool grow_m = now > top + kLazy;
    if (__any_sync(0xffffffffu, grow_m)) {
      const float f = grow_m ? fast_ex2(top - now) : 1.0f;  // 0 for a row's first keys
      if (grow_m) top = now;
#pragma unroll
      for (int i = 0; i < 2; ++i) sum[i] = __fmul2_rn(make_float2(checked(sum[i].x, top), checked(sum[i].y, top)), make_float2(f, f));
      if (j > 0) {
#pragma unroll
        for (int x = 0; x < D; x += 16) {
          uint32_t o[16];
          tmem_ld16(o_col + x, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st16(o_col + x, o);
        }
      }
    }
    // V rows past the length: zeroed before the product reads them
    if (j == n - 1 && len < p.Sk && (j + 1) * kTile > len) {
      const int idx = 3 * j + 2;
      ok = wait_inline_warp(&bars->slot_full[idx % C::kSlots], (idx / C::kSlots) & 1, ctl, ST_SM);
      if (!ok) break;
      if (j * kTile + row >= len) zero_row<D>(smem + C::kOffRing + (idx % C::kSlots) * C::kTileBytes, row);
      fence_proxy_async_smem();
    }
    const float base = top == -__builtin_huge_valf() ? 0.f : -top;  // a row without keys so far: 2^(-inf)
    auto arrive = [&](uint64_t* bar) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    if (masked) {  // hidden keys are -inf: exactly 0 by the hardware's exponential alone
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        exponentials<F16, 0>(s[i], c, base, sum, s_col + 16 * i);
        if (i == 1) arrive(&bars->p_half[m]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        exponentials<F16, kPolyPairs>(s[i], c, base, sum, s_col + 16 * i);
        if (i == 1) arrive(&bars->p_half[m]);
      }
    }
    arrive(&bars->p_full[m]);
  }
  // epilogue: out = O1 / l1 - lambda O2 / l2, a warpgroup half of the columns
  float* inv = reinterpret_cast<float*>(smem + C::kOffBar + 1024);
  const float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  float l = checked(all, top);
  if (top == -__builtin_huge_valf() && all < 1.0f) l = last >= 0 ? __uint_as_float(0x7fffffffu) : 0.f;
  inv[m * kTile + row] = l == 0.f ? 0.f : 1.0f / l;
  const long long bh = static_cast<long long>(b) * p.H + h, n_bh = static_cast<long long>(p.B) * p.H;
  if (p.lse && grow < p.Sq) p.lse[(m * n_bh + bh) * p.Sq + grow] = l == 0.f ? __builtin_huge_valf() : top + log2f(l);
  if (ok && n > 0) ok = wait_inline_warp(&bars->o_full, 0, ctl, ST_SM);
  tc_fence_after();
  named_barrier_and(1, kSoftmaxThreads, true);
  const float i1 = inv[row], i2 = inv[kTile + row], lam = lambda_at(p.lam, b, h);
  uint8_t* stage = smem + C::kOffRing;
  uint8_t* stage1 = stage + C::kTileBytes;
  uint8_t* stage2 = stage1 + kTile * D * 4;
  // 32 columns at a time; a warpgroup's boxes leave as soon as they are staged
  const bool leader = (warp & 3) == 0 && lane == 0;
#pragma unroll
  for (int x = m * (D / 2); x < (m + 1) * (D / 2); x += 32) {
    if (ok) {
      float a[32], d[32];
      if (n > 0) {
        uint32_t u[32], v[32];
        tmem_ld32(tmem + lane_off + C::o_col(0) + x, u);
        tmem_ld32(tmem + lane_off + C::o_col(1) + x, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          a[i] = __uint_as_float(u[i]) * i1;
          d[i] = __uint_as_float(v[i]) * i2;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) a[i] = d[i] = 0.f;
      }
      if (p.o12) {
        stage_f32(stage1, row, x, a);
        stage_f32(stage2, row, x, d);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) a[i] -= lam * d[i];
      stage_16<F16>(stage, row, x, a);
      fence_proxy_async_smem();
    }
    if (p.o12) {
      ok = named_barrier_and(2 + m, 128, ok);
      if (ok && leader) {
        const int box = x / 32;
        tma_store_3d(&tp.m.o12, stage1 + box * C::kBoxBytes, x, qt * kTile, static_cast<int>(bh));
        tma_store_3d(&tp.m.o12, stage2 + box * C::kBoxBytes, x, qt * kTile, static_cast<int>(n_bh + bh));
      }
    }
  }
  ok = named_barrier_and(1, kSoftmaxThreads, ok);
  if (ok && warp == 0 && lane == 0)
    for (int x = 0; x < D / 64; ++x) tma_store_3d(&tp.m.out, stage + x * C::kBoxBytes, 64 * x, qt * kTile, static_cast<int>(bh));
  if (leader) {
    bulk_commit_group();
    bulk_wait_group_read0();
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1) sdiff_tc_fwd_kernel(const __grid_constant__ SdTcParams tp) {
  using C = FC<D, F16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  FBars* bars = reinterpret_cast<FBars*>(smem + C::kOffBar);
  const SdParams& p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int bh, qt;
  tile_of_block(blockIdx.x, tp.n_qt, p.q_together, bh, qt);
  qt = tp.n_qt - 1 - qt;  // longest rows first
  const int b = bh / p.H, h = bh % p.H, kvh = h / p.group;
  const int len = keys_of(p, b);
  int n_keys = len;
  if (p.causal) n_keys = max(0, min(len, min((qt + 1) * kTile, p.Sq) + p.Sk - p.Sq));
  const int n = (n_keys + kTile - 1) / kTile;
  int primed = 0;
  if (warp == 8 && lane == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->o_full, 1);
    mbar_init(&bars->drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_half[i], 4);
      mbar_init(&bars->p_full[i], 4);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], 1);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
    if (n > 0) primed = prime<D, F16>(tp, smem, bars, b, h, kvh, qt, n);
  }
  if (warp == 9) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const WaitCtl ctl = make_wait_ctl(&bars->abort_flag, tp.status, tp.timeout_ns);
  if (warp < 8) {
    more_registers<kManyRegs>();
    softmax<D, F16>(tp, smem, bars, ctl, tmem, b, h, qt, n, len, warp, lane);
  } else {
    fewer_registers<kFewRegs>();
    if (n > 0 && warp == 8 && lane == 0) produce<D, F16>(tp, smem, bars, ctl, b, kvh, n, primed);
    if (n > 0 && warp == 9) issue<D, F16>(smem, bars, ctl, uniform(tmem), n);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool F16>
cudaError_t launch(const SdTcParams& tp, cudaStream_t s) {
  using C = FC<D, F16>;
  auto k = sdiff_tc_fwd_kernel<D, F16>;
  if (cudaError_t e = allow_shared<sdiff_tc_fwd_kernel<D, F16>>(C::kSmem)) return e;
  k<<<static_cast<unsigned>(tp.p.B * tp.p.H * tp.n_qt), kThreads, C::kSmem, s>>>(tp);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_sdiff_tc_fwd(const SdTcParams& tp, int dtype, int D, cudaStream_t s) {
  if (dtype == TDA_BF16) return D == 64 ? launch<64, false>(tp, s) : launch<128, false>(tp, s);
  return D == 64 ? launch<64, true>(tp, s) : launch<128, true>(tp, s);
}

}  // namespace tda
