// Backward of softmax differential attention on the tensor cores (tcgen05,
// TMEM, TMA): bf16 or fp16, head_dim 64 / 128.  Formulas in tda_sdiff.h; row
// table -L_m(i), -D_m(i) from the row-sum pass (rows past Sq: -inf, 0).
//
// Two kernels, no atomic sums (the same bits every time):
//   dkv, a CTA a tile of 128 keys of one kv head.  Rows are keys: per query tile
//     S^T = K_m Q_m^T, dP^T = V dout^T, then dV += P'^T dout, dK_m += dS^T Q_m,
//     P'_1 = P_1, P'_2 = -lambda P_2 (L and D are subtracted by the products).  It walks map 1's query tiles of every head
//     of the group, writes dK_1, then map 2's: dV sums both maps and all heads in TMEM.
//   dq, a CTA a tile of 128 queries of one head, both maps: per key tile
//     S1 = Q1 K1^T and dP = dout V^T, dP into registers for both maps, S2 = Q2 K2^T
//     over dP, then dQ1 += dS1 K1, dQ2 += dS2 K2: five products instead of six, and
//     each map's S is computed while the other map's weights are formed.
// Sixteen warps (a row's 128 columns over four) hold the weights between the two halves of a step: while they
// exponentiate S, the tensor cores run dK (dQ) of the last step and dP; while
// they form dS, dV and the next S.  P and dS enter the products as one 16-bit
// value each (2^-9 / 2^-12 of an element, averaged over a row; P in dV with its
// rest where rows see few keys, see few_tiles); sums, the
// difference dP - D and the exponent stay in fp32.  O_1, O_2 come in fp32 for D.
// Measured on B200, bf16, 8 heads of (8192, 128), causal: dkv 473 us, tensor pipe
// 66% active (a step's four products take 2048 cycles of its 3000: weights of the
// next step wait for S, S for the last weights' product); dq 334 us, 55% active
// (its warps' own work, 2 x 128 x 128 weights a tile, is longer than its products).
#include <cstring>

#include "tda_sdiff_tc.cuh"

namespace tda {
namespace {

using namespace sd;

constexpr int kProd = 16, kIssue = 17;  // warps after the sixteen; two more fill their warpgroup
constexpr int kThreads = 640;
// registers: 96 a thread at launch (61440); 128 x 64 + 512 x 104 = 61440
constexpr int kFewRegs = 64, kManyRegs = 104;
constexpr int kPolyPairs = 3;  // of 8 go to the FMA pipe instead of the exponential unit
constexpr int kWorkThreads = 512;
constexpr int kTab = 2;
constexpr int ST_KP = 0x901, ST_KM = 0x902, ST_KW = 0x903, ST_QP = 0xa01, ST_QM = 0xa02, ST_QW = 0xa03;

template <int D, bool F16>
struct KvC : Geo<D, F16> {
  using G = Geo<D, F16>;
  static constexpr int kSlots = 4;
  static constexpr int kOffRing = 2 * G::kTileBytes;  // K, V, then the Q / dout ring
  static constexpr int kOffTab = kOffRing + kSlots * G::kTileBytes;  // L and D tables of a step, kTab steps
  static constexpr int kTabBytes = 2 * kAuxTileBytes;
  static constexpr int kOffOnes = kOffTab + kTab * kTabBytes;
  static constexpr int kOffBar = kOffOnes + kAuxTileBytes;
  static constexpr int kSmem = kOffBar + 1024 + 1024;
  static_assert(kSmem <= kSmemBudget, "shared memory");
  static constexpr uint32_t kS = 0, kP = 128, kDV = 256, kDK = 384;
};

struct KvBars {
  uint64_t k_full, v_full, k_free, s_full, dp_full, p_full, ds_full, map_done, drain;
  uint64_t slot_full[4], slot_empty[4], tab_full[kTab], tab_empty[kTab];
  uint32_t tmem_base;
  int abort_flag;
  int weight_exp, ds_exp;  // fp16: see kv_exponents
};

struct KvWork {
  int b, kvh, kt, i0, per_map;  // first query tile, steps of one map
  int few;                      // query tiles whose rows see few keys
};

// K1 and V, issued by the thread that set the barriers up while the others still
// allocate and synchronise
template <int D, bool F16>
__device__ void kv_prime(const SdTcParams& tp, uint8_t* smem, KvBars* bars, const KvWork& w) {
  using C = KvC<D, F16>;
  mbar_arrive_expect_tx(&bars->k_full, C::kTileBytes);
  load_tile<D, F16>(smem, &tp.m.k[0], &bars->k_full, w.kt * kTile, w.kvh, w.b);
  mbar_arrive_expect_tx(&bars->v_full, C::kTileBytes);
  load_tile<D, F16>(smem + C::kTileBytes, &tp.m.v, &bars->v_full, w.kt * kTile, w.kvh, w.b);
}

// Query tiles (the first ones) whose rows see so few keys, 512 at most, that their
// weights, large and few, make most of dV's norm in a causal sequence: there dV
// takes the weights with what rounding left of them, a second product.  Measured
// on B200: dV 2.6e-3 -> 2.0e-3 of its 64-bit value (bf16, causal, 4 heads on 1,
// 4096 of 128; its own rounding is 1.7e-3), dkv 1900 -> 1990 us at (4, 32 on 8,
// 4096, 128) for 10 of its 528 tile pairs a map and head, where all of them take
// 2450 us.  Longer uncausal calls keep 2.6e-3: with it for all of their tiles the
// backward takes 10-12% longer ((6, 16, 1999, 64) fp16 1142 -> 1250 us).
__device__ __forceinline__ int few_tiles(const SdParams& p, int len, int n_qt) {
  if (len <= 512) return n_qt;
  return p.causal ? max(0, 512 - (p.Sk - p.Sq)) / kTile : 0;
}

template <int D, bool F16>
__device__ void kv_produce(const SdTcParams& tp, uint8_t* smem, KvBars* bars, const WaitCtl& ctl, const KvWork& w) {
  using C = KvC<D, F16>;
  const SdParams& p = tp.p;
  bool ok = true;
  int t = 0, idx = 0, n_k = 0;
  for (int m = 0; m < 2 && ok; ++m) {
    if (m == 1) {
      ok = wait_inline(&bars->k_free, 0, ctl, ST_KP);
      if (!ok) break;
      mbar_arrive_expect_tx(&bars->k_full, C::kTileBytes);
      load_tile<D, F16>(smem, &tp.m.k[1], &bars->k_full, w.kt * kTile, w.kvh, w.b);
    }
    ++n_k;
    for (int h = w.kvh * p.group; h < (w.kvh + 1) * p.group && ok; ++h) {
      for (int i = w.i0; i < tp.n_qt; ++i, ++t) {
        const int e = t % kTab;
        ok = wait_inline(&bars->tab_empty[e], ((t / kTab) & 1) ^ 1, ctl, ST_KP);
        if (!ok) break;
        mbar_arrive_expect_tx(&bars->tab_full[e], C::kTabBytes);
        const long long tile = ((static_cast<long long>(m) * p.B + w.b) * p.H + h) * (p.pad / kTile) + i;
        bulk_load(smem + C::kOffTab + e * C::kTabBytes, static_cast<const uint8_t*>(p.aux) + tile * C::kTabBytes, C::kTabBytes,
                  &bars->tab_full[e]);
        for (int x = 0; x < 2; ++x) {
          const int slot = idx % C::kSlots;
          ok = wait_inline(&bars->slot_empty[slot], ((idx / C::kSlots) & 1) ^ 1, ctl, ST_KP);
          if (!ok) break;
          mbar_arrive_expect_tx(&bars->slot_full[slot], C::kTileBytes);
          load_tile<D, F16>(smem + C::kOffRing + slot * C::kTileBytes, x ? &tp.m.dout : &tp.m.q[m], &bars->slot_full[slot], i * kTile, h,
                            w.b);
          ++idx;
        }
        if (!ok) {
          ++t;  // its table entry is in flight
          break;
        }
      }
    }
  }
  if (!ok) {
    drain_wait(&bars->v_full, 0, ctl);
    if (n_k > 0) drain_wait(&bars->k_full, (n_k - 1) & 1, ctl);
    for (int i = idx > C::kSlots ? idx - C::kSlots : 0; i < idx; ++i)
      drain_wait(&bars->slot_full[i % C::kSlots], (i / C::kSlots) & 1, ctl);
    for (int i = t > kTab ? t - kTab : 0; i < t; ++i) drain_wait(&bars->tab_full[i % kTab], (i / kTab) & 1, ctl);
  }
}

template <int D, bool F16>
__device__ void kv_issue(uint8_t* smem, KvBars* bars, const WaitCtl& ctl, uint32_t tmem, int per_map, int i0, int n_qt, int few) {
  using C = KvC<D, F16>;
  const uint32_t k = smem_u32(smem), v = k + C::kTileBytes, ring = smem_u32(smem + C::kOffRing);
  const uint32_t tab = smem_u32(smem + C::kOffTab), ones = smem_u32(smem + C::kOffOnes);
  int i = i0;  // query tile of step t
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = wait_inline_warp(bar, parity, ctl, ST_KM);
    if (ok) tc_fence_after();
  };
  auto acquire = [&](int idx) {
    wait(&bars->slot_full[idx % C::kSlots], (idx / C::kSlots) & 1);
    return ring + (idx % C::kSlots) * C::kTileBytes;
  };
  auto slot = [&](int idx) { return ring + (idx % C::kSlots) * C::kTileBytes; };
  auto score = [&](int t) {  // S^T(t) = K Q(t)^T
    const uint32_t q = acquire(2 * t);
    wait(&bars->tab_full[t % kTab], (t / kTab) & 1);
    if (!ok) return;
    mma_score<D, F16>(tmem + C::kS, k, q);
    mma_offsets<F16>(tmem + C::kS, ones, tab + (t % kTab) * C::kTabBytes);
    commit(&bars->s_full);
  };
  auto dprob = [&](int t) {  // dP^T(t) = V dout(t)^T
    const uint32_t g = acquire(2 * t + 1);
    if (!ok) return;
    mma_score<D, F16>(tmem + C::kP, v, g);
    mma_offsets<F16>(tmem + C::kP, ones, tab + (t % kTab) * C::kTabBytes + kAuxTileBytes);
    commit(&bars->tab_empty[t % kTab]);
    commit(&bars->dp_full);
  };
  wait(&bars->v_full, 0);
  for (int m = 0; m < 2 && ok; ++m) {
    const int t0 = m * per_map, t1 = t0 + per_map;
    wait(&bars->k_full, m);
    score(t0);
    dprob(t0);
    for (int t = t0; t < t1 && ok; ++t) {
      wait(&bars->p_full, t & 1);
      if (!ok) break;
      mma_weights<D, F16, true>(tmem + C::kDV, tmem + C::kS, slot(2 * t + 1), t > 0);
      if (i < few) mma_weights<D, F16, true>(tmem + C::kDV, tmem + C::kS + 16, slot(2 * t + 1), true);
      if (++i == n_qt) i = i0;
      if (t + 1 < t1) score(t + 1);
      wait(&bars->ds_full, t & 1);
      if (!ok) break;
      mma_weights<D, F16, true>(tmem + C::kDK, tmem + C::kP, slot(2 * t), t > t0);
      commit(&bars->slot_empty[(2 * t) % C::kSlots]);
      commit(&bars->slot_empty[(2 * t + 1) % C::kSlots]);
      if (t + 1 < t1) dprob(t + 1);
    }
    if (ok) commit(&bars->map_done);
  }
  if (!ok) {
    commit(&bars->drain);
    drain_wait(&bars->drain, 0, ctl);
  }
}

// fp16 keeps its bits between 2^-14 and 2^16 alone: weights enter the products times
// 2^weight_exp, at most 2^14 with lambda, dS times 2^ds_exp, and the accumulators are
// scaled back.  One thread finds both while the others set up; they are read
// again at the end, since registers kept for them cost dq 5%.
template <int D>
__device__ void kv_exponents(const SdParams& p, KvBars* bars, const KvWork& w) {
  float largest = 1.0f;
  for (int h = w.kvh * p.group; h < (w.kvh + 1) * p.group; ++h) largest = fmaxf(largest, fabsf(lambda_at(p.lam, w.b, h)));
  bars->weight_exp = 14 - exponent_above(largest);
  bars->ds_exp = ds_exponent(p, w.b, w.kvh, D, largest);
}
__device__ __forceinline__ int again(const int& x) { return *const_cast<const volatile int*>(&x); }

// 32 accumulator columns of this thread's row, scaled, into the staged 16-bit tile
template <int D, bool F16>
__device__ __forceinline__ void stage_accumulator(uint8_t* boxes, uint32_t col, int row, int wg, float scale, bool zero) {
#pragma unroll
  for (int x = 32 * wg; x < D; x += 128) {
    float a[32];
    if (!zero) {
      uint32_t u[32];
      tmem_ld32(col + x, u);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) a[i] = __uint_as_float(u[i]) * scale;
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) a[i] = 0.f;
    }
    stage_16<F16>(boxes, row, x, a);
  }
}

// a thread's 32 weights as 16-bit values in the first 16 of its 32 columns
// (REST: what rounding left of them in the other 16)
template <bool F16, bool REST = false>
__device__ __forceinline__ void store_weights(uint32_t col, const float (&x)[32]) {
  uint32_t u[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) u[y] = pack2<F16>(x[2 * y], x[2 * y + 1]);
  tmem_st16(col, u);
  if constexpr (REST) {
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      const float2 h = F16 ? unpack_f16x2(u[y]) : unpack_bf16x2(u[y]);
      const float2 d = __fadd2_rn(make_float2(x[2 * y], x[2 * y + 1]), make_float2(-h.x, -h.y));
      u[y] = pack2<F16>(d.x, d.y);
    }
    tmem_st16(col + 16, u);
  }
}

template <int D, bool F16>
__device__ void kv_work(const SdTcParams& tp, uint8_t* smem, KvBars* bars, const WaitCtl& ctl, uint32_t tmem, const KvWork& w, int len,
                        int warp, int lane) {
  using C = KvC<D, F16>;
  const SdParams& p = tp.p;
  const int wg = warp >> 2, row = (warp & 3) * 32 + lane, key = w.kt * kTile + row, off = p.Sk - p.Sq;
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t s_col = tmem + lane_off + C::kS + 32 * wg, p_col = tmem + lane_off + C::kP + 32 * wg;
  const bool dead = key >= len;          // past the sequence's length: no weight, whatever K and V hold there
  const bool lone = len <= 1;            // weight 1 whatever the score: no dS, but of a NaN
  const float c = p.c;
  const float kf = F16 ? static_cast<float>(bars->weight_exp) : 0.f;
  const float more = F16 ? exp2i(bars->ds_exp - bars->weight_exp) : 1.0f;
  bool ok = true;
  int t = 0;
  if (w.per_map > 0) ok = wait_inline_warp(&bars->v_full, 0, ctl, ST_KW);
  for (int m = 0; m < 2; ++m) {
    for (int h = w.kvh * p.group; h < (w.kvh + 1) * p.group && ok; ++h) {
      const float wt = m ? -lambda_at(p.lam, w.b, h) : 1.0f;
      for (int i = w.i0; i < tp.n_qt && w.per_map > 0; ++i, ++t) {
        ok = wait_inline_warp(&bars->s_full, t & 1, ctl, ST_KW);
        if (!ok) break;
        tc_fence_after();
        const bool masked = (w.kt + 1) * kTile > len || (p.causal && i * kTile + off < (w.kt + 1) * kTile - 1) || lone;
        // queries of this tile in front of `lo` do not see the key
        const int lo = dead ? kTile : (p.causal ? key - off - i * kTile : 0);
        float pr[32];
        {
          uint32_t s[32];
          tmem_ld32(s_col, s);
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            const float2 x = f2u(s[y], s[y + 1]);  // s - L / c
            const float2 z = F16 ? __ffma2_rn(x, make_float2(c, c), make_float2(kf, kf)) : __fmul2_rn(x, make_float2(c, c));
            // a row without a softmax has a NaN for L, and its weights go into dV by themselves
            const float2 ez = (y / 2 * kPolyPairs) % 8 < kPolyPairs ? poly_ex2<F16, true>(z) : make_float2(fast_ex2(z.x), fast_ex2(z.y));
            const float2 r = __fmul2_rn(ez, make_float2(wt, wt));
            pr[y] = r.x;
            pr[y + 1] = r.y;
          }
        }
        if (masked) {
#pragma unroll
          for (int y = 0; y < 32; ++y) pr[y] = 32 * wg + y >= lo ? pr[y] : 0.f;
        }
        if (i < w.few)
          store_weights<F16, true>(s_col, pr);
        else
          store_weights<F16>(s_col, pr);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full);

        ok = wait_inline_warp(&bars->dp_full, t & 1, ctl, ST_KW);
        if (!ok) break;
        tc_fence_after();
        {
          uint32_t s[32];
          tmem_ld32(p_col, s);
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            float2 r = make_float2(pr[y], pr[y + 1]);
            if constexpr (F16) r = __fmul2_rn(r, make_float2(more, more));
            r = __fmul2_rn(r, f2u(s[y], s[y + 1]));  // P (dP - D)
            pr[y] = r.x;
            pr[y + 1] = r.y;
          }
        }
        if (masked) {
#pragma unroll
          for (int y = 0; y < 32; ++y) pr[y] = 32 * wg + y >= lo && !(lone && pr[y] == pr[y]) ? pr[y] : 0.f;
        }
        store_weights<F16>(p_col, pr);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ds_full);
      }
    }
    // dK_m through the K buffer (idle once every product of the map is done), and dV through V's at the end
    if (ok && w.per_map > 0) ok = wait_inline_warp(&bars->map_done, m, ctl, ST_KW);
    tc_fence_after();
    if (ok) {
      stage_accumulator<D, F16>(smem, tmem + lane_off + C::kDK, row, wg, F16 ? p.scale * exp2i(-again(bars->ds_exp)) : p.scale, w.per_map == 0);
      if (m == 1) stage_accumulator<D, F16>(smem + C::kTileBytes, tmem + lane_off + C::kDV, row, wg, F16 ? exp2i(-again(bars->weight_exp)) : 1.0f, w.per_map == 0);
      fence_proxy_async_smem();
    }
    tc_fence_before();
    ok = named_barrier_and(1, kWorkThreads, ok);
    if (!ok) break;
    if (warp == 0 && lane == 0) {
      const int at = w.b * p.Hkv + w.kvh;
      for (int x = 0; x < D / 64; ++x) {
        tma_store_3d(&tp.m.dk[m], smem + x * C::kBoxBytes, 64 * x, w.kt * kTile, at);
        if (m == 1) tma_store_3d(&tp.m.dv, smem + C::kTileBytes + x * C::kBoxBytes, 64 * x, w.kt * kTile, at);
      }
      bulk_commit_group();
      bulk_wait_group_read0();
      if (m == 0 && w.per_map > 0) mbar_arrive(&bars->k_free);
    }
    if (w.per_map == 0) named_barrier_and(2, kWorkThreads, true);  // the staged zeros were read before they are written again
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1) sdiff_tc_dkv_kernel(const __grid_constant__ SdTcParams tp) {
  using C = KvC<D, F16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  KvBars* bars = reinterpret_cast<KvBars*>(smem + C::kOffBar);
  const SdParams& p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  KvWork w;
  int bh;
  tile_of_block(blockIdx.x, tp.n_kt, p.k_together, bh, w.kt);  // the first keys see the most queries
  w.b = bh / p.Hkv;
  w.kvh = bh % p.Hkv;
  const int len = keys_of(p, w.b);
  w.i0 = p.causal ? max(0, w.kt * kTile - (p.Sk - p.Sq)) / kTile : 0;
  w.few = few_tiles(p, len, tp.n_qt);
  w.per_map = w.kt * kTile < len ? p.group * max(0, tp.n_qt - w.i0) : 0;
  if (warp == kProd && lane == 0) {
    uint64_t* one[] = {&bars->k_full, &bars->v_full, &bars->k_free, &bars->s_full, &bars->dp_full, &bars->map_done, &bars->drain};
    for (uint64_t* x : one) mbar_init(x, 1);
    mbar_init(&bars->p_full, 16);
    mbar_init(&bars->ds_full, 16);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], 1);
    }
    for (int i = 0; i < kTab; ++i) {
      mbar_init(&bars->tab_full[i], 1);
      mbar_init(&bars->tab_empty[i], 1);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
    if (w.per_map > 0) kv_prime<D, F16>(tp, smem, bars, w);
  }
  if (threadIdx.x >= 128 && threadIdx.x < 256) {  // the columns' units in every row
    const int r = threadIdx.x - 128;
    uint32_t u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const auto unit = [](int x) { return x / 3 < aux_units(F16) ? aux_unit(F16, x / 3) : 0.f; };
      u[k] = pack2<F16>(unit(2 * k), unit(2 * k + 1));
    }
    uint4* at = reinterpret_cast<uint4*>(smem + C::kOffOnes + (r >> 3) * 256 + (r & 7) * 16);
    at[0] = make_uint4(u[0], u[1], u[2], u[3]);
    at[8] = make_uint4(u[4], u[5], u[6], u[7]);
    fence_proxy_async_smem();
  }
  if constexpr (F16)
    if (threadIdx.x == 0) kv_exponents<D>(p, bars, w);
  if (warp == kIssue) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const WaitCtl ctl = make_wait_ctl(&bars->abort_flag, tp.status, tp.timeout_ns);
  if (warp < kProd) {
    more_registers<kManyRegs>();
    kv_work<D, F16>(tp, smem, bars, ctl, tmem, w, len, warp, lane);
  } else {
    fewer_registers<kFewRegs>();
    if (w.per_map > 0 && warp == kProd && lane == 0) kv_produce<D, F16>(tp, smem, bars, ctl, w);
    if (w.per_map > 0 && warp == kIssue) kv_issue<D, F16>(smem, bars, ctl, uniform(tmem), uniform(w.per_map), uniform(w.i0), tp.n_qt, uniform(w.few));
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssue) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ================================================================== dq
template <int D, bool F16>
struct QC : Geo<D, F16> {
  using G = Geo<D, F16>;
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kOffRing = 3 * G::kTileBytes;  // Q1, Q2, dout, then the K1 / V / K2 ring
  static constexpr int kOffBar = kOffRing + kSlots * G::kTileBytes;
  static constexpr int kSmem = kOffBar + 1024 + 1024;
  static_assert(kSmem <= kSmemBudget, "shared memory");
  static constexpr uint32_t kA = 0, kB = 128;  // S1, then dS1 / dP, then S2, then dS2
  static __device__ __forceinline__ constexpr uint32_t dq_col(int m) { return 256u + 128u * m; }
};

struct QBars {
  uint64_t q_full, o_full, drain, dp_full, dp_free;
  uint64_t s_full[2], ds_full[2];  // per map
  uint64_t slot_full[8], slot_empty[8];
  uint32_t tmem_base;
  int abort_flag;
  int ds_exp;  // fp16: dS enters the products times 2^ds_exp, by the exponent of the weights
};

// tile idx of the ring: K1, V, K2 of key tile idx / 3
template <int D, bool F16>
__device__ __forceinline__ void q_fetch(const SdTcParams& tp, uint8_t* smem, QBars* bars, int b, int kvh, int idx) {
  using C = QC<D, F16>;
  const int slot = idx % C::kSlots, x = idx % 3;
  mbar_arrive_expect_tx(&bars->slot_full[slot], C::kTileBytes);
  load_tile<D, F16>(smem + C::kOffRing + slot * C::kTileBytes, x == 1 ? &tp.m.v : &tp.m.k[x >> 1], &bars->slot_full[slot], idx / 3 * kTile,
                    kvh, b);
}

// the loads that wait for nothing, as in the forward
template <int D, bool F16>
__device__ int q_prime(const SdTcParams& tp, uint8_t* smem, QBars* bars, int b, int h, int kvh, int qt, int n) {
  using C = QC<D, F16>;
  mbar_arrive_expect_tx(&bars->q_full, 3 * C::kTileBytes);
  load_tile<D, F16>(smem, &tp.m.q[0], &bars->q_full, qt * kTile, h, b);
  q_fetch<D, F16>(tp, smem, bars, b, kvh, 0);
  load_tile<D, F16>(smem + 2 * C::kTileBytes, &tp.m.dout, &bars->q_full, qt * kTile, h, b);
  load_tile<D, F16>(smem + C::kTileBytes, &tp.m.q[1], &bars->q_full, qt * kTile, h, b);
  const int primed = min(3 * n, C::kSlots);
  for (int idx = 1; idx < primed; ++idx) q_fetch<D, F16>(tp, smem, bars, b, kvh, idx);
  return primed;
}

template <int D, bool F16>
__device__ void q_produce(const SdTcParams& tp, uint8_t* smem, QBars* bars, const WaitCtl& ctl, int b, int kvh, int n, int idx) {
  using C = QC<D, F16>;
  bool ok = true;
  for (; idx < 3 * n; ++idx) {
    ok = wait_inline(&bars->slot_empty[idx % C::kSlots], ((idx / C::kSlots) & 1) ^ 1, ctl, ST_QP);
    if (!ok) break;
    q_fetch<D, F16>(tp, smem, bars, b, kvh, idx);
  }
  if (!ok) {
    drain_wait(&bars->q_full, 0, ctl);
    for (int i = idx > C::kSlots ? idx - C::kSlots : 0; i < idx; ++i)
      drain_wait(&bars->slot_full[i % C::kSlots], (i / C::kSlots) & 1, ctl);
  }
}

template <int D, bool F16>
__device__ void q_issue(uint8_t* smem, QBars* bars, const WaitCtl& ctl, uint32_t tmem, int n) {
  using C = QC<D, F16>;
  const uint32_t q = smem_u32(smem), g = q + 2 * C::kTileBytes, ring = smem_u32(smem + C::kOffRing);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = wait_inline_warp(bar, parity, ctl, ST_QM);
    if (ok) tc_fence_after();
  };
  auto slot = [&](int idx) { return ring + (idx % C::kSlots) * C::kTileBytes; };
  auto acquire = [&](int idx) {
    wait(&bars->slot_full[idx % C::kSlots], (idx / C::kSlots) & 1);
    return slot(idx);
  };
  auto score = [&](int t, int m) {
    const uint32_t k = acquire(3 * t + 2 * m);
    if (!ok) return;
    mma_score<D, F16>(tmem + (m ? C::kB : C::kA), q + m * C::kTileBytes, k);
    commit(&bars->s_full[m]);
  };
  auto dprob = [&](int t) {
    const uint32_t v = acquire(3 * t + 1);
    if (!ok) return;
    mma_score<D, F16>(tmem + C::kB, g, v);
    commit(&bars->slot_empty[(3 * t + 1) % C::kSlots]);
    commit(&bars->dp_full);
  };
  wait(&bars->q_full, 0);
  if (ok) {
    score(0, 0);
    dprob(0);
  }
  for (int t = 0; t < n && ok; ++t) {
    wait(&bars->dp_free, t & 1);
    if (ok) score(t, 1);
    wait(&bars->ds_full[0], t & 1);
    if (!ok) break;
    mma_weights<D, F16, true>(tmem + C::dq_col(0), tmem + C::kA, slot(3 * t), t > 0);
    commit(&bars->slot_empty[(3 * t) % C::kSlots]);
    if (t + 1 < n) score(t + 1, 0);
    wait(&bars->ds_full[1], t & 1);
    if (!ok) break;
    mma_weights<D, F16, true>(tmem + C::dq_col(1), tmem + C::kB, slot(3 * t + 2), t > 0);
    commit(&bars->slot_empty[(3 * t + 2) % C::kSlots]);
    if (t + 1 < n) dprob(t + 1);
  }
  if (ok) {
    commit(&bars->o_full);
  } else {
    commit(&bars->drain);
    drain_wait(&bars->drain, 0, ctl);
  }
}

template <int D, bool F16>
__device__ void q_work(const SdTcParams& tp, uint8_t* smem, QBars* bars, const WaitCtl& ctl, uint32_t tmem, int b, int h, int qt, int n,
                       int len, int warp, int lane) {
  using C = QC<D, F16>;
  const SdParams& p = tp.p;
  const int wg = warp >> 2, row = (warp & 3) * 32 + lane, grow = qt * kTile + row, off = p.Sk - p.Sq;
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t a_col = tmem + lane_off + C::kA + 32 * wg, b_col = tmem + lane_off + C::kB + 32 * wg;
  const long long bh = static_cast<long long>(b) * p.H + h;
  float minus_l[2], minus_d[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float* t = p.table + 2 * ((static_cast<long long>(m) * p.B * p.H + bh) * p.pad + qt * kTile) + row;
    minus_l[m] = t[0];
    minus_d[m] = t[kTile];
  }
  const float c = p.c;
  if constexpr (F16) {
    minus_l[0] += static_cast<float>(bars->ds_exp);
    minus_l[1] += static_cast<float>(bars->ds_exp);
  }
  const int last = p.causal ? min(len - 1, grow + off) : len - 1;
  const bool lone = len <= 1;  // weight 1 whatever the score: no dS, but of a NaN
  bool ok = true;
  for (int t = 0; t < n && ok; ++t) {
    const bool masked = (t + 1) * kTile > len || (p.causal && (t + 1) * kTile - 1 > qt * kTile + off);
    const bool tail = t == n - 1 && len < p.Sk && (t + 1) * kTile > len;
    const int lim = last - t * kTile - 32 * wg;
    float dp[32];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      ok = wait_inline_warp(&bars->s_full[m], t & 1, ctl, ST_QW);
      if (!ok) break;
      tc_fence_after();
      float pr[32];
      {
        uint32_t s[32];
        tmem_ld32(m ? b_col : a_col, s);
        tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
          const float2 z = __ffma2_rn(f2u(s[y], s[y + 1]), make_float2(c, c), make_float2(minus_l[m], minus_l[m]));
          // where L is NaN so is D, which the weight is multiplied by below
          const float2 ez = (y / 2 * kPolyPairs) % 8 < kPolyPairs ? poly_ex2<F16>(z) : make_float2(fast_ex2(z.x), fast_ex2(z.y));
          pr[y] = ez.x;
          pr[y + 1] = ez.y;
        }
      }
      if (m == 0) {  // dP serves both maps
        ok = wait_inline_warp(&bars->dp_full, t & 1, ctl, ST_QW);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32];
        tmem_ld32(b_col, s);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->dp_free);
#pragma unroll
        for (int y = 0; y < 32; ++y) dp[y] = __uint_as_float(s[y]);
      }
#pragma unroll
      for (int y = 0; y < 32; y += 2) {
        const float2 d = __fadd2_rn(make_float2(dp[y], dp[y + 1]), make_float2(minus_d[m], minus_d[m]));
        const float2 r = __fmul2_rn(make_float2(pr[y], pr[y + 1]), d);
        pr[y] = r.x;
        pr[y + 1] = r.y;
      }
      if (masked) {
#pragma unroll
        for (int y = 0; y < 32; ++y) pr[y] = y <= lim && !(lone && pr[y] == pr[y]) ? pr[y] : 0.f;
      }
      // K rows past the length: zeroed (S is done with them) before the product with dS reads them
      if (tail) {
        if (wg == 0 && t * kTile + row >= len) zero_row<D>(smem + C::kOffRing + ((3 * t + 2 * m) % C::kSlots) * C::kTileBytes, row);
        fence_proxy_async_smem();
      }
      store_weights<F16>(m ? b_col : a_col, pr);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ds_full[m]);
    }
  }
  if (ok && n > 0) ok = wait_inline_warp(&bars->o_full, 0, ctl, ST_QW);
  tc_fence_after();
  uint8_t* stage = smem + C::kOffRing;
  if (ok) {
    const float back = F16 ? p.scale * exp2i(-again(bars->ds_exp)) : p.scale;
    const float w2 = -lambda_at(p.lam, b, h) * back;
    stage_accumulator<D, F16>(stage, tmem + lane_off + C::dq_col(0), row, wg, back, n == 0);
    stage_accumulator<D, F16>(stage + C::kTileBytes, tmem + lane_off + C::dq_col(1), row, wg, w2, n == 0);
    fence_proxy_async_smem();
  }
  ok = named_barrier_and(2, kWorkThreads, ok);
  if (ok && warp == 0 && lane == 0) {
    for (int m = 0; m < 2; ++m)
      for (int x = 0; x < D / 64; ++x)
        tma_store_3d(&tp.m.dq[m], stage + m * C::kTileBytes + x * C::kBoxBytes, 64 * x, qt * kTile, static_cast<int>(bh));
    bulk_commit_group();
    bulk_wait_group_read0();
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1) sdiff_tc_dq_kernel(const __grid_constant__ SdTcParams tp) {
  using C = QC<D, F16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  QBars* bars = reinterpret_cast<QBars*>(smem + C::kOffBar);
  const SdParams& p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int bh, qt;
  tile_of_block(blockIdx.x, tp.n_qt, p.q_together, bh, qt);
  qt = tp.n_qt - 1 - qt;  // longest rows first
  const int b = bh / p.H, h = bh % p.H, kvh = h / p.group;
  const int len = keys_of(p, b);
  int n_keys = len;
  if (p.causal) n_keys = max(0, min(n_keys, min((qt + 1) * kTile, p.Sq) + p.Sk - p.Sq));
  const int n = (n_keys + kTile - 1) / kTile;
  int primed = 0;
  if (warp == kProd && lane == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->o_full, 1);
    mbar_init(&bars->drain, 1);
    mbar_init(&bars->dp_full, 1);
    mbar_init(&bars->dp_free, 16);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->ds_full[i], 16);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&bars->slot_full[i], 1);
      mbar_init(&bars->slot_empty[i], 1);
    }
    bars->abort_flag = 0;
    fence_mbar_init();
    if (n > 0) primed = q_prime<D, F16>(tp, smem, bars, b, h, kvh, qt, n);
  }
  if constexpr (F16)
    if (threadIdx.x == 0) bars->ds_exp = ds_exponent(p, b, kvh, D, 1.0f);
  if (warp == kIssue) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const WaitCtl ctl = make_wait_ctl(&bars->abort_flag, tp.status, tp.timeout_ns);
  if (warp < kProd) {
    more_registers<kManyRegs>();
    q_work<D, F16>(tp, smem, bars, ctl, tmem, b, h, qt, n, len, warp, lane);
  } else {
    fewer_registers<kFewRegs>();
    if (n > 0 && warp == kProd && lane == 0) q_produce<D, F16>(tp, smem, bars, ctl, b, kvh, n, primed);
    if (n > 0 && warp == kIssue) q_issue<D, F16>(smem, bars, ctl, uniform(tmem), n);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssue) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool F16>
cudaError_t launch(const SdTcParams& tp, cudaStream_t s) {
  auto kq = sdiff_tc_dq_kernel<D, F16>;
  auto kk = sdiff_tc_dkv_kernel<D, F16>;
  if (cudaError_t e = allow_shared<sdiff_tc_dq_kernel<D, F16>>(QC<D, F16>::kSmem)) return e;
  if (cudaError_t e = allow_shared<sdiff_tc_dkv_kernel<D, F16>>(KvC<D, F16>::kSmem)) return e;
  kk<<<static_cast<unsigned>(tp.p.B * tp.p.Hkv * tp.n_kt), kThreads, KvC<D, F16>::kSmem, s>>>(tp);
  if (cudaError_t e = cudaGetLastError()) return e;
  kq<<<static_cast<unsigned>(tp.p.B * tp.p.H * tp.n_qt), kThreads, QC<D, F16>::kSmem, s>>>(tp);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_sdiff_tc_bwd(const SdTcParams& tp, int dtype, int D, cudaStream_t s) {
  if (dtype == TDA_BF16) return D == 64 ? launch<64, false>(tp, s) : launch<128, false>(tp, s);
  return D == 64 ? launch<64, true>(tp, s) : launch<128, true>(tp, s);
}

}  // namespace tda
