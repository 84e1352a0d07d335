// Attention of one new token a request over the 4-bit paged cache.
//
//   softmax form:    out = (softmax(c q1 K1^T) - lambda softmax(c q2 K2^T)) V
//   threshold form:  out = (P1 - clamp(lambda) P2) V, P_m = relu(qh_m Kh_m^T - tau)^p,
//                    tau = beta sqrt(2 ln(len) / D), qh = q / max(|q|, 1e-12) with a cache of normalized keys
//
// Bound by the cache bytes, 3 (D/2 + D/16) a token and kv head (216 at D = 128),
// and next to them by issuing: about 500 instructions a slab and warp.  Measured
// on B200, D = 128, 32 query heads on 8: 64 requests of 8192 tokens 208 us (906 MB,
// 4.4 TB/s, 67% of a copy's rate; issue slots 60%, logic pipe 53% busy), 128
// uneven ones of up to 16384 380-435 us by their lengths; the threshold form 147 us
// for 555 MB.
// Each warp walks slabs of 16 tokens by itself: one bulk copy a slab into its
// own ring in shared memory, several slabs ahead, no barrier with other warps.
// The products are m16n8k16 with the cache as the A operand, stored in fragment
// order (tda_cache4.cuh), and 8 columns of queries: up to 4 heads of the kv
// head's group times the two maps, so that both maps share one pass over V:
//   S^T (16 tokens x 8) = K1 [Q1 0]^T + K2 [0 Q2]^T
//   O^T (D x 8) += V^T (P s)^T
// Codes become fp16 by the exponent trick, (w & 0x000f000f) | 0x6400 = 1024 + n
// and (w & 0x00f000f0) | 0x6400 = 1024 + 16 n, n = code + 8: one logic operation
// a register and a shift every fourth (logic operations issue at half rate and
// are what bounds the kernel next to DRAM).  The factor 16 is divided out of
// those dims of q, and of those rows of O at the end.  For K the product starts
// from minus the offset's share, which removes it without an instruction (exact
// products summed in fp32: an error near 1e-4 of |q| times a code unit).  V
// subtracts it (exact), and so does the threshold form with fp16 queries for the
// nibbles of the larger offset: its weights are powers of s - tau, where the error
// would show (4e-4 of the output; a bf16 output's own rounding is 2e-3).  K's scale multiplies a group's fp32 product.
// q enters as fp16 after division by a power of two that brings its largest
// element to [2^14, 2^15), next to the end of fp16's range, half of its dims a
// sixteenth of that: an element is rounded there by 2^-25 at most, so a bf16
// element is exact down to 2^-27 of the largest, an fp16 one to 2^-24.
// V's scale goes into the weight, w = p s, rounded to fp16 (2^-12) relative to a
// running bound M >= log2 of the largest w so far (minus 8): weights lie below
// 2^8 and small scales do not underflow.  As long as all scales are zero, M bounds p
// alone (no weight is added yet, and a bound on w would be -infinity), and the first
// scale that is not zero joins it; M stays above -120, below which 2^-M
// has no float and w adds nothing to a 16-bit output.  The threshold form forms its whole
// weight (p1 - lambda p2) s at once, which takes the columns of one map, so the
// other four carry what rounding left: nothing is lost where the maps cancel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "tda_cache4.cuh"
#include "tda_host.h"
#include "tda_ptx.cuh"
#include "tda_transform.cuh"
#include "tda_wait.cuh"

namespace tda {

int cache4_check(const void* cache, int64_t num_pages, int64_t heads, int64_t D, int64_t page);

namespace {

constexpr int kWarps = 4;
constexpr int kHeadsPerBlock = 4;
constexpr int ST_CACHE = 0xb01;
constexpr float kInf = __builtin_huge_valf();

template <int D>
struct DC {
  static constexpr int kSlabBytes = cache4_slab_bytes(D);
  // blocks an SM: at D = 128 registers without spills beat a fourth block (381 against 410 us)
  static constexpr int kResident = D == 128 ? 3 : 4;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kRing = kStages * kSlabBytes;
  static constexpr int kStride = D + 4;  // floats of a joined row
  static constexpr int kSmem = kWarps * kRing;
  static_assert(kSmem >= kWarps * 8 * kStride * 4, "the ring holds the warps' results at the end");
};

struct AttnParams {
  const void* q1;
  const void* q2;
  long long q_sb[2], q_sh[2];
  const uint8_t* cache;
  const int* table;
  const int* lengths;
  void* out;
  float* part;  // [b][head][chunk][kPart]
  long long table_stride;
  LambdaRef lam;
  int* status;
  unsigned long long timeout_ns;
  int num_pages;
  int width;
  int page_log2;
  int B;
  int heads;
  int kv_heads;
  int group;      // heads / kv_heads
  int head_blocks;
  int chunk;      // tokens of one block
  int n_chunks;
  float scale;    // softmax: log2(e) * scale
  float beta;
  float relu_power;
  int normalize;
};

// floats of one partial result: softmax {M1, l1, M2, l2, -, -, -, -, O1[D], O2[D]}, threshold O[D]
template <int D, bool THR>
__host__ __device__ constexpr int part_floats() {
  return THR ? D : 8 + 2 * D;
}

__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// d = a b + {c0, c1, c0, c1}
__device__ __forceinline__ void mma16816_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                              float c0, float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two nibbles as 1024 + n, and two more as 1024 + 16 n: (w & mask) | 0x6400 twice
// is one three-input operation, which takes one constant as an immediate; the
// other one comes from a register that the compiler may not fold back.
struct Magic {
  uint32_t base;
  __device__ __forceinline__ Magic() { asm volatile("mov.b32 %0, 0x64006400;" : "=r"(base)); }
  template <uint32_t kMask>
  __device__ __forceinline__ uint32_t take(uint32_t w) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(kMask), "r"(base));
    return r;
  }
  __device__ __forceinline__ uint32_t low(uint32_t w) const { return take<0x000f000fu>(w); }
  __device__ __forceinline__ uint32_t high(uint32_t w) const { return take<0x00f000f0u>(w); }
};
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// codes -7..7, and 16 times them
__device__ __forceinline__ uint32_t low_codes(const Magic& m, uint32_t w) { return sub_f16x2(m.low(w), 0x64086408u); }    // 1032
__device__ __forceinline__ uint32_t high_codes(const Magic& m, uint32_t w) { return sub_f16x2(m.high(w), 0x64806480u); }  // 1152

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ float scale_of(const uint32_t* w, int i) {
  const uint32_t x = w[i >> 1];
  return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
}

template <int PM>
__device__ __forceinline__ float relu_pow(float z, float p) {
  const float x = fmaxf(z, 0.0f);
  if constexpr (PM == POW_1) return x;
  if constexpr (PM == POW_2) return x * x;
  if constexpr (PM == POW_3) return x * x * x;
  return x > 0.0f ? fast_ex2(p * fast_lg2(x + 1e-10f)) : 0.0f;
}

// a map's part of the output; nothing was seen where the sum is zero
__device__ __forceinline__ float share(float o, float l) { return l == 0.0f ? 0.0f : o / l; }

__device__ __forceinline__ int length_of(const AttnParams& p, int b) { return max(0, min(p.lengths[b], p.width << p.page_log2)); }

template <bool F16>
__device__ __forceinline__ void write_out(const AttnParams& p, int b, int head, int D, int d, float y) {
  const long long at = (static_cast<long long>(b) * p.heads + head) * D + d;
  if constexpr (F16)
    static_cast<__half*>(p.out)[at] = __float2half_rn(y);
  else
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
}

// one (chunk, kv head x head block, request)
template <int D, bool THR, bool F16, int PM>
__global__ void __launch_bounds__(32 * kWarps, DC<D>::kResident) cache4_attn_kernel(const __grid_constant__ AttnParams p) {
  using C = DC<D>;
  constexpr int W = D / 32;  // groups
  constexpr bool kExactLow = THR && F16;
  constexpr int S = C::kStages;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t full[kWarps][S];
  __shared__ float s_m[kWarps][8], s_l[kWarps][8];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z;
  const int kvh = blockIdx.y / p.head_blocks, hb = blockIdx.y % p.head_blocks;
  const int len = length_of(p, b);
  const int lo = blockIdx.x * p.chunk, hi = min(len, lo + p.chunk);
  if (lo >= hi && !(blockIdx.x == 0 && p.n_chunks == 1)) return;
  const int head0 = kvh * p.group + hb * kHeadsPerBlock;
  const int n_heads = min(kHeadsPerBlock, p.group - hb * kHeadsPerBlock);
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full[warp][i], 1);
    if (warp == 0) abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const WaitCtl ctl = make_wait_ctl(&abort_flag, p.status, p.timeout_ns);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // this warp's slabs: tokens lo + 16 (i kWarps + warp)
  uint8_t* ring = ring_all + warp * C::kRing;
  const int* row = p.table + b * p.table_stride;
  const int n = max(0, (hi - lo - 16 * warp + 16 * kWarps - 1) / (16 * kWarps));
  const int page_mask = (1 << p.page_log2) - 1;
  auto token = [&](int i) { return lo + 16 * (i * kWarps + warp); };
  auto page_of = [&](int i) { return i < n ? __ldg(row + (token(i) >> p.page_log2)) : -1; };
  uint32_t in_cache = 0;  // bit i % 32: slab i's page lies in the cache
  const size_t page_bytes = p.kv_heads * cache4_block_bytes(page_mask + 1, D);
  const uint8_t* head_base = p.cache + kvh * cache4_block_bytes(page_mask + 1, D);
  auto fetch = [&](int i, int pg) {
    const bool good = static_cast<unsigned>(pg) < static_cast<unsigned>(p.num_pages);
    in_cache = (in_cache & ~(1u << (i & 31))) | (static_cast<uint32_t>(good) << (i & 31));
    if (lane == 0) {
      uint64_t* bar = &full[warp][i % S];
      if (good) {
        mbar_arrive_expect_tx(bar, C::kSlabBytes);
        bulk_load(ring + (i % S) * C::kSlabBytes, head_base + pg * page_bytes + ((token(i) & page_mask) >> 4) * C::kSlabBytes,
                  C::kSlabBytes, bar);
      } else {
        mbar_arrive(bar);  // nothing to copy: the phase completes all the same
      }
    }
  };
  {
    int pg[S - 1];
#pragma unroll
    for (int i = 0; i < S - 1; ++i) pg[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < n) fetch(i, pg[i]);
  }
  int next_page = page_of(S - 1);

  // queries: column g is head g % 4 of map g / 4; lane t holds dims 16 s + 4 t..
  uint32_t q1[2 * W][2], q2[2 * W][2];
  float off[W][2];  // of this lane's columns 2t, 2t + 1: minus the offset's share of a group's product
  float rq[2];      // what a column's product is multiplied by
  {
    const int m = g >> 2, j = g & 3;
    const bool live = j < n_heads;
    const char* base = static_cast<const char*>(m ? p.q2 : p.q1) + 2 * (b * p.q_sb[m] + (head0 + (live ? j : 0)) * p.q_sh[m]);
    float x[2 * W][4], ss = 0.f, top = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * W; ++s) {
      uint2 v = make_uint2(0u, 0u);
      if (live) v = *reinterpret_cast<const uint2*>(base + 2 * (16 * s + 4 * t));
      const float2 a = F16 ? unpack_f16x2(v.x) : unpack_bf16x2(v.x), c = F16 ? unpack_f16x2(v.y) : unpack_bf16x2(v.y);
      x[s][0] = a.x, x[s][1] = a.y, x[s][2] = c.x, x[s][3] = c.y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ss = fmaf(x[s][i], x[s][i], ss);
        top = fmaxf(top, fabsf(x[s][i]));
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    // 2^e <= top < 2^(e + 1): down = 2^(14 - e), up its inverse, both normal numbers for
    // any top; a query of zeros keeps its size
    const uint32_t e = top > 0.f ? min(max(__float_as_uint(top) >> 23, 15u), 252u) : 127u + 14u;
    const float up = __uint_as_float((e - 14u) << 23), down = __uint_as_float((268u - e) << 23);
    float sum[W];
#pragma unroll
    for (int s = 0; s < 2 * W; ++s) {
      const uint32_t a = pack_f16x2(x[s][0] * down, x[s][1] * down);
      const uint32_t c = pack_f16x2(x[s][2] * (down * 0.0625f), x[s][3] * (down * 0.0625f));
      q1[s][0] = m ? 0u : a;
      q1[s][1] = m ? 0u : c;
      q2[s][0] = m ? a : 0u;
      q2[s][1] = m ? c : 0u;
      const float2 ra = unpack_f16x2(a), rc = unpack_f16x2(c);
      const float add = (kExactLow ? 0.f : -1032.0f) * (ra.x + ra.y) - 1152.0f * (rc.x + rc.y);
      sum[s >> 1] = (s & 1) ? sum[s >> 1] + add : add;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
#pragma unroll
      for (int w = 0; w < W; ++w) sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], o);
    const float r = up * (THR ? (p.normalize ? 1.0f / fmaxf(sqrtf(ss), 1e-12f) : 1.0f) : p.scale);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int w = 0; w < W; ++w) off[w][c] = __shfl_sync(0xffffffffu, sum[w], 4 * (2 * t + c));
      rq[c] = __shfl_sync(0xffffffffu, r, 4 * (2 * t + c));
    }
  }
  const float tau = THR ? p.beta * sqrtf(2.0f * logf(static_cast<float>(max(len, 1))) / static_cast<float>(D)) : 0.f;
  const bool second = t >= 2;  // this lane's columns belong to map 2
  float lam[2] = {0.f, 0.f};   // threshold form: of the lane's two heads
  if constexpr (THR)
    for (int c = 0; c < 2; ++c)
      if (2 * (t & 1) + c < n_heads) lam[c] = fminf(fmaxf(lambda_at(p.lam, b, head0 + 2 * (t & 1) + c), 0.f), 1.f);

  float o[D / 16][4];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-kInf, -kInf}, l[2] = {0.f, 0.f};  // M and the sum of 2^(score - M), per column
  uint32_t bound = 0u;                                 // the largest scale so far, twice
  float limit[2] = {THR ? 0.f : -kInf, THR ? 0.f : -kInf}, down[2] = {1.f, 1.f};

  const Magic mg;
  auto low = [&](uint32_t w) { return kExactLow ? low_codes(mg, w) : mg.low(w); };  // K's low nibbles
  bool ok = true;
  int i = 0;
  for (; i < n; ++i) {
    ok = wait_inline_warp(&full[warp][i % S], (i / S) & 1, ctl, ST_CACHE);
    if (!ok) break;
    // every lane is done with slab i - 1: its stage takes slab i + S - 1
    if (i + S - 1 < n) {
      fetch(i + S - 1, next_page);
      next_page = page_of(i + S);
    }
    if (!((in_cache >> (i & 31)) & 1u)) continue;
    const uint8_t* slab = ring + (i % S) * C::kSlabBytes;
    const int tok = token(i);
    uint32_t vs[2][D / 64];
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    {
      uint32_t k[2][2][W], ks[2][D / 64];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_words(k[0][h], slab + cache4_codes_at(0, D) + cache4_k_word(g + 8 * h, t, 0, D));
        load_words(k[1][h], slab + cache4_codes_at(1, D) + cache4_k_word(g + 8 * h, t, 0, D));
        load_words(ks[h], slab + cache4_scales_at(0, D) + (second ? kSlab4 * cache4_scale_bytes(D) : 0) + (g + 8 * h) * cache4_scale_bytes(D));
        load_words(vs[h], slab + cache4_scales_at(2, D) + (g + 8 * h) * cache4_scale_bytes(D));
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float acc[4];
#pragma unroll
        for (int mp = 0; mp < 2; ++mp) {
          const uint32_t x = k[mp][0][w], y = k[mp][1][w], x8 = x >> 8, y8 = y >> 8;
          const uint32_t(&q)[2 * W][2] = mp ? q2 : q1;
          if (mp == 0)
            mma16816_from(acc, low(x), low(y), mg.high(x), mg.high(y), q[2 * w][0], q[2 * w][1], off[w][0], off[w][1]);
          else
            mma16816(acc, low(x), low(y), mg.high(x), mg.high(y), q[2 * w][0], q[2 * w][1]);
          mma16816(acc, low(x8), low(y8), mg.high(x8), mg.high(y8), q[2 * w + 1][0], q[2 * w + 1][1]);
        }
        const float s0 = scale_of(ks[0], w), s1 = scale_of(ks[1], w);
        s[0] = fmaf(acc[0], s0, s[0]);
        s[1] = fmaf(acc[1], s0, s[1]);
        s[2] = fmaf(acc[2], s1, s[2]);
        s[3] = fmaf(acc[3], s1, s[3]);
      }
    }
    if (tok + kSlab4 > hi) {  // rows past the length hold no token: their scales may be anything
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = tok + g + 8 * h < hi;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) vs[h][u] = in ? vs[h][u] : 0u;
        s[2 * h] = in ? s[2 * h] : -kInf;
        s[2 * h + 1] = in ? s[2 * h + 1] : -kInf;
      }
    }
    uint32_t big = bound;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < D / 64; ++u) big = max_bf16x2(big, vs[h][u]);
    float pr[4];
    if constexpr (THR) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        pr[x] = relu_pow<PM>(fmaf(s[x], rq[x & 1], -tau), p.relu_power);
        const float other = __shfl_xor_sync(0xffffffffu, pr[x], 2);  // the same head's other map
        pr[x] = second ? fmaf(-lam[x & 1], pr[x], other) : fmaf(-lam[x & 1], other, pr[x]);
      }
      if (!__any_sync(0xffffffffu, !(pr[0] == 0.f && pr[1] == 0.f && pr[2] == 0.f && pr[3] == 0.f))) continue;
    }
    float top[2];  // largest score (threshold: weight) of the lane's columns
#pragma unroll
    for (int c = 0; c < 2; ++c) top[c] = THR ? fmaxf(fabsf(pr[c]), fabsf(pr[2 + c])) : fmaxf(s[c], s[2 + c]) * rq[c];
    // M moves only when a weight passes it by 2^8: most slabs need neither the reductions nor the rescaling
    if (__any_sync(0xffffffffu, top[0] > limit[0] || top[1] > limit[1] || big != bound)) {
#pragma unroll
      for (int y = 1; y < 32; y <<= 1) big = max_bf16x2(big, __shfl_xor_sync(0xffffffffu, big, y));
      const float2 halves = unpack_bf16x2(big);
      const float largest = fmaxf(halves.x, halves.y);
      const float lb = largest > 0.f ? fast_lg2(fmaxf(largest, 0x1p-100f)) : 0.f;
      const float first = bound == 0u ? lb : 0.f;  // M bounds p alone so far
      bound = pack_bf16x2(largest, largest);
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = top[c];
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
        if constexpr (THR) {
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));  // a head's two columns hold one weight
          x = x > 0.f ? fast_lg2(x) : -kInf;
        }
        x = fmaxf(x + lb, m[c] + first);
        if constexpr (THR) x = x == -kInf ? x : fmaxf(x, -120.f);
        f[c] = m[c] == x ? 1.f : fast_ex2(m[c] - x);
        m[c] = x;
        l[c] *= f[c];
        limit[c] = THR ? (x == -kInf ? 0.f : fast_ex2(x + 8.f - lb)) : x + 8.f - lb;
        if constexpr (THR) down[c] = x == -kInf ? 1.f : fast_ex2(-x);
      }
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[x][y] *= f[y & 1];
    }
    if constexpr (THR) {
#pragma unroll
      for (int x = 0; x < 4; ++x) pr[x] *= down[x & 1];
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) pr[x] = fast_ex2(fmaf(s[x], rq[x & 1], -m[x & 1]));
      l[0] += pr[0] + pr[2];
      l[1] += pr[1] + pr[3];
    }
    uint32_t bf[W][2];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float s0 = scale_of(vs[0], w), s1 = scale_of(vs[1], w);
      const float x0 = pr[0] * s0, x1 = pr[1] * s0, x2 = pr[2] * s1, x3 = pr[3] * s1;
      uint32_t r0 = pack_f16x2(x0, x1), r1 = pack_f16x2(x2, x3);
      if constexpr (THR) {
        if (second) {
          const float2 h0 = unpack_f16x2(r0), h1 = unpack_f16x2(r1);
          r0 = pack_f16x2(x0 - h0.x, x1 - h0.y);
          r1 = pack_f16x2(x2 - h1.x, x3 - h1.y);
        }
      }
      bf[w][0] = movm(r0);
      bf[w][1] = movm(r1);
    }
    uint32_t v[4][D / 64];
    {
      const uint8_t* at = slab + cache4_codes_at(2, D) + lane * 16;
      const uint4 x = *reinterpret_cast<const uint4*>(at);
      if constexpr (D == 128) {
        const uint4 y = *reinterpret_cast<const uint4*>(at + 512);
        v[0][0] = x.x, v[0][1] = x.y, v[1][0] = x.z, v[1][1] = x.w;
        v[2][0] = y.x, v[2][1] = y.y, v[3][0] = y.z, v[3][1] = y.w;
      } else {
        v[0][0] = x.x, v[1][0] = x.y, v[2][0] = x.z, v[3][0] = x.w;
      }
    }
#pragma unroll
    for (int u = 0; u < D / 64; ++u)
#pragma unroll
      for (int y = 0; y < 2; ++y) {  // nibbles 0-3, 4-7 of every word
        const uint32_t a = __byte_perm(v[0][u], v[1][u], y ? 0x7632 : 0x5410), c = __byte_perm(v[2][u], v[3][u], y ? 0x7632 : 0x5410);
        const int mt = 4 * u + 2 * y;
        mma16816(o[mt], low_codes(mg, a), high_codes(mg, a), low_codes(mg, c), high_codes(mg, c), bf[mt >> 1][0], bf[mt >> 1][1]);
        mma16816(o[mt + 1], low_codes(mg, a >> 8), high_codes(mg, a >> 8), low_codes(mg, c >> 8), high_codes(mg, c >> 8), bf[mt >> 1][0], bf[mt >> 1][1]);
      }
  }
  if (!ok)
    for (int j = i; j < min(n, i + S - 1); ++j) tc::drain_wait(&full[warp][j % S], (j / S) & 1, ctl);

  // join the warps, through the ring's memory
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
  if (g == 0) {
    s_m[warp][2 * t] = m[0];
    s_m[warp][2 * t + 1] = m[1];
    s_l[warp][2 * t] = l[0];
    s_l[warp][2 * t + 1] = l[1];
  }
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(ring_all);
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    const int d = 32 * (mt >> 1) + 4 * g + 2 * (mt & 1);
    *reinterpret_cast<float2*>(s_o + (warp * 8 + 2 * t) * C::kStride + d) = make_float2(o[mt][0], o[mt][2] * 0.0625f);
    *reinterpret_cast<float2*>(s_o + (warp * 8 + 2 * t + 1) * C::kStride + d) = make_float2(o[mt][1], o[mt][3] * 0.0625f);
  }
  __syncthreads();
  constexpr int kPart = part_floats<D, THR>();
  for (int x = threadIdx.x; x < n_heads * D; x += 32 * kWarps) {
    const int j = x / D, d = x % D, head = head0 + j;
    float mm[2], ll[2], oo[2];
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      const int c = 4 * mp + j;
      float top = -kInf, sl = 0.f, so = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][c]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp that saw nothing adds its zeros; a threshold weight goes back to its own size
        const float f = s_m[w][c] == -kInf ? 1.f : fast_ex2(THR ? s_m[w][c] : s_m[w][c] - top);
        sl = fmaf(s_l[w][c], f, sl);
        so = fmaf(s_o[(w * 8 + c) * C::kStride + d], f, so);
      }
      mm[mp] = top;
      ll[mp] = sl;
      oo[mp] = so;
    }
    if (p.n_chunks == 1) {
      write_out<F16>(p, b, head, D, d, THR ? oo[0] + oo[1] : share(oo[0], ll[0]) - lambda_at(p.lam, b, head) * share(oo[1], ll[1]));
    } else {
      float* part = p.part + ((static_cast<long long>(b) * p.heads + head) * p.n_chunks + blockIdx.x) * kPart;
      if constexpr (THR) {
        part[d] = oo[0] + oo[1];
      } else {
        part[8 + d] = oo[0];
        part[8 + D + d] = oo[1];
        if (d == 0) *reinterpret_cast<float4*>(part) = make_float4(mm[0], ll[0], mm[1], ll[1]);
      }
    }
  }
}

// Joins a request's chunks: a block a head, G groups of 2 D threads (a map and a
// dim each) over every G-th chunk, then the groups in order.
// The chunks' weights 2^(M_c - M) are formed once, in shared memory, so that the
// sums are independent loads: a request of 74 chunks waits for memory a few times,
// not 74.
constexpr int kMaxChunks = 1024;

template <int D, bool THR, bool F16, int G>
__global__ void __launch_bounds__(2 * D * G) cache4_join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kThreads = 2 * D * G, kPart = part_floats<D, THR>();
  __shared__ float s_f[2][kMaxChunks];
  __shared__ float s_o[G][2][D];
  __shared__ float s_w[kThreads / 32][2];
  __shared__ float s_top[2], s_l[2];
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int grp = threadIdx.x / (2 * D), mp = threadIdx.x / D % 2, d = threadIdx.x % D;
  const int n = (length_of(p, b) + p.chunk - 1) / p.chunk;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float* part = p.part + (static_cast<long long>(b) * p.heads + head) * p.n_chunks * kPart;
  auto block_reduce = [&](float x, float y, bool max) {  // of a pair, into every thread by way of s_w
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, x, o), v = __shfl_xor_sync(0xffffffffu, y, o);
      x = max ? fmaxf(x, u) : x + u;
      y = max ? fmaxf(y, v) : y + v;
    }
    __syncthreads();
    if (lane == 0) {
      s_w[warp][0] = x;
      s_w[warp][1] = y;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      float r = s_w[0][threadIdx.x];
      for (int w = 1; w < kThreads / 32; ++w) r = max ? fmaxf(r, s_w[w][threadIdx.x]) : r + s_w[w][threadIdx.x];
      (max ? s_top : s_l)[threadIdx.x] = r;
    }
    __syncthreads();
  };
  if constexpr (!THR) {
    float m[2] = {-kInf, -kInf}, l[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < n; c += kThreads) {
      const float4 x = *reinterpret_cast<const float4*>(part + static_cast<long long>(c) * kPart);
      m[0] = fmaxf(m[0], x.x);
      m[1] = fmaxf(m[1], x.z);
    }
    block_reduce(m[0], m[1], true);
    for (int c = threadIdx.x; c < n; c += kThreads) {
      const float4 x = *reinterpret_cast<const float4*>(part + static_cast<long long>(c) * kPart);
      const float f0 = x.x == -kInf ? 0.f : fast_ex2(x.x - s_top[0]), f1 = x.z == -kInf ? 0.f : fast_ex2(x.z - s_top[1]);
      s_f[0][c] = f0;
      s_f[1][c] = f1;
      l[0] = fmaf(x.y, f0, l[0]);
      l[1] = fmaf(x.w, f1, l[1]);
    }
    block_reduce(l[0], l[1], false);
  }
  float o = 0.f;
  if constexpr (THR) {
    const float* at = part + d;
#pragma unroll 8
    for (int c = 2 * grp + mp; c < n; c += 2 * G) o += at[static_cast<long long>(c) * kPart];
  } else {
    const float* at = part + 8 + mp * D + d;
#pragma unroll 8
    for (int c = grp; c < n; c += G) o = fmaf(at[static_cast<long long>(c) * kPart], s_f[mp][c], o);
  }
  s_o[grp][mp][d] = o;
  __syncthreads();
  if (threadIdx.x < D) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      x += s_o[g][0][d];
      y += s_o[g][1][d];
    }
    write_out<F16>(p, b, head, D, d, THR ? x + y : share(x, s_l[0]) - lambda_at(p.lam, b, head) * share(y, s_l[1]));
  }
}

template <int D, bool THR, bool F16, int PM>
cudaError_t launch(const AttnParams& p, cudaStream_t s) {
  auto k = cache4_attn_kernel<D, THR, F16, PM>;
  if (cudaError_t e = allow_shared<cache4_attn_kernel<D, THR, F16, PM>>(DC<D>::kSmem)) return e;
  k<<<dim3(p.n_chunks, p.kv_heads * p.head_blocks, p.B), 32 * kWarps, DC<D>::kSmem, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.n_chunks == 1) return e;
  // the join's blocks start while the last chunks run and wait for the grid in front of them
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.heads, p.B);
  const bool many = p.n_chunks > 24;  // four groups: one request of 74 chunks 53 -> 33 us; 128 requests of 8 pay 40 us for them
  cfg.blockDim = dim3(2 * D * (many ? 4 : 1));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return many ? cudaLaunchKernelEx(&cfg, cache4_join_kernel<D, THR, F16, 4>, p) : cudaLaunchKernelEx(&cfg, cache4_join_kernel<D, THR, F16, 1>, p);
}

template <int D, bool F16>
cudaError_t dispatch(const AttnParams& p, bool thr, cudaStream_t s) {
  if (!thr) return launch<D, false, F16, POW_1>(p, s);
  switch (pow_mode_of(p.relu_power)) {
    case POW_1: return launch<D, true, F16, POW_1>(p, s);
    case POW_2: return launch<D, true, F16, POW_2>(p, s);
    case POW_3: return launch<D, true, F16, POW_3>(p, s);
    default: return launch<D, true, F16, POW_GENERAL>(p, s);
  }
}

// Tokens a block takes: one wave of resident blocks (3 an SM) where the table's
// width allows it, at least two slabs a warp, at most 1024, or 2048 where that
// still makes eight waves (uneven lengths then spread over the device: 32 requests
// of up to 8192 tokens and 16 heads take 158 us with 1024 and 164 with 2048, 128
// of up to 16384 and 8 heads 428 and 410), more only where the join could not hold
// the chunks of one request.
int64_t chunk_tokens(int64_t B, int64_t head_groups, int64_t max_len) {
  const int64_t want = 148 * 3 / (B * head_groups) + 1;  // chunks of one request
  int64_t chunk = ceil_div(ceil_div(max_len, want), 64) * 64;
  if (chunk < 128) chunk = 128;
  const int64_t cap = B * head_groups * ceil_div(max_len, 2048) >= 148 * 3 * 8 ? 2048 : 1024;
  if (chunk > cap) chunk = cap;
  const int64_t least = ceil_div(ceil_div(max_len, kMaxChunks), 64) * 64;
  return chunk < least ? least : chunk;
}

}  // namespace
}  // namespace tda

using namespace tda;

extern "C" {

size_t tda_cache4_workspace_size(int map, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 int64_t page_size, int64_t table_width) {
  // sizes that tda_cache4_attention refuses need none (and would divide by zero or overflow below)
  if (batch < 1 || batch > 65535 || kv_heads < 1 || heads < kv_heads || heads > 65535 || heads % kv_heads != 0) return 0;
  if (tda_cache4_block_bytes(page_size, head_dim) == 0 || table_width < 1 || table_width > 0x7fffffffll / page_size - 8) return 0;
  const int64_t hb = ceil_div(heads / kv_heads, kHeadsPerBlock);
  const int64_t max_len = table_width * page_size;
  const int64_t n = ceil_div(max_len, chunk_tokens(batch, kv_heads * hb, max_len));
  if (n <= 1) return 0;
  return static_cast<size_t>(batch * heads * n) * (map == 1 ? head_dim : 8 + 2 * head_dim) * sizeof(float);
}

int tda_cache4_attention(int map, const void* q1, const void* q2, int dtype, const int64_t* q_strides, void* out,
                         int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, const void* cache,
                         int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t table_stride,
                         int64_t table_width, const int32_t* lengths, const void* lambda, int lambda_dtype,
                         int64_t lambda_stride_b, int64_t lambda_stride_h, float lambda_value, float scale, float beta,
                         float relu_power, int normalize, void* workspace, size_t workspace_bytes, int* status,
                         void* stream) {
  if (map != TDA_MAP_SOFTMAX && map != TDA_MAP_THRESHOLD) return fail(TDA_ERR_INVALID, "map must be TDA_MAP_SOFTMAX or TDA_MAP_THRESHOLD");
  if (int e = cache4_check(cache, num_pages, kv_heads, head_dim, page_size)) return e;
  if (dtype != TDA_BF16 && dtype != TDA_F16) return fail(TDA_ERR_UNSUPPORTED, "queries must be TDA_BF16 or TDA_F16");
  if (batch < 1 || batch > 65535) return fail(TDA_ERR_INVALID, "batch must be in [1, 65535] (got %lld)", static_cast<long long>(batch));
  if (heads < kv_heads || heads % kv_heads != 0) return fail(TDA_ERR_INVALID, "kv heads must divide the query heads");
  if (heads > 65535) return fail(TDA_ERR_INVALID, "too many heads");
  if (!q1 || !q2 || !aligned(q1, 16) || !aligned(q2, 16) || !out || !aligned(out, 16))
    return fail(TDA_ERR_INVALID, "q1, q2 and out must be non-NULL and 16-byte aligned");
  if (!block_table || !lengths || !aligned(block_table, 4) || !aligned(lengths, 4))
    return fail(TDA_ERR_INVALID, "block_table and lengths must be non-NULL int32");
  if (table_width < 1 || table_stride < table_width) return fail(TDA_ERR_INVALID, "block table needs a width >= 1 and a stride >= the width");
  if (table_width > 0x7fffffffll / page_size - 8) return fail(TDA_ERR_INVALID, "table width * page_size must fit 31 bits");
  if (map == TDA_MAP_SOFTMAX && !(std::isfinite(scale) && scale > 0.f)) return fail(TDA_ERR_INVALID, "scale must be finite and positive");
  if (map == TDA_MAP_THRESHOLD && !(relu_power == relu_power)) return fail(TDA_ERR_INVALID, "relu_power is NaN");
  if (!status) return fail(TDA_ERR_INVALID, "status must point to a device int32");
  AttnParams p;
  p.status = status;
  p.timeout_ns = wait_timeout_ns();
  p.q1 = q1;
  p.q2 = q2;
  for (int i = 0; i < 2; ++i) {
    p.q_sb[i] = q_strides ? q_strides[2 * i] : heads * head_dim;
    p.q_sh[i] = q_strides ? q_strides[2 * i + 1] : head_dim;
    if (p.q_sb[i] < 0 || p.q_sh[i] <= 0 || (p.q_sb[i] | p.q_sh[i]) % 8 != 0)
      return fail(TDA_ERR_INVALID, "query strides must be positive multiples of 8 elements");
  }
  p.lam = LambdaRef{lambda, lambda_dtype, lambda_stride_b, lambda_stride_h, lambda_value};
  if (int e = check_lambda(p.lam)) return e;
  p.cache = static_cast<const uint8_t*>(cache);
  p.table = block_table;
  p.lengths = lengths;
  p.out = out;
  p.table_stride = table_stride;
  p.num_pages = static_cast<int>(num_pages);
  p.width = static_cast<int>(table_width);
  p.page_log2 = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  p.B = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(heads / kv_heads);
  p.head_blocks = static_cast<int>(ceil_div(p.group, kHeadsPerBlock));
  const int64_t max_len = table_width * page_size;
  p.chunk = static_cast<int>(chunk_tokens(batch, kv_heads * p.head_blocks, max_len));
  p.n_chunks = static_cast<int>(ceil_div(max_len, p.chunk));
  p.scale = scale * 1.4426950408889634f;
  p.beta = beta;
  p.relu_power = relu_power;
  p.normalize = normalize != 0;
  const size_t need = tda_cache4_workspace_size(map, batch, heads, kv_heads, head_dim, page_size, table_width);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(TDA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed", need);
  p.part = static_cast<float*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool thr = map == TDA_MAP_THRESHOLD, f16 = dtype == TDA_F16;
  cudaError_t e = head_dim == 64 ? (f16 ? dispatch<64, true>(p, thr, s) : dispatch<64, false>(p, thr, s))
                                 : (f16 ? dispatch<128, true>(p, thr, s) : dispatch<128, false>(p, thr, s));
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "cache attention launch");
}

}  // extern "C"
