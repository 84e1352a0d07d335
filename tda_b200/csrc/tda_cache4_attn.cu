// Attention of one new token a request over the 4-bit paged cache.
//
//   softmax form:    out = (softmax(c q1 K1^T) - lambda softmax(c q2 K2^T)) V
//   threshold form:  out = (P1 - clamp(lambda) P2) V, P_m = relu(qh_m Kh_m^T - tau)^p,
//                    tau = beta sqrt(2 ln(len) / D), qh = q / max(|q|, 1e-12) with a cache of normalized keys
//
// Bound by the cache bytes: 3 (D/2 + D/16) a token and kv head (216 at D = 128).
// A warp takes slabs of 16 tokens straight from global memory, the next slab's
// loads in flight while it computes on one: K rows and V rows are stored in
// the order of matrix fragments (tda_cache4.cuh), so nothing passes through
// shared memory.  The products are m16n8k16 with the cache as the A operand
// and 8 columns of queries: up to 4 heads of the kv head's group times the two
// maps, so that both maps share one pass over V:
//   S^T (16 tokens x 8) = K Q^T       a lane keeps the product of its columns' map
//   O^T (D x 8) += V^T (P s)^T
// Codes become 16-bit floats by the exponent trick: (word >> 4i) & 0x000f000f
// | magic is 128 + n (bf16) or 1024 + n (fp16), n = code + 8.  For K the
// product starts from -(136 or 1032) times the sum of the group's q, which
// removes the offset without an instruction (the cancelled part is exact
// products summed in fp32: an error near 1e-5 of |q| times a code unit).  V
// subtracts it (exact).  K's scale multiplies a group's fp32 product, V's
// scale the weight.  Weights round to bf16.  Softmax: bf16(p s), 2^-9 of a
// weight, far below the 2^-4 of a code.  The threshold form knows its whole
// weight w = (p1 - lambda p2) s at once, which takes the columns of one map, so
// the other four carry what rounding w left: 2^-17, and nothing is lost where
// the two maps cancel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "tda_cache4.cuh"
#include "tda_host.h"
#include "tda_ptx.cuh"

namespace tda {

int cache4_check(const void* cache, int64_t num_pages, int64_t heads, int64_t D, int64_t page);

namespace {

constexpr int kWarps = 4;
constexpr int kSlab = 16;
constexpr int kHeadsPerBlock = 4;

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
  long long num_pages;
  LambdaRef lam;
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

// floats of one partial result: softmax {m1, l1, m2, l2, -, -, -, -, O1[D], O2[D]}, threshold O[D]
template <int D, bool THR>
__host__ __device__ constexpr int part_floats() {
  return THR ? D : 8 + 2 * D;
}

__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, float c0, float c1, float c2, float c3) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

template <bool F16>
__device__ __forceinline__ uint32_t widen(uint32_t w, int i) {
  return ((w >> (4 * i)) & 0x000f000fu) | (F16 ? 0x64006400u : 0x43004300u);
}

// 128 + n -> n - 8, exact in bf16
__device__ __forceinline__ uint32_t widen_v(uint32_t w, int i) {
  const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x43084308u));
  return r;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (N == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

__device__ __forceinline__ float scale_of(const uint32_t* w, int i) {
  const uint32_t x = w[i >> 1];
  return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
}

template <int D>
struct Slab {
  uint32_t k[2][2][D / 32];  // map, row g / g + 8
  uint32_t v[4][D / 64];     // tokens 2t, 2t+1, 2t+8, 2t+9
  uint32_t ks[2][D / 64];    // K scales of the lane's map, rows g / g + 8
  uint32_t vs[2][D / 64];
  bool ok;                   // the page lies in the cache
};

template <int D>
__device__ __forceinline__ void load_slab(Slab<D>& s, const AttnParams& p, const int* row, int kvh, int tok, int len,
                                          int g, int t) {
  if (tok >= len) return;
  const int page = 1 << p.page_log2;
  const int pg = __ldg(row + (tok >> p.page_log2));
  s.ok = pg >= 0 && pg < p.num_pages;
  if (!s.ok) return;
  const uint8_t* blk = p.cache + (static_cast<size_t>(pg) * p.kv_heads + kvh) * cache4_block_bytes(page, D);
  const int r0 = tok & (page - 1);
  const int rb = static_cast<int>(cache4_row_bytes(D)), sb = static_cast<int>(cache4_scale_bytes(D));
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      load_words(s.k[m][h], blk + cache4_codes_at(m, page, D) + (r0 + g + 8 * h) * rb + t * (D / 8));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load_words(s.ks[h], blk + cache4_scales_at(t >> 1, page, D) + (r0 + g + 8 * h) * sb);
    load_words(s.vs[h], blk + cache4_scales_at(2, page, D) + (r0 + g + 8 * h) * sb);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    load_words(s.v[i], blk + cache4_codes_at(2, page, D) + (r0 + 2 * t + (i & 1) + 8 * (i >> 1)) * rb + g * (D / 16));
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

// one (chunk, kv head x head block, request)
template <int D, bool THR, bool F16, int PM>
__global__ void __launch_bounds__(32 * kWarps) cache4_attn_kernel(const AttnParams p) {
  constexpr int W = D / 32;   // groups
  constexpr int kStride = D + 4;
  __shared__ float s_m[kWarps][8], s_l[kWarps][8];
  __shared__ float s_o[kWarps][8][kStride];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z;
  const int kvh = blockIdx.y / p.head_blocks, hb = blockIdx.y % p.head_blocks;
  const int len = max(0, min(p.lengths[b], p.width << p.page_log2));
  const int lo = blockIdx.x * p.chunk, hi = min(len, lo + p.chunk);
  if (lo >= hi && !(blockIdx.x == 0 && p.n_chunks == 1)) return;
  const int head0 = kvh * p.group + hb * kHeadsPerBlock;
  const int n_heads = min(kHeadsPerBlock, p.group - hb * kHeadsPerBlock);

  // queries: column g is head g % 4 of map g / 4; lane t holds dims 16 s + 4 t..
  uint32_t q[2 * W][2];
  float qsum[W][2];  // of this lane's columns 2t, 2t + 1, times the offset
  float rq[2] = {1.f, 1.f};
  {
    const int m = g >> 2, j = g & 3;
    const bool live = j < n_heads;
    const char* base = static_cast<const char*>(m ? p.q2 : p.q1) +
                       2 * (b * p.q_sb[m] + (head0 + (live ? j : 0)) * p.q_sh[m]);
    float sum[W], ss = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * W; ++s) {
      uint2 v = make_uint2(0u, 0u);
      if (live) v = *reinterpret_cast<const uint2*>(base + 2 * (16 * s + 4 * t));
      q[s][0] = v.x;
      q[s][1] = v.y;
      const float2 x = F16 ? unpack_f16x2(v.x) : unpack_bf16x2(v.x), y = F16 ? unpack_f16x2(v.y) : unpack_bf16x2(v.y);
      const float add = (x.x + x.y) + (y.x + y.y);
      sum[s >> 1] = (s & 1) ? sum[s >> 1] + add : add;
      ss = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(y.x, y.x, fmaf(y.y, y.y, ss))));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
#pragma unroll
      for (int w = 0; w < W; ++w) sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], o);
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    const float r = p.normalize ? 1.0f / fmaxf(sqrtf(ss), 1e-12f) : 1.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int w = 0; w < W; ++w) qsum[w][c] = (F16 ? -1032.0f : -136.0f) * __shfl_sync(0xffffffffu, sum[w], 4 * (2 * t + c));
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
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int* row = p.table + b * p.table_stride;

  Slab<D> cur, nxt;
  cur.ok = nxt.ok = false;
  int tok = lo + warp * kSlab;
  load_slab(cur, p, row, kvh, tok, hi, g, t);
  for (; tok < hi; tok += kWarps * kSlab) {
    nxt.ok = false;
    load_slab(nxt, p, row, kvh, tok + kWarps * kSlab, hi, g, t);
    if (cur.ok) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float acc[2][4];
#pragma unroll
        for (int mp = 0; mp < 2; ++mp) {
          const uint32_t x = cur.k[mp][0][w], y = cur.k[mp][1][w];
          mma16816<F16>(acc[mp], widen<F16>(x, 0), widen<F16>(y, 0), widen<F16>(x, 1), widen<F16>(y, 1), q[2 * w][0],
                        q[2 * w][1], qsum[w][0], qsum[w][1], qsum[w][0], qsum[w][1]);
          mma16816<F16>(acc[mp], widen<F16>(x, 2), widen<F16>(y, 2), widen<F16>(x, 3), widen<F16>(y, 3),
                        q[2 * w + 1][0], q[2 * w + 1][1], acc[mp][0], acc[mp][1], acc[mp][2], acc[mp][3]);
        }
        const float s0 = scale_of(cur.ks[0], w), s1 = scale_of(cur.ks[1], w);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(second ? acc[1][i] : acc[0][i], i < 2 ? s0 : s1, s[i]);
      }
      const bool in0 = tok + g < hi, in1 = tok + g + 8 < hi;
      float pr[4];
      if constexpr (THR) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = fmaf(s[i], rq[i & 1], -tau);
          pr[i] = (i < 2 ? in0 : in1) ? relu_pow<PM>(z, p.relu_power) : 0.f;
          const float other = __shfl_xor_sync(0xffffffffu, pr[i], 2);  // the same head's other map
          pr[i] = second ? fmaf(-lam[i & 1], pr[i], other) : fmaf(-lam[i & 1], other, pr[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = (i < 2 ? in0 : in1) ? s[i] * p.scale : -INFINITY;
        // the running maximum moves only when a score passes it by 2^8: weights stay below 256
        // and most slabs need neither the reduction nor the rescaling
        const bool grow = fmaxf(s[0], s[2]) > m[0] + 8.f || fmaxf(s[1], s[3]) > m[1] + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          float n0 = fmaxf(s[0], s[2]), n1 = fmaxf(s[1], s[3]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
          }
          n0 = fmaxf(n0, m[0]);
          n1 = fmaxf(n1, m[1]);
          const float f0 = m[0] == n0 ? 1.f : fast_ex2(m[0] - n0), f1 = m[1] == n1 ? 1.f : fast_ex2(m[1] - n1);
          m[0] = n0;
          m[1] = n1;
          l[0] *= f0;
          l[1] *= f1;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[i][0] *= f0;
            o[i][2] *= f0;
            o[i][1] *= f1;
            o[i][3] *= f1;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = fast_ex2(s[i] - m[i & 1]);
        l[0] += pr[0] + pr[2];
        l[1] += pr[1] + pr[3];
      }
      bool work = true;
      if constexpr (THR) work = __any_sync(0xffffffffu, !(pr[0] == 0.f && pr[1] == 0.f && pr[2] == 0.f && pr[3] == 0.f));
      if (work) {
        uint32_t bf[W][2];
#pragma unroll
        for (int w = 0; w < W; ++w) {
          // rows past the length hold no token: their scales may be anything
          const float s0 = in0 ? scale_of(cur.vs[0], w) : 0.f, s1 = in1 ? scale_of(cur.vs[1], w) : 0.f;
          uint32_t r0 = pack_bf16x2(pr[0] * s0, pr[1] * s0), r1 = pack_bf16x2(pr[2] * s1, pr[3] * s1);
          if constexpr (THR) {
            if (second) {
              const float2 h0 = unpack_bf16x2(r0), h1 = unpack_bf16x2(r1);
              r0 = pack_bf16x2(pr[0] * s0 - h0.x, pr[1] * s0 - h0.y);
              r1 = pack_bf16x2(pr[2] * s1 - h1.x, pr[3] * s1 - h1.y);
            }
          }
          bf[w][0] = movm(r0);
          bf[w][1] = movm(r1);
        }
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          uint32_t a[2], c[2];
          a[0] = __byte_perm(cur.v[0][u], cur.v[1][u], 0x5410);
          a[1] = __byte_perm(cur.v[0][u], cur.v[1][u], 0x7632);
          c[0] = __byte_perm(cur.v[2][u], cur.v[3][u], 0x5410);
          c[1] = __byte_perm(cur.v[2][u], cur.v[3][u], 0x7632);
#pragma unroll
          for (int mm = 0; mm < 4; ++mm) {
            const int n = 2 * (mm & 1), x = mm >> 1, mt = 4 * u + mm;
            mma16816<false>(o[mt], widen_v(a[x], n), widen_v(a[x], n + 1), widen_v(c[x], n), widen_v(c[x], n + 1),
                            bf[mt >> 1][0], bf[mt >> 1][1], o[mt][0], o[mt][1], o[mt][2], o[mt][3]);
          }
        }
      }
    }
    cur = nxt;
  }

  // join the warps
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
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    const int d = 32 * (mt >> 1) + 4 * g + 2 * (mt & 1);
    *reinterpret_cast<float2*>(&s_o[warp][2 * t][d]) = make_float2(o[mt][0], o[mt][2]);
    *reinterpret_cast<float2*>(&s_o[warp][2 * t + 1][d]) = make_float2(o[mt][1], o[mt][3]);
  }
  __syncthreads();
  constexpr int kPart = part_floats<D, THR>();
  for (int i = threadIdx.x; i < n_heads * D; i += 32 * kWarps) {
    const int j = i / D, d = i % D, head = head0 + j;
    float mm[2], ll[2], oo[2];
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      const int c = 4 * mp + j;
      float top = -INFINITY, sl = 0.f, so = 0.f;
      if constexpr (!THR)
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][c]);
      for (int w = 0; w < kWarps; ++w) {
        const float f = THR ? 1.f : (s_m[w][c] == -INFINITY ? 0.f : fast_ex2(s_m[w][c] - top));
        // a warp without a token adds nothing, whatever its sums are (they are zeros)
        sl = fmaf(s_l[w][c], f, sl);
        so = fmaf(s_o[w][c][d], f, so);
      }
      mm[mp] = top;
      ll[mp] = sl;
      oo[mp] = so;
    }
    if (p.n_chunks == 1) {
      float y;
      if constexpr (THR)
        y = oo[0] + oo[1];
      else
        y = share(oo[0], ll[0]) - lambda_at(p.lam, b, head) * share(oo[1], ll[1]);
      const long long at = (static_cast<long long>(b) * p.heads + head) * D + d;
      if constexpr (F16)
        static_cast<__half*>(p.out)[at] = __float2half_rn(y);
      else
        static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
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

// Joins a request's chunks, in order: out of one head a block of D threads.
template <int D, bool THR, bool F16>
__global__ void __launch_bounds__(D) cache4_join_kernel(const AttnParams p) {
  const int head = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int len = max(0, min(p.lengths[b], p.width << p.page_log2));
  const int n = (len + p.chunk - 1) / p.chunk;
  constexpr int kPart = part_floats<D, THR>();
  const float* part = p.part + (static_cast<long long>(b) * p.heads + head) * p.n_chunks * kPart;
  float y = 0.f;
  if constexpr (THR) {
    for (int c = 0; c < n; ++c) y += part[static_cast<long long>(c) * kPart + d];
  } else if (n > 0) {
    float top[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2] = {0.f, 0.f};
    for (int c = 0; c < n; ++c) {
      const float* q = part + static_cast<long long>(c) * kPart;
      const float4 s = *reinterpret_cast<const float4*>(q);
#pragma unroll
      for (int mp = 0; mp < 2; ++mp) {
        const float mc = mp ? s.z : s.x, lc = mp ? s.w : s.y, oc = q[8 + mp * D + d];
        const float nt = fmaxf(top[mp], mc);
        const float f = top[mp] == -INFINITY ? 0.f : fast_ex2(top[mp] - nt), h = mc == -INFINITY ? 0.f : fast_ex2(mc - nt);
        l[mp] = l[mp] * f + lc * h;
        o[mp] = o[mp] * f + oc * h;
        top[mp] = nt;
      }
    }
    y = share(o[0], l[0]) - lambda_at(p.lam, b, head) * share(o[1], l[1]);
  }
  const long long at = (static_cast<long long>(b) * p.heads + head) * D + d;
  if constexpr (F16)
    static_cast<__half*>(p.out)[at] = __float2half_rn(y);
  else
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
}

template <int D, bool THR, bool F16, int PM>
cudaError_t launch(const AttnParams& p, cudaStream_t s) {
  const dim3 grid(p.n_chunks, p.kv_heads * p.head_blocks, p.B);
  cache4_attn_kernel<D, THR, F16, PM><<<grid, 32 * kWarps, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.n_chunks == 1) return e;
  cache4_join_kernel<D, THR, F16><<<dim3(p.heads, p.B), D, 0, s>>>(p);
  return cudaGetLastError();
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

// Tokens a block takes.  Enough blocks to fill the device a few times when the
// table allows it, and at least 64 tokens (a slab a warp).
int64_t chunk_tokens(int64_t B, int64_t head_groups, int64_t max_len) {
  const int64_t want = 148 * 8 / (B * head_groups) + 1;  // chunks of one request
  int64_t chunk = ceil_div(ceil_div(max_len, want), 64) * 64;
  if (chunk < 128) chunk = 128;
  if (chunk > 1024) chunk = 1024;
  return chunk;
}

}  // namespace
}  // namespace tda

using namespace tda;

extern "C" {

size_t tda_cache4_workspace_size(int map, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 int64_t page_size, int64_t table_width) {
  if (batch < 1 || kv_heads < 1 || heads % kv_heads != 0 || table_width < 1) return 0;
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
                         float relu_power, int normalize, void* workspace, size_t workspace_bytes, void* stream) {
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
  AttnParams p;
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
  p.num_pages = num_pages;
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
