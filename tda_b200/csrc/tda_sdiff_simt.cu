// Softmax differential attention on the CUDA cores: fp32 arithmetic for every
// type and head_dim 16-256, the path of fp32 inputs and of head dims that the
// tensor-core kernels do not take.  Also the row sums the backward starts from.
//
// One block takes a tile of BT rows (queries, or keys in the dk / dv kernel)
// and walks tiles of the other side; 256 threads as 16 x 16, each with R x R
// scores (R = BT / 16) from shared memory and R x D/16 accumulators.  Bound by
// fp32 FMA issue: a map's scores and its product with V are 2 D FMAs a visible
// pair, loads from shared memory are 8 of 16 bytes per 64 FMAs.  A training step
// at (2, 16 heads on 8, 1024, 64) takes 1.6 ms on B200 (24 TFLOP/s of executed
// products, FMA pipe 41-48% busy while an SM works); 8 x 4 scores a thread with half
// the threads took the same, two-wide FMAs 3-5% less from head_dim 32 and 14% more
// at 16.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tda_ptx.cuh"
#include "tda_sdiff.h"

namespace tda {
namespace {

constexpr float kInf = __builtin_huge_valf();

template <int D>
struct SC {
  static constexpr int BT = simt_tile_rows(D);
  static constexpr int R = BT / 16;
  static constexpr int LD = D + 4;       // row stride of a tile, floats
  static constexpr int LP = BT + 4;      // row stride of a weight tile
  static constexpr int C = D / 16;       // accumulator columns of a thread
  static constexpr int VEC = D >= 64 ? 4 : 1;
  static constexpr int kTile = BT * LD;
  static constexpr int kP = BT * LP;
  static constexpr int kFwdSmem = (3 * kTile + kP) * 4;
  static constexpr int kDqSmem = (4 * kTile + kP) * 4;
  static constexpr int kDkvSmem = (4 * kTile + 2 * kP + 2 * BT) * 4;
  // column of accumulator c of thread tx
  static __device__ __forceinline__ int col(int tx, int c) { return VEC == 4 ? (c >> 2) * 64 + tx * 4 + (c & 3) : tx + 16 * c; }
};

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_f16x2(v.x), b = unpack_f16x2(v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half_rn(x); }

// rows [r0, r0 + BT) of one head into shared memory as fp32, zeros from row `end`
template <typename T, int D>
__device__ __forceinline__ void load_tile(float* dst, const SdView& x, int b, int h, int r0, int end) {
  using C = SC<D>;
  const T* base = static_cast<const T*>(x.p) + b * x.sb + h * x.sh;
  for (int i = threadIdx.x; i < C::BT * (D / 4); i += 256) {
    const int r = i / (D / 4), c = (i % (D / 4)) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < end) v = load4(base + static_cast<long long>(r0 + r) * x.ss + c);
    *reinterpret_cast<float4*>(dst + r * C::LD + c) = v;
  }
}

// s[r][c] = a row (ty R + r) . b row (tx + 16 c)
template <int D>
__device__ __forceinline__ void dots(float (&s)[SC<D>::R][SC<D>::R], const float* a, const float* b, int ty, int tx) {
  using C = SC<D>;
#pragma unroll
  for (int r = 0; r < C::R; ++r)
#pragma unroll
    for (int c = 0; c < C::R; ++c) s[r][c] = 0.f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 x[C::R], y[C::R];
#pragma unroll
    for (int r = 0; r < C::R; ++r) x[r] = *reinterpret_cast<const float4*>(a + (ty * C::R + r) * C::LD + d);
#pragma unroll
    for (int c = 0; c < C::R; ++c) y[c] = *reinterpret_cast<const float4*>(b + (tx + 16 * c) * C::LD + d);
#pragma unroll
    for (int r = 0; r < C::R; ++r)
#pragma unroll
      for (int c = 0; c < C::R; ++c)
        s[r][c] = fmaf(x[r].x, y[c].x, fmaf(x[r].y, y[c].y, fmaf(x[r].z, y[c].z, fmaf(x[r].w, y[c].w, s[r][c]))));
  }
}

// o[r][:] += sum_j w[ty R + r][j] x[j][:].  A tile's sum is formed by itself and
// then added: thousands of products in one chain lose twice the bits that plain
// matrix products do.
template <int D>
__device__ __forceinline__ void accumulate(float (&sum)[SC<D>::R][SC<D>::C], const float* w, const float* x, int ty, int tx) {
  using C = SC<D>;
  float o[C::R][C::C];
#pragma unroll
  for (int r = 0; r < C::R; ++r)
#pragma unroll
    for (int c = 0; c < C::C; ++c) o[r][c] = 0.f;
#pragma unroll 2
  for (int j = 0; j < C::BT; j += 4) {
    float4 p[C::R];
#pragma unroll
    for (int r = 0; r < C::R; ++r) p[r] = *reinterpret_cast<const float4*>(w + (ty * C::R + r) * C::LP + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      float v[C::C];
      const float* row = x + (j + jj) * C::LD;
      if constexpr (C::VEC == 4) {
#pragma unroll
        for (int c = 0; c < C::C; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(row + C::col(tx, c));
          v[c] = f.x, v[c + 1] = f.y, v[c + 2] = f.z, v[c + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int c = 0; c < C::C; ++c) v[c] = row[C::col(tx, c)];
      }
#pragma unroll
      for (int r = 0; r < C::R; ++r) {
        const float q = jj == 0 ? p[r].x : jj == 1 ? p[r].y : jj == 2 ? p[r].z : p[r].w;
#pragma unroll
        for (int c = 0; c < C::C; ++c) o[r][c] = fmaf(q, v[c], o[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < C::R; ++r)
#pragma unroll
    for (int c = 0; c < C::C; ++c) sum[r][c] += o[r][c];
}

__device__ __forceinline__ int keys_of(const SdParams& p, int b) {
  return p.key_lengths ? max(0, min(p.key_lengths[b], p.Sk)) : p.Sk;
}
__device__ __forceinline__ bool sees(const SdParams& p, int i, int j, int n_keys) {
  return j < n_keys && (!p.causal || j <= i + p.Sk - p.Sq);
}
__device__ __forceinline__ long long row_at(const SdParams& p, int m, int b, int h, int i) {
  return ((static_cast<long long>(m) * p.B + b) * p.H + h) * p.Sq + i;
}

// -L of row i of map m and (batch, head) bh; its -D lies kTile behind
__device__ __forceinline__ long long table_at(const SdParams& p, int m, long long bh, int i) {
  return 2 * ((static_cast<long long>(m) * p.B * p.H + bh) * p.pad + i / kTile * kTile) + i % kTile;
}

// ================================================================== forward
template <typename T, int D>
__global__ void __launch_bounds__(256) sdiff_simt_fwd_kernel(const SdParams p) {
  using C = SC<D>;
  extern __shared__ float sm[];
  float *qs = sm, *ks = qs + C::kTile, *vs = ks + C::kTile, *ps = vs + C::kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n_t = (p.Sq + C::BT - 1) / C::BT;
  int bh, qt;
  tile_of_block(blockIdx.x, n_t, p.q_together, bh, qt);
  qt = n_t - 1 - qt;  // longest rows first
  const int b = bh / p.H, h = bh % p.H, kvh = h / p.group, i0 = qt * C::BT;
  int n_keys = keys_of(p, b);
  const int len = n_keys;
  if (p.causal) n_keys = max(0, min(n_keys, min(i0 + C::BT, p.Sq) + p.Sk - p.Sq));
  const float lam = lambda_at(p.lam, b, h);
  float o1[C::R][C::C], o[C::R][C::C];
  for (int m = 0; m < 2; ++m) {
    float top[C::R], sum[C::R];
#pragma unroll
    for (int r = 0; r < C::R; ++r) {
      top[r] = -kInf;
      sum[r] = 0.f;
#pragma unroll
      for (int c = 0; c < C::C; ++c) o[r][c] = 0.f;
    }
    __syncthreads();
    load_tile<T, D>(qs, p.q[m], b, h, i0, p.Sq);
    for (int j0 = 0; j0 < n_keys; j0 += C::BT) {
      __syncthreads();
      load_tile<T, D>(ks, p.k[m], b, kvh, j0, len);
      load_tile<T, D>(vs, p.v, b, kvh, j0, len);
      __syncthreads();
      float s[C::R][C::R];
      dots<D>(s, qs, ks, ty, tx);
#pragma unroll
      for (int r = 0; r < C::R; ++r) {
        float mx = top[r];
#pragma unroll
        for (int c = 0; c < C::R; ++c) {
          s[r][c] = sees(p, i0 + ty * C::R + r, j0 + tx + 16 * c, len) ? s[r][c] * p.c : -kInf;
          mx = fmaxf(mx, s[r][c]);
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float f = mx == top[r] ? 1.f : exp2f(top[r] - mx);
        const float base = mx == -kInf ? 0.f : mx;
        top[r] = mx;
        float part = 0.f;
#pragma unroll
        for (int c = 0; c < C::R; ++c) {
          s[r][c] = exp2f(s[r][c] - base);
          part += s[r][c];
          ps[(ty * C::R + r) * C::LP + tx + 16 * c] = s[r][c];
        }
        sum[r] = sum[r] * f + part;
#pragma unroll
        for (int c = 0; c < C::C; ++c) o[r][c] *= f;
      }
      __syncwarp();  // a row's weights come from, and go to, the 16 threads of its ty
      accumulate<D>(o, ps, vs, ty, tx);
      __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < C::R; ++r) {
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);
      const int i = i0 + ty * C::R + r;
      // keys, but -infinity for every score: no softmax, where a row without keys is zeros
      if (sum[r] == 0.f && sees(p, i, 0, len)) sum[r] = __uint_as_float(0x7fffffffu);
      const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];
      if (tx == 0 && i < p.Sq && p.lse) p.lse[row_at(p, m, b, h, i)] = sum[r] == 0.f ? kInf : top[r] + log2f(sum[r]);
      const long long at = row_at(p, 0, b, h, i) * D;
#pragma unroll
      for (int c = 0; c < C::C; ++c) {
        o[r][c] *= inv;
        if (m == 0) {
          o1[r][c] = o[r][c];
        } else if (i < p.Sq) {
          store1(static_cast<T*>(p.out) + at + C::col(tx, c), o1[r][c] - lam * o[r][c]);
          if (p.o12) {
            p.o12[at + C::col(tx, c)] = o1[r][c];
            p.o12[row_at(p, 1, b, h, i) * D + C::col(tx, c)] = o[r][c];
          }
        }
      }
    }
  }
}

// ================================================================== backward
// A number of one row of the product tables as three values of T and zeros.
template <typename T>
__device__ __forceinline__ void put_aux(uint8_t* table, int r, float x) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  int g = 0;
#pragma unroll
  for (int u = 0; u + 1 < aux_units(kF16); ++u) g += !(fabsf(x) >= aux_unit(kF16, u));
  float rest = x / aux_unit(kF16, g);
  if (kF16 && fabsf(rest) > 65504.0f) rest = __uint_as_float(0x7fffffffu);  // no fp16 values add up to it: not a wrong gradient in silence
  if (x == -kInf) rest = kF16 ? -65504.0f : -1e30f;  // a row without keys: what no score reaches
  float part[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    T v;
    store1(&v, rest);
    part[k] = static_cast<float>(v);
    rest -= part[k];
  }
  alignas(16) T column[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) store1(column + k, k / 3 == g && k / 3 < aux_units(kF16) ? part[k % 3] : 0.f);
  uint4* at = reinterpret_cast<uint4*>(table + (r >> 3) * 256 + (r & 7) * 16);
  at[0] = reinterpret_cast<uint4*>(column)[0];
  at[8] = reinterpret_cast<uint4*>(column)[1];
}

// D_1 = dout . O_1 and D_2 = dout . O_2, a warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) sdiff_delta_kernel(const SdParams p) {
  const long long rows = static_cast<long long>(p.B) * p.H * p.pad, all = static_cast<long long>(p.B) * p.H * p.Sq;
  const int lane = threadIdx.x & 31;
  constexpr int kLanes = D / 4 < 32 ? D / 4 : 32;
  constexpr int kPerWarp = 32 / kLanes;
  const long long warp = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const long long row = warp * kPerWarp + lane / kLanes;
  const int l = lane % kLanes;
  float a = 0.f, c = 0.f;
  const long long bh = row / p.pad;
  const int i = static_cast<int>(row % p.pad);
  const long long at = bh * p.Sq + i;
  if (row < rows && i < p.Sq) {
    const int h = static_cast<int>(bh % p.H), b = static_cast<int>(bh / p.H);
    const T* g = static_cast<const T*>(p.dout.p) + b * p.dout.sb + h * p.dout.sh + i * p.dout.ss;
#pragma unroll
    for (int d = 4 * l; d < D; d += 4 * kLanes) {
      const float4 x = load4(g + d), y = load4(p.o12 + at * D + d), z = load4(p.o12 + (all + at) * D + d);
      a += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
      c += x.x * z.x + x.y * z.y + x.z * z.z + x.w * z.w;
    }
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  // four lanes, a number each: -L_1, -D_1, -L_2, -D_2
  if (row < rows && l < 4) {
    const int m = l >> 1;
    const float x = l & 1 ? -(m ? c : a) : (i < p.Sq ? -p.lse[m * all + at] : -kInf);
    p.table[table_at(p, m, bh, i) + (l & 1) * kTile] = x;
    if constexpr (sizeof(T) == 2)
      if (p.aux)
        put_aux<T>(static_cast<uint8_t*>(p.aux) + ((m * rows + row) / kTile * 2 + (l & 1)) * kAuxTileBytes, static_cast<int>(row % kTile),
                   l & 1 ? x : x / p.c);
  }
}

// The numbers of sizes_of, after the tables are written: a block a tile of 128 rows
// of dout or v.  A maximum is the same in any order.  Infinities and NaN, which
// spoil what they enter anyway, do not take the others' bits.
template <int D>
__global__ void __launch_bounds__(256) sdiff_sizes_kernel(const SdParams p) {
  const int n_q = (p.Sq + kTile - 1) / kTile, n_k = (p.Sk + kTile - 1) / kTile;
  long long block = blockIdx.x;
  const bool values = block >= static_cast<long long>(p.B) * p.H * n_q;
  if (values) block -= static_cast<long long>(p.B) * p.H * n_q;
  const SdView& x = values ? p.v : p.dout;
  const int heads = values ? p.Hkv : p.H, tiles = values ? n_k : n_q;
  const int h = static_cast<int>(block / tiles % heads), b = static_cast<int>(block / tiles / heads);
  const int r0 = static_cast<int>(block % tiles) * kTile, end = min(r0 + kTile, values ? keys_of(p, b) : p.Sq);
  const __half* base = static_cast<const __half*>(x.p) + b * x.sb + h * x.sh + threadIdx.x % (D / 8) * 8;
  uint32_t top = 0;
#pragma unroll 4
  for (int r = r0 + threadIdx.x / (D / 8); r < end; r += 256 / (D / 8)) {
    const uint4 u = *reinterpret_cast<const uint4*>(base + r * x.ss);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = (i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w) & 0x7fff7fffu;
      top = __vmaxu2(top, m & ~__vcmpgeu2(m, 0x7c007c00u));
    }
  }
  __shared__ uint32_t part[8];
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) top = max(top, part[w]);
    if (top) atomicMax(sizes_of(p, b, values ? h : h / p.group) + values, top);
  }
}

// dlambda of one (batch, head): a fixed tree over its rows, the same sum every time
__global__ void __launch_bounds__(256) sdiff_dlam_kernel(const SdParams p) {
  __shared__ float part[256];
  const long long bh = blockIdx.x;
  float s = 0.f;
  for (int i = threadIdx.x; i < p.Sq; i += 256) s += p.table[table_at(p, 1, bh, i) + kTile];  // -D_2
  part[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.dlam[bh] = part[0];
}

// dq of one map and tile of queries
template <typename T, int D>
__global__ void __launch_bounds__(256) sdiff_simt_dq_kernel(const SdParams p) {
  using C = SC<D>;
  extern __shared__ float sm[];
  float *qs = sm, *gs = qs + C::kTile, *ks = gs + C::kTile, *vs = ks + C::kTile, *ps = vs + C::kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, m = blockIdx.y;
  const int n_t = (p.Sq + C::BT - 1) / C::BT;
  int bh, qt;
  tile_of_block(blockIdx.x, n_t, p.q_together, bh, qt);
  qt = n_t - 1 - qt;
  const int b = bh / p.H, h = bh % p.H, kvh = h / p.group, i0 = qt * C::BT;
  const int len = keys_of(p, b);
  int n_keys = len;
  if (p.causal) n_keys = max(0, min(n_keys, min(i0 + C::BT, p.Sq) + p.Sk - p.Sq));
  const float w = (m ? -lambda_at(p.lam, b, h) : 1.f) * p.scale;
  load_tile<T, D>(qs, p.q[m], b, h, i0, p.Sq);
  load_tile<T, D>(gs, p.dout, b, h, i0, p.Sq);
  float lse[C::R], del[C::R], o[C::R][C::C];
#pragma unroll
  for (int r = 0; r < C::R; ++r) {
    const int i = i0 + ty * C::R + r;
    const float* t = p.table + table_at(p, m, bh, min(i, p.Sq - 1));
    lse[r] = i < p.Sq ? -t[0] : kInf;
    del[r] = -t[kTile];
#pragma unroll
    for (int c = 0; c < C::C; ++c) o[r][c] = 0.f;
  }
  for (int j0 = 0; j0 < n_keys; j0 += C::BT) {
    __syncthreads();
    load_tile<T, D>(ks, p.k[m], b, kvh, j0, len);
    load_tile<T, D>(vs, p.v, b, kvh, j0, len);
    __syncthreads();
    float s[C::R][C::R], dp[C::R][C::R];
    dots<D>(s, qs, ks, ty, tx);
    dots<D>(dp, gs, vs, ty, tx);
#pragma unroll
    for (int r = 0; r < C::R; ++r)
#pragma unroll
      for (int c = 0; c < C::R; ++c) {
        const float pr = exp2f(fmaf(s[r][c], p.c, -lse[r]));
        const float dsx = pr * (dp[r][c] - del[r]);  // a lone key's is 0: its weight is 1 whatever its score, but for a NaN
        ps[(ty * C::R + r) * C::LP + tx + 16 * c] =
            sees(p, i0 + ty * C::R + r, j0 + tx + 16 * c, len) && !(len <= 1 && dsx == dsx) ? dsx : 0.f;
      }
    __syncwarp();
    accumulate<D>(o, ps, ks, ty, tx);
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < C::R; ++r) {
    const int i = i0 + ty * C::R + r;
    if (i >= p.Sq) continue;
#pragma unroll
    for (int c = 0; c < C::C; ++c)
      store1(static_cast<T*>(p.dq[m]) + row_at(p, 0, b, h, i) * D + C::col(tx, c), w * o[r][c]);
  }
}

// dk of both maps and dv of one tile of keys, over the group's query heads
template <typename T, int D>
__global__ void __launch_bounds__(256) sdiff_simt_dkv_kernel(const SdParams p) {
  using C = SC<D>;
  extern __shared__ float sm[];
  float *ks = sm, *vs = ks + C::kTile, *qs = vs + C::kTile, *gs = qs + C::kTile, *ps = gs + C::kTile, *ds = ps + C::kP,
        *ls = ds + C::kP, *es = ls + C::BT;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n_t = (p.Sk + C::BT - 1) / C::BT;
  int bh, j0;
  tile_of_block(blockIdx.x, n_t, p.k_together, bh, j0);
  j0 *= C::BT;
  const int b = bh / p.Hkv, kvh = bh % p.Hkv;
  const int len = keys_of(p, b);
  const int first = p.causal ? max(0, j0 - (p.Sk - p.Sq)) / C::BT * C::BT : 0;
  float dv[C::R][C::C], dk[C::R][C::C];
#pragma unroll
  for (int r = 0; r < C::R; ++r)
#pragma unroll
    for (int c = 0; c < C::C; ++c) dv[r][c] = 0.f;
  load_tile<T, D>(vs, p.v, b, kvh, j0, len);
  for (int m = 0; m < 2; ++m) {
    __syncthreads();
    load_tile<T, D>(ks, p.k[m], b, kvh, j0, len);
#pragma unroll
    for (int r = 0; r < C::R; ++r)
#pragma unroll
      for (int c = 0; c < C::C; ++c) dk[r][c] = 0.f;
    for (int h = kvh * p.group; h < (kvh + 1) * p.group && j0 < len; ++h) {
      const float w = m ? -lambda_at(p.lam, b, h) : 1.f;
      for (int i0 = first; i0 < p.Sq; i0 += C::BT) {
        __syncthreads();
        load_tile<T, D>(qs, p.q[m], b, h, i0, p.Sq);
        load_tile<T, D>(gs, p.dout, b, h, i0, p.Sq);
        if (threadIdx.x < C::BT) {
          const int i = i0 + threadIdx.x;
          const float* t = p.table + table_at(p, m, static_cast<long long>(b) * p.H + h, min(i, p.Sq - 1));
          ls[threadIdx.x] = i < p.Sq ? -t[0] : kInf;
          es[threadIdx.x] = -t[kTile];
        }
        __syncthreads();
        float s[C::R][C::R], dp[C::R][C::R];
        dots<D>(s, ks, qs, ty, tx);
        dots<D>(dp, vs, gs, ty, tx);
#pragma unroll
        for (int r = 0; r < C::R; ++r)
#pragma unroll
          for (int c = 0; c < C::R; ++c) {
            const int x = tx + 16 * c;
            const bool on = i0 + x < p.Sq && sees(p, i0 + x, j0 + ty * C::R + r, len);
            const float pr = on ? w * exp2f(fmaf(s[r][c], p.c, -ls[x])) : 0.f;
            ps[(ty * C::R + r) * C::LP + x] = pr;
            const float dsx = pr * (dp[r][c] - es[x]);
            ds[(ty * C::R + r) * C::LP + x] = on && !(len <= 1 && dsx == dsx) ? dsx : 0.f;  // a lone key's is 0, or NaN
          }
        __syncwarp();
        accumulate<D>(dv, ps, gs, ty, tx);
        accumulate<D>(dk, ds, qs, ty, tx);
      }
    }
#pragma unroll
    for (int r = 0; r < C::R; ++r) {
      const int j = j0 + ty * C::R + r;
      if (j >= p.Sk) continue;
      const long long at = ((static_cast<long long>(b) * p.Hkv + kvh) * p.Sk + j) * D;
#pragma unroll
      for (int c = 0; c < C::C; ++c) store1(static_cast<T*>(p.dk[m]) + at + C::col(tx, c), p.scale * dk[r][c]);
    }
  }
#pragma unroll
  for (int r = 0; r < C::R; ++r) {
    const int j = j0 + ty * C::R + r;
    if (j >= p.Sk) continue;
    const long long at = ((static_cast<long long>(b) * p.Hkv + kvh) * p.Sk + j) * D;
#pragma unroll
    for (int c = 0; c < C::C; ++c) store1(static_cast<T*>(p.dv) + at + C::col(tx, c), dv[r][c]);
  }
}

template <typename T, int D>
cudaError_t fwd(const SdParams& p, cudaStream_t s) {
  using C = SC<D>;
  if (cudaError_t e = allow_shared<sdiff_simt_fwd_kernel<T, D>>(C::kFwdSmem)) return e;
  const unsigned grid = static_cast<unsigned>(p.B * p.H * ceil_div(p.Sq, C::BT));
  sdiff_simt_fwd_kernel<T, D><<<grid, 256, C::kFwdSmem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t delta(const SdParams& p, cudaStream_t s) {
  const long long rows = static_cast<long long>(p.B) * p.H * p.pad;
  constexpr int kPerBlock = 8 * (32 / (D / 4 < 32 ? D / 4 : 32));
  sdiff_delta_kernel<T, D><<<static_cast<unsigned>(ceil_div(rows, kPerBlock)), 256, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if constexpr (std::is_same<T, __half>::value && (D == 64 || D == 128)) {
    if (e == cudaSuccess && p.aux) {
      const long long blocks = static_cast<long long>(p.B) * p.H * ceil_div(p.Sq, kTile) + static_cast<long long>(p.B) * p.Hkv * ceil_div(p.Sk, kTile);
      sdiff_sizes_kernel<D><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
      e = cudaGetLastError();
    }
  }
  if (e != cudaSuccess || !p.dlam) return e;
  sdiff_dlam_kernel<<<static_cast<unsigned>(p.B * p.H), 256, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t bwd(const SdParams& p, cudaStream_t s) {
  using C = SC<D>;
  if (cudaError_t e = allow_shared<sdiff_simt_dq_kernel<T, D>>(C::kDqSmem)) return e;
  if (cudaError_t e = allow_shared<sdiff_simt_dkv_kernel<T, D>>(C::kDkvSmem)) return e;
  sdiff_simt_dq_kernel<T, D><<<dim3(static_cast<unsigned>(p.B * p.H * ceil_div(p.Sq, C::BT)), 2), 256, C::kDqSmem, s>>>(p);
  if (cudaError_t e = cudaGetLastError()) return e;
  sdiff_simt_dkv_kernel<T, D><<<static_cast<unsigned>(p.B * p.Hkv * ceil_div(p.Sk, C::BT)), 256, C::kDkvSmem, s>>>(p);
  return cudaGetLastError();
}

#define TDA_SD_DIMS(fn, T)                 \
  switch (D) {                             \
    case 16: return fn<T, 16>(p, s);       \
    case 32: return fn<T, 32>(p, s);       \
    case 64: return fn<T, 64>(p, s);       \
    case 128: return fn<T, 128>(p, s);     \
    case 256: return fn<T, 256>(p, s);     \
    default: return cudaErrorInvalidValue; \
  }
#define TDA_SD_TYPES(fn)                               \
  if (dtype == TDA_F32) TDA_SD_DIMS(fn, float)         \
  if (dtype == TDA_BF16) TDA_SD_DIMS(fn, __nv_bfloat16) \
  if (dtype == TDA_F16) TDA_SD_DIMS(fn, __half)        \
  return cudaErrorInvalidValue;

}  // namespace

cudaError_t launch_sdiff_simt_fwd(const SdParams& p, int dtype, int D, cudaStream_t s) { TDA_SD_TYPES(fwd) }
cudaError_t launch_sdiff_simt_bwd(const SdParams& p, int dtype, int D, cudaStream_t s) { TDA_SD_TYPES(bwd) }
cudaError_t launch_sdiff_delta(const SdParams& p, int dtype, int D, cudaStream_t s) { TDA_SD_TYPES(delta) }

}  // namespace tda
