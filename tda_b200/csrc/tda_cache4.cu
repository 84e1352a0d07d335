// The 4-bit paged cache: page plan of a serving step, append (quantise and
// scatter) and read (gather and widen), with their C entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tda_cache4.cuh"
#include "tda_host.h"

namespace tda {
namespace {

// ================================================================== page plan
// Request r holds len[r] tokens in ceil(len / page) pages and gets new[r] more.
// Pages wanted are handed out in request order from free[head..]; a request
// that the list cannot serve keeps what it got and drops its last tokens, and so
// does one whose tokens pass the last row: a token without a row is never written,
// so it takes no page and no length counts it.
struct PlanParams {
  const int* lengths;
  const int* added;
  int* table;
  const int* free_pages;
  const int* free_head;
  int* slots;
  int* positions;
  int* requests;
  int* starts;
  int* lengths_out;
  int* free_head_out;
  int* dropped;
  long long table_stride;
  int B;
  int width;
  int n_free;
  int page;
  int rows;
};

constexpr int kPlanThreads = 512;
constexpr int kPlanScan = 2048;   // requests scanned at a time
constexpr int kPlanRows = 2048;   // token rows of one block

// Counts are added up to 2^31 - 1 and stay there: new_tokens may sum to more, and
// a wrapped sum would place rows and pages in front of their arrays.  Capped
// addition of non-negative numbers is associative, so a scan may use it.
__device__ __forceinline__ int add_capped(int a, int b) {
  return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), 0x7fffffffu));
}

// Exclusive prefix sum of a over the block and its total, capped.
__device__ void block_scan(int& a, int& total, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o);
    if (lane >= o) a = add_capped(a, x);
  }
  if (lane == 31) warp_sums[warp] = a;
  a = __shfl_up_sync(0xffffffffu, a, 1);
  if (lane == 0) a = 0;
  __syncthreads();
  int front = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) front = add_capped(front, warp_sums[w]);
    total = add_capped(total, warp_sums[w]);
  }
  a = add_capped(a, front);
  __syncthreads();
}

// Sum of x over the block, in thread 0.
__device__ long long block_sum(long long x, long long* warp_sums) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < kPlanThreads / 32; ++w) x += warp_sums[w];
  __syncthreads();
  return x;
}

// Every block scans all requests (a few KB from L2) and then writes its own
// rows, so the plan is one launch: 512 requests and 1 M rows take 18 us, 256
// requests of one token what a launch takes.  The table entries of request r are written
// by block r % gridDim.x; rows take fresh pages from the free list itself, so
// no block reads an entry that another one writes.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const PlanParams p) {
  __shared__ int s_start[kPlanScan + 1], s_first[kPlanScan], s_len[kPlanScan], s_after[kPlanScan],
      s_got[kPlanScan];
  __shared__ int warp_sums[kPlanThreads / 32];
  __shared__ long long warp_totals[kPlanThreads / 32];
  const int tid = threadIdx.x;
  const int head = max(0, *p.free_head);
  const int left = max(0, p.n_free - head);
  const long long row0 = static_cast<long long>(blockIdx.x) * kPlanRows;
  const int row_end = static_cast<int>(min(static_cast<long long>(p.rows), row0 + kPlanRows));
  int base_tok = 0, base_page = 0;
  long long lost = 0, taken = 0;  // of this thread's requests: tokens without a place, pages handed out
  constexpr int kPer = kPlanScan / kPlanThreads;
  for (int r0 = 0; r0 < p.B; r0 += kPlanScan) {
    const int n = min(kPlanScan, p.B - r0);
    int add[kPer], fits[kPer], want[kPer], held[kPer], sa = 0, sw = 0, ta, tw;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = tid * kPer + i;
      add[i] = r < n ? max(0, p.added[r0 + r]) : 0;
      sa = add_capped(sa, add[i]);
    }
    block_scan(sa, ta, warp_sums);
    sa = add_capped(sa, base_tok);
    int start = sa;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = tid * kPer + i;
      fits[i] = want[i] = held[i] = 0;
      if (r < n) {
        const int len = max(0, min(p.lengths[r0 + r], p.width * p.page));  // a table holds no more
        fits[i] = min(add[i], max(0, p.rows - start));  // tokens that have a row
        held[i] = (len + p.page - 1) / p.page;
        const long long last = (static_cast<long long>(len) + fits[i] + p.page - 1) / p.page;
        want[i] = static_cast<int>(min(last, static_cast<long long>(p.width))) - held[i];
        s_len[r] = len;
      }
      start = add_capped(start, add[i]);
      sw = add_capped(sw, want[i]);
    }
    block_scan(sw, tw, warp_sums);
    sw = add_capped(sw, base_page);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = tid * kPer + i;
      if (r < n) {
        const int got = min(want[i], max(0, left - sw));
        const int len = s_len[r];
        const int after = static_cast<int>(min(static_cast<long long>(len) + fits[i],
                                               static_cast<long long>(held[i] + got) * p.page));
        s_start[r] = sa;
        s_first[r] = sw;
        s_after[r] = after;
        s_got[r] = got;
        lost += static_cast<long long>(add[i]) - (after - len);
        taken += got;
        if (blockIdx.x == 0) {
          p.starts[r0 + r] = sa;
          p.lengths_out[r0 + r] = after;
        }
      }
      sa = add_capped(sa, add[i]);
      sw = add_capped(sw, want[i]);
    }
    base_tok = add_capped(base_tok, ta);
    base_page = add_capped(base_page, tw);
    if (tid == 0) s_start[n] = base_tok;
    __syncthreads();
    // fresh table entries: a warp a request
    for (int r = blockIdx.x + (tid >> 5) * gridDim.x; r < n; r += gridDim.x * (kPlanThreads / 32)) {
      const int held0 = (s_len[r] + p.page - 1) / p.page;
      for (int c = tid & 31; c < s_got[r]; c += 32)
        p.table[(r0 + r) * p.table_stride + held0 + c] = p.free_pages[head + s_first[r] + c];
    }
    // rows of these requests that belong to this block
    const int lo = min(max(static_cast<int>(row0), s_start[0]), row_end), hi = min(row_end, s_start[n]);
    for (int i = lo + tid; i < hi; i += kPlanThreads) {
      int a = 0, b = n - 1;  // last request whose start is <= i
      while (a < b) {
        const int m = (a + b + 1) >> 1;
        if (s_start[m] <= i)
          a = m;
        else
          b = m - 1;
      }
      const int len = s_len[a], pos = len + (i - s_start[a]);
      int slot = -1;
      if (pos < s_after[a]) {
        const int held0 = (len + p.page - 1) / p.page, c = pos / p.page;
        const int pg = c < held0 ? p.table[(r0 + a) * p.table_stride + c] : p.free_pages[head + s_first[a] + c - held0];
        slot = pg * p.page + pos % p.page;
      }
      p.slots[i] = slot;
      p.positions[i] = pos;
      p.requests[i] = r0 + a;
    }
    __syncthreads();
  }
  for (int i = min(max(static_cast<int>(row0), base_tok), row_end) + tid; i < row_end; i += kPlanThreads)
    p.slots[i] = p.positions[i] = p.requests[i] = -1;
  if (blockIdx.x == 0) {
    lost = block_sum(lost, warp_totals);
    taken = block_sum(taken, warp_totals);
    if (tid == 0) {
      p.starts[p.B] = base_tok;
      *p.free_head_out = head + static_cast<int>(taken);
      *p.dropped = static_cast<int>(min(lost, 0x7fffffffll));
    }
  }
}

// byte offset of the slab that holds a slot's rows of one head
template <int D>
__device__ __forceinline__ size_t slab_of(int slot, int h, int heads, int page_log2) {
  const int page = 1 << page_log2;
  return (static_cast<size_t>(slot >> page_log2) * heads + h) * cache4_block_bytes(page, D) +
         static_cast<size_t>((slot & (page - 1)) / kSlab4) * cache4_slab_bytes(D);
}

// Both row kernels: a thread takes one 32-bit word of codes (8 elements, two
// runs of 4) of a token, so D / 8 neighbouring threads take a row; a block
// takes kPass rows at a time of one head and tensor, kUnroll passes with all
// loads in front.  32768 tokens of 8 heads of 128, bf16, on B200: append 117 us (2.1
// TB/s; 80% of issue slots: 266 instructions a word), read 58 us (4.4 TB/s).
constexpr int kRowThreads = 256;
template <int D>
struct RC {
  static constexpr int kPer = D / 8;
  static constexpr int kPass = kRowThreads / kPer;
  static constexpr int kUnroll = 2;
  static constexpr int kRows = kPass * kUnroll;  // tokens of a block
};

// word e of a row: its lane in fragment order, word index and the dims of its two runs
template <bool V>
__device__ __forceinline__ void word_of(int e, int& lane, int& w, int& d0, int& d1) {
  w = V ? e / 8 : e / 4;
  lane = V ? e % 8 : e % 4;
  d0 = V ? 64 * w + 4 * lane : 32 * w + 4 * lane;
  d1 = V ? d0 + 32 : d0 + 16;
}
// nibble of element j of run r
template <bool V>
__device__ __forceinline__ constexpr int nibble_of(int r, int j) {
  return V ? 4 * r + j : (2 * r + (j >> 1)) + 4 * (j & 1);
}

// ================================================================== append
struct AppendParams {
  const void* x[3];  // k1, k2, v: (tokens, heads, D)
  long long st[3], sh[3];
  const int* slots;
  uint8_t* cache;
  int num_slots;
  int tokens;
  int heads;
  int page_log2;
  int normalize;
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ void load4(const float* p, float (&x)[8], int at) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[at] = v.x, x[at + 1] = v.y, x[at + 2] = v.z, x[at + 3] = v.w;
  }
  static __device__ __forceinline__ void store4(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[8], int at) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[at] = __uint_as_float(v.x << 16), x[at + 1] = __uint_as_float(v.x & 0xffff0000u);
    x[at + 2] = __uint_as_float(v.y << 16), x[at + 3] = __uint_as_float(v.y & 0xffff0000u);
  }
  static __device__ __forceinline__ void store4(__nv_bfloat16* p, const float* x) {
    __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ void load4(const __half* p, float (&x)[8], int at) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    x[at] = a.x, x[at + 1] = a.y, x[at + 2] = b.x, x[at + 3] = b.y;
  }
  static __device__ __forceinline__ void store4(__half* p, const float* x) {
    __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
};

// The nibble 8 + round-half-even(7 x / amax) without a division.  Adding 1.5 2^23 +
// 8 to an approximate quotient leaves 8 + c in the sum's last bits, c the nearest
// whole number or one beside it; the remainder 7 x - c amax is exact in fp32 for
// bf16 and fp16 inputs and says which: past amax / 2 the neighbour is nearer, and
// at amax / 2 (a tie) it is taken when c is odd.  Returned with other bits above.
// Of an fp32 input (WIDE) 7 x has up to 27 bits: its rounding rest is kept beside it,
// c amax is subtracted from the rounded part exactly (they agree to amax / 2), and the
// distance from amax / 2, exact as well, is corrected by the rest.
template <bool WIDE>
__device__ __forceinline__ uint32_t nibble(float x, float amax, float half, float inv7) {
  const float shifted = fmaf(x, inv7, 12582920.0f);
  const uint32_t n = __float_as_uint(shifted);
  const float seven = 7.0f * x, rem = fmaf(-(shifted - 12582920.0f), amax, seven);
  const int step = (static_cast<int>(__float_as_uint(rem)) >> 31) | 1;
  if constexpr (WIDE) {
    const float past = (fabsf(rem) - half) + static_cast<float>(step) * fmaf(7.0f, x, -seven);
    return n + (past > 0.f || (past == 0.f && (n & 1u)) ? step : 0);
  }
  const float edge = __uint_as_float(__float_as_uint(half) - (n & 1u));
  return n + (fabsf(rem) > edge ? step : 0);
}

__device__ __forceinline__ uint32_t max_bits(uint32_t a, float x) { return max(a, __float_as_uint(x) & 0x7fffffffu); }

// one word of codes and the scales of its runs' groups from 8 elements
template <int D, bool V, bool WIDE>
__device__ __forceinline__ uint32_t quantise(float (&x)[8], bool normalize, float (&sc)[2]) {
  // largest magnitude of each run's group, as bits so that a NaN wins
  uint32_t m[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i >> 2] = max_bits(m[i >> 2], x[i]);
  if (!V) m[0] = m[1] = max(m[0], m[1]);
#pragma unroll
  for (int o = 1; o < (V ? 8 : 4); o <<= 1) {
    m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
    if (V) m[1] = max(m[1], __shfl_xor_sync(0xffffffffu, m[1], o));
  }
  if (!V) m[1] = m[0];
  float inv_norm = 1.0f;
  if (normalize && !V) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 1; o < RC<D>::kPer; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    inv_norm = 1.0f / fmaxf(sqrtf(ss), 1e-12f);
  }
  // A largest magnitude near an end of the exponent's range (rare) is moved away from
  // it, with its group, so that neither 7 / amax nor 7 x leaves the range.
  float lift[2] = {1.0f, 1.0f};
  if (__any_sync(0xffffffffu, min(m[0], m[1]) < 0x22000000u || max(m[0], m[1]) > 0x5e000000u)) {  // 2^-59, 2^61
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      lift[r] = m[r] < 0x22000000u ? 0x1p80f : (m[r] > 0x5e000000u ? 0x1p-64f : 1.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * r + j] *= lift[r];
    }
  }
  uint32_t word = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float amax = __uint_as_float(m[r]) * lift[r], half = 0.5f * amax, inv7 = __fdividef(7.0f, amax);
    uint32_t part = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = 4 * nibble_of<V>(r, j);
      part |= (nibble<WIDE>(x[4 * r + j], amax, half, inv7) << at) & (15u << at);
    }
    // a group of zeros, or one that holds an infinity or a NaN (whose scale is NaN): codes of zero
    uint32_t zeros = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) zeros |= 8u << (4 * nibble_of<V>(r, j));
    word |= m[r] - 1u < 0x7f7fffffu ? part : zeros;
  }
#pragma unroll
  for (int r = 0; r < (V ? 2 : 1); ++r)
    sc[r] = m[r] < 0x7f800000u ? __uint_as_float(m[r]) / 7.0f * inv_norm : __uint_as_float(0x7fc00000u);
  return word;
}

template <int D, typename T, bool V>
__device__ __forceinline__ void append_rows(const AppendParams& p, const T* x, long long st, long long sh, int tensor, int h) {
  using C = RC<D>;
  int lane, w, d0, d1;
  word_of<V>(threadIdx.x % C::kPer, lane, w, d0, d1);
  const int t0 = blockIdx.x * C::kRows + threadIdx.x / C::kPer;
  float v[C::kUnroll][8];
  int slot[C::kUnroll];
#pragma unroll
  for (int u = 0; u < C::kUnroll; ++u) {
    const int t = t0 + u * C::kPass;
    slot[u] = t < p.tokens ? p.slots[t] : -1;
    if (t < p.tokens) {
      const T* src = x + t * st + h * sh;
      Elem<T>::load4(src + d0, v[u], 0);
      Elem<T>::load4(src + d1, v[u], 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < C::kUnroll; ++u) {
    float sc[2];
    const uint32_t word = quantise<D, V, sizeof(T) == 4>(v[u], p.normalize != 0, sc);
    if (static_cast<unsigned>(slot[u]) >= static_cast<unsigned>(p.num_slots)) continue;
    uint8_t* slab = p.cache + slab_of<D>(slot[u], h, p.heads, p.page_log2);
    const int r = slot[u] % kSlab4;
    *reinterpret_cast<uint32_t*>(slab + cache4_codes_at(tensor, D) + (V ? cache4_v_word(r, lane, w, D) : cache4_k_word(r, lane, w, D))) = word;
    if (lane == 0) {
      __nv_bfloat16* s = reinterpret_cast<__nv_bfloat16*>(slab + cache4_scales_at(tensor, D) + r * cache4_scale_bytes(D));
      if (V)
        *reinterpret_cast<__nv_bfloat162*>(s + 2 * w) = __floats2bfloat162_rn(sc[0], sc[1]);
      else
        s[w] = __float2bfloat16_rn(sc[0]);
    }
  }
}

// grid (token blocks, heads, tensors)
template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) cache4_append_kernel(const __grid_constant__ AppendParams p) {
  if (blockIdx.z == 0)
    append_rows<D, T, false>(p, static_cast<const T*>(p.x[0]), p.st[0], p.sh[0], 0, blockIdx.y);
  else if (blockIdx.z == 1)
    append_rows<D, T, false>(p, static_cast<const T*>(p.x[1]), p.st[1], p.sh[1], 1, blockIdx.y);
  else
    append_rows<D, T, true>(p, static_cast<const T*>(p.x[2]), p.st[2], p.sh[2], 2, blockIdx.y);
}

// ================================================================== read
struct ReadParams {
  const uint8_t* cache;
  const int* slots;
  void* y[3];
  int num_slots;
  int tokens;
  int heads;
  int page_log2;
};

template <int D, typename T, bool V>
__device__ __forceinline__ void read_rows(const ReadParams& p, T* y, int tensor, int h) {
  using C = RC<D>;
  int lane, w, d0, d1;
  word_of<V>(threadIdx.x % C::kPer, lane, w, d0, d1);
  const int t0 = blockIdx.x * C::kRows + threadIdx.x / C::kPer;
  uint32_t word[C::kUnroll];
  float s[C::kUnroll][2];
#pragma unroll
  for (int u = 0; u < C::kUnroll; ++u) {
    const int t = t0 + u * C::kPass;
    const int slot = t < p.tokens ? p.slots[t] : -1;
    word[u] = 0x88888888u;
    s[u][0] = s[u][1] = 0.f;
    if (static_cast<unsigned>(slot) < static_cast<unsigned>(p.num_slots)) {
      const uint8_t* slab = p.cache + slab_of<D>(slot, h, p.heads, p.page_log2);
      const int r = slot % kSlab4;
      word[u] = *reinterpret_cast<const uint32_t*>(slab + cache4_codes_at(tensor, D) +
                                                   (V ? cache4_v_word(r, lane, w, D) : cache4_k_word(r, lane, w, D)));
      const __nv_bfloat16* sp = reinterpret_cast<const __nv_bfloat16*>(slab + cache4_scales_at(tensor, D) + r * cache4_scale_bytes(D));
      s[u][0] = __bfloat162float(sp[V ? 2 * w : w]);
      s[u][1] = V ? __bfloat162float(sp[2 * w + 1]) : s[u][0];
    }
  }
#pragma unroll
  for (int u = 0; u < C::kUnroll; ++u) {
    const int t = t0 + u * C::kPass;
    if (t >= p.tokens) continue;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)  // 2^23 + n - (2^23 + 8)
      x[i] = (__uint_as_float(((word[u] >> (4 * nibble_of<V>(i >> 2, i & 3))) & 15u) | 0x4b000000u) - 8388616.0f) * s[u][i >> 2];
    T* row = y + (static_cast<long long>(t) * p.heads + h) * D;
    Elem<T>::store4(row + d0, x);
    Elem<T>::store4(row + d1, x + 4);
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) cache4_read_kernel(const __grid_constant__ ReadParams p) {
  if (blockIdx.z == 0)
    read_rows<D, T, false>(p, static_cast<T*>(p.y[0]), 0, blockIdx.y);
  else if (blockIdx.z == 1)
    read_rows<D, T, false>(p, static_cast<T*>(p.y[1]), 1, blockIdx.y);
  else
    read_rows<D, T, true>(p, static_cast<T*>(p.y[2]), 2, blockIdx.y);
}

template <int D, typename P, typename K>
cudaError_t launch_rows(K kernel, const P& p, cudaStream_t s) {
  kernel<<<dim3(static_cast<unsigned>(ceil_div(p.tokens, RC<D>::kRows)), p.heads, 3), kRowThreads, 0, s>>>(p);
  return cudaGetLastError();
}

int log2_page(int64_t page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

int check_cache(const void* cache, int64_t num_pages, int64_t heads, int64_t D, int64_t page) {
  if (D != 64 && D != 128) return fail(TDA_ERR_UNSUPPORTED, "the 4-bit cache needs head_dim 64 or 128 (got %lld)", static_cast<long long>(D));
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(TDA_ERR_INVALID, "page_size must be 16, 32, 64 or 128 (got %lld)", static_cast<long long>(page));
  if (heads < 1 || num_pages < 1) return fail(TDA_ERR_INVALID, "num_pages and kv heads must be >= 1");
  if (num_pages > 0x7fffffffll / page) return fail(TDA_ERR_INVALID, "num_pages * page_size must fit 31 bits");
  if (!cache || !aligned(cache, 16)) return fail(TDA_ERR_INVALID, "cache must be non-NULL and 16-byte aligned");
  return TDA_OK;
}

int check_rows(int64_t tokens, int64_t heads) {
  if (tokens < 1 || tokens > 0x7fffffffll - 1024) return fail(TDA_ERR_INVALID, "tokens must be in [1, 2^31 - 1024)");
  if (heads > 65535) return fail(TDA_ERR_INVALID, "too many kv heads");
  return TDA_OK;
}

}  // namespace

int cache4_check(const void* cache, int64_t num_pages, int64_t heads, int64_t D, int64_t page) {
  return check_cache(cache, num_pages, heads, D, page);
}

}  // namespace tda

using namespace tda;

extern "C" {

size_t tda_cache4_block_bytes(int64_t page_size, int64_t head_dim) {
  if ((head_dim != 64 && head_dim != 128) || page_size < 16 || page_size > 128 || (page_size & (page_size - 1)) != 0) return 0;
  return cache4_block_bytes(static_cast<int>(page_size), static_cast<int>(head_dim));
}

int tda_plan_pages(const int32_t* lengths, const int32_t* new_tokens, int64_t requests, int32_t* block_table,
                   int64_t table_stride, int64_t table_width, const int32_t* free_pages, int64_t num_free,
                   const int32_t* free_head, int64_t page_size, int64_t rows, int32_t* slots, int32_t* positions,
                   int32_t* request_ids, int32_t* starts, int32_t* lengths_out, int32_t* free_head_out,
                   int32_t* dropped, void* stream) {
  if (requests < 1 || requests > (1 << 24)) return fail(TDA_ERR_INVALID, "requests must be in [1, 2^24]");
  if (table_width < 1 || table_stride < table_width) return fail(TDA_ERR_INVALID, "block table needs a width >= 1 and a stride >= the width");
  if (page_size < 1 || page_size > (1 << 16)) return fail(TDA_ERR_INVALID, "page_size must be in [1, 65536]");
  if (table_width > (1ll << 30) / page_size) return fail(TDA_ERR_INVALID, "table width * page_size must fit 30 bits");
  if (num_free < 0 || num_free > 0x7fffffffll / page_size) return fail(TDA_ERR_INVALID, "free list too long");
  if (rows < 0 || rows > (1ll << 30)) return fail(TDA_ERR_INVALID, "rows must be in [0, 2^30]");
  const void* need[] = {lengths, new_tokens, block_table, free_head, starts, lengths_out, free_head_out, dropped};
  for (const void* x : need)
    if (!x || !aligned(x, 4)) return fail(TDA_ERR_INVALID, "plan arrays must be non-NULL int32");
  if (num_free > 0 && !free_pages) return fail(TDA_ERR_INVALID, "free_pages is NULL");
  if (rows > 0 && (!slots || !positions || !request_ids)) return fail(TDA_ERR_INVALID, "row outputs are NULL");
  PlanParams p;
  p.lengths = lengths;
  p.added = new_tokens;
  p.table = block_table;
  p.free_pages = free_pages;
  p.free_head = free_head;
  p.slots = slots;
  p.positions = positions;
  p.requests = request_ids;
  p.starts = starts;
  p.lengths_out = lengths_out;
  p.free_head_out = free_head_out;
  p.dropped = dropped;
  p.table_stride = table_stride;
  p.B = static_cast<int>(requests);
  p.width = static_cast<int>(table_width);
  p.n_free = static_cast<int>(num_free);
  p.page = static_cast<int>(page_size);
  p.rows = static_cast<int>(rows);
  const int64_t blocks = rows > 0 ? ceil_div(rows, kPlanRows) : 1;
  plan_pages_kernel<<<static_cast<unsigned>(blocks), kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "page plan launch");
}

int tda_cache4_append(const void* k1, const void* k2, const void* v, int dtype, const int64_t* strides,
                      const int32_t* slots, int64_t tokens, void* cache, int64_t num_pages, int64_t kv_heads,
                      int64_t head_dim, int64_t page_size, int normalize_keys, void* stream) {
  if (int e = check_cache(cache, num_pages, kv_heads, head_dim, page_size)) return e;
  if (int e = check_rows(tokens, kv_heads)) return e;
  if (!slots || !aligned(slots, 4)) return fail(TDA_ERR_INVALID, "slots must be non-NULL int32");
  AppendParams p;
  const void* xs[3] = {k1, k2, v};
  for (int i = 0; i < 3; ++i) {
    if (!xs[i] || !aligned(xs[i], 16)) return fail(TDA_ERR_INVALID, "k1, k2 and v must be non-NULL and 16-byte aligned");
    p.x[i] = xs[i];
    p.st[i] = strides ? strides[2 * i] : kv_heads * head_dim;
    p.sh[i] = strides ? strides[2 * i + 1] : head_dim;
    if (p.st[i] <= 0 || p.sh[i] <= 0 || (p.st[i] | p.sh[i]) % 8 != 0)
      return fail(TDA_ERR_INVALID, "input strides must be positive multiples of 8 elements");
  }
  p.slots = slots;
  p.cache = static_cast<uint8_t*>(cache);
  p.num_slots = static_cast<int>(num_pages * page_size);
  p.tokens = static_cast<int>(tokens);
  p.heads = static_cast<int>(kv_heads);
  p.page_log2 = log2_page(page_size);
  p.normalize = normalize_keys != 0;
  const int D = static_cast<int>(head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define TDA_APPEND(T) (D == 64 ? launch_rows<64>(cache4_append_kernel<64, T>, p, s) \
                               : launch_rows<128>(cache4_append_kernel<128, T>, p, s))
  if (dtype == TDA_BF16)
    e = TDA_APPEND(__nv_bfloat16);
  else if (dtype == TDA_F16)
    e = TDA_APPEND(__half);
  else if (dtype == TDA_F32)
    e = TDA_APPEND(float);
  else
    return fail(TDA_ERR_INVALID, "dtype must be TDA_F32, TDA_BF16 or TDA_F16");
#undef TDA_APPEND
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "cache append launch");
}

int tda_cache4_read(const void* cache, int64_t num_pages, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                    const int32_t* slots, int64_t tokens, void* k1, void* k2, void* v, int dtype, void* stream) {
  if (int e = check_cache(cache, num_pages, kv_heads, head_dim, page_size)) return e;
  if (int e = check_rows(tokens, kv_heads)) return e;
  if (!slots || !aligned(slots, 4)) return fail(TDA_ERR_INVALID, "slots must be non-NULL int32");
  ReadParams p;
  void* ys[3] = {k1, k2, v};
  for (int i = 0; i < 3; ++i) {
    if (!ys[i] || !aligned(ys[i], 16)) return fail(TDA_ERR_INVALID, "k1, k2 and v must be non-NULL and 16-byte aligned");
    p.y[i] = ys[i];
  }
  p.cache = static_cast<const uint8_t*>(cache);
  p.slots = slots;
  p.num_slots = static_cast<int>(num_pages * page_size);
  p.tokens = static_cast<int>(tokens);
  p.heads = static_cast<int>(kv_heads);
  p.page_log2 = log2_page(page_size);
  const int D = static_cast<int>(head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define TDA_READ(T) (D == 64 ? launch_rows<64>(cache4_read_kernel<64, T>, p, s) \
                             : launch_rows<128>(cache4_read_kernel<128, T>, p, s))
  if (dtype == TDA_BF16)
    e = TDA_READ(__nv_bfloat16);
  else if (dtype == TDA_F16)
    e = TDA_READ(__half);
  else if (dtype == TDA_F32)
    e = TDA_READ(float);
  else
    return fail(TDA_ERR_INVALID, "dtype must be TDA_F32, TDA_BF16 or TDA_F16");
#undef TDA_READ
  return e == cudaSuccess ? TDA_OK : cuda_fail(e, "cache read launch");
}

}  // extern "C"
