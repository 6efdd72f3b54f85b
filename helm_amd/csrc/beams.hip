// Beam search over a paged cache: the choice of a step's continuations (helm_beam_select)
// and the block tables that follow from it (helm_beam_tables).
//
// Selection.  Beam k of a request with running score s_k offers token t at
//   s_k + x_kt - lse_k,   lse_k = log(sum over t of e^{x_kt}),
// and the n best of the request's K V candidates are wanted, ties to the lowest k V + t.
// Within a row the order is the logits' own, so one pass over them gives a chunk's
// largest value, its sum and its n best, and the rows meet in a second, small kernel.
// Bound by memory: the logits are read once.  The order is of the 64-bit sums
// (s_k - lse_k) + x_kt, ties to the lowest k V + t.  Exponentials are in 32 bits, and so are their
// sums over a thread's up to 32 values and over its wave; waves, chunks, logarithms and scores
// are added in 64.  That leaves lse off by some 1e-7 (2^-18 if every one of its 42 roundings fell
// the same way), so candidates of one row are in order, and two of different rows change places
// only where their scores are as near as that.
//
// A chunk's n best: the n-th largest of the 256 threads' maxima, which every wave finds for
// itself by a search over the value's leading bits with ballots, is at most the n-th largest of
// the chunk and leaves little more than n values (34 of 32, 74 of 64 in a random row).  They
// are put in a list and ranked by counting.  Where ties or a sorted row leave more than the
// list holds, the workgroup searches value and index bit by bit instead.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cfloat>
#include <string>
#include <type_traits>

#include "attn_kernel.h"
#include "helm_amd.h"
#include "ranges.h"

namespace helm {
int report_error(int code, const std::string& msg);
}

namespace {

using helm::bf16_t;
using helm::f16_t;

constexpr int kBeamThreads = 256;
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kList = 512;                   // values that a chunk's bound may leave
constexpr int kJoinList = 2048;              // and a request's

struct SelectArgs {
  const void* logits;
  int64_t b_stride, k_stride;                // elements
  const float* scores;
  int B, K, V, n, chunks, size;              // chunks of a row, logits of one
  double* part_sum;                          // [B K][chunks]
  float* part_max;                          // [B K][chunks]
  float* cand_x;                             // [B][n][K chunks], -inf: none; a chunk's n best are
  int* cand_t;                               // a column, best first
  float* out_scores;
  int64_t* out_tokens;
  int32_t* out_parents;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed)) Any16 { u32x4 v; };

// Whole numbers in the order of the floats (no NaN).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);          // (-0 is +0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __longlong_as_double((long long)(u >> 63 ? u & 0x7fffffffffffffffull : ~u));
}
// A reduction over the wave's 64 lanes, `none` its neutral value; the result is uniform.
template <typename F> __device__ __forceinline__ float wave_reduce(float x, float none, F f) {
  const int o = __builtin_bit_cast(int, none);
  auto with = [&](auto ctrl, auto rows) {
    const int y = __builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                              decltype(rows)::value, 0xf, false);
    x = f(x, __builtin_bit_cast(float, y));
  };
  using std::integral_constant;
  with(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
  with(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  with(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  with(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  with(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // row_bcast 15, 31
  with(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The n-th largest (1 <= n <= 64) of the workgroup's keys in sh, one a thread, in its leading
// kBits bits, the others zero: every wave finds it for itself.  Up to 40 of them, of the
// largest of each four, of which there are 64: nearly as good a bound (44 values for the best 32
// of a random row) for a quarter of the ballots.
// (Rolled up: a kernel's first pass over its code waits for it, 64 bytes at a time.)
template <int kBits> __device__ __forceinline__ uint32_t nth_key(const uint32_t* sh, int n) {
  u32x4 k = reinterpret_cast<const u32x4*>(sh)[threadIdx.x & 63];
  uint32_t t = 0;
  if (n <= 40) {
    const uint32_t top = max(max(k[0], k[1]), max(k[2], k[3]));
#pragma unroll 2
    for (int b = 31; b >= 32 - kBits; --b) {
      const uint32_t c = t | 1u << b;
      if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(top >= c)) >= n) t = c;
    }
    return t;
  }
#pragma unroll 1
  for (int b = 31; b >= 32 - kBits; --b) {
    const uint32_t c = t | 1u << b;
    int have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      have += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k[i] >= c));
    if (have >= n) t = c;
  }
  return t;
}

__device__ __forceinline__ int block_sum(int x, int* sh) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < kBeamWaves; ++w) s += sh[w];
  return s;
}

template <typename T> struct Elem;           // the values of 16 bytes
template <> struct Elem<float> {
  static constexpr int kPer = 4;
  __device__ static float get(const u32x4& w, int j) { return __uint_as_float(w[j]); }
  __device__ static float read(const float* x) { return *x; }
};
template <> struct Elem<bf16_t> {
  static constexpr int kPer = 8;
  __device__ static float get(const u32x4& w, int j) {
    return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
  }
  __device__ static float read(const bf16_t* x) { return __uint_as_float((uint32_t)x->x << 16); }
};
template <> struct Elem<f16_t> {
  static constexpr int kPer = 8;
  __device__ static float get(const u32x4& w, int j) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j >> 1] >> (16 * (j & 1))));
  }
  __device__ static float read(const f16_t* x) { return (float)__builtin_bit_cast(_Float16, x->x); }
};

// Chunk blockIdx.x of row blockIdx.y: its maximum, sum and n best.  A thread holds NV runs
// of 16 bytes in registers, a chunk is 256 times that.
template <typename T, int NV>
__global__ __launch_bounds__(kBeamThreads) void beam_scan_kernel(SelectArgs a) {
  constexpr int E = Elem<T>::kPer;
  constexpr int kSize = kBeamThreads * NV * E;
  __shared__ float sh_max[kBeamWaves];
  __shared__ __attribute__((aligned(16))) uint32_t sh_key[kBeamThreads];
  __shared__ float sh_sum[kBeamWaves];
  __shared__ int sh_n[kBeamWaves], sh_count;
  __shared__ int list_t[kList];
  __shared__ uint64_t list[kList];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.y, n = a.n;
  const int first = blockIdx.x * kSize;
  const T* x = reinterpret_cast<const T*>(a.logits) + row / a.K * a.b_stride +
               row % a.K * a.k_stride + first;
  const int left = a.V - first;               // values of this chunk and those behind it
  u32x4 raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * kBeamThreads + tid) * E;
    if (at + E <= left) {
      raw[v] = reinterpret_cast<const Any16*>(x + at)->v;   // (rows at any alignment)
    } else {
      // the row's last values and -inf behind them
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          w[j] = at + j < left ? reinterpret_cast<const uint32_t*>(x)[at + j] : 0xff800000u;
        } else {
          const uint32_t none = sizeof(T) == 2 && __is_same(T, bf16_t) ? 0xff80u : 0xfc00u;
          const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
          const uint32_t lo = at + 2 * j < left ? h[at + 2 * j] : none;
          const uint32_t hi = at + 2 * j + 1 < left ? h[at + 2 * j + 1] : none;
          w[j] = lo | hi << 16;
        }
      }
      raw[v] = u32x4{w[0], w[1], w[2], w[3]};
    }
  }
  if (tid == 0) sh_count = 0;
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < E; ++j) top = fmaxf(top, Elem<T>::get(raw[v], j));
  float m = wave_reduce(top, -INFINITY, [](float p, float q) { return fmaxf(p, q); });
  if (lane == 0) sh_max[wave] = m;
  sh_key[tid] = ordered(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBeamWaves; ++w) m = fmaxf(m, sh_max[w]);
  // (16 bits of it: a bf16 value whole; 32 took half as long again as the sums)
  const float least =
      fmaxf(unordered(max(nth_key<16>(sh_key, n), ordered(-INFINITY))), -FLT_MAX);

  // the sum of e^(x - m) (NaN or an infinity where the row has one): 1 for the largest itself
  const float base = m == -INFINITY ? 0.f : m;
  float part = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < E; ++j)
      part += __builtin_amdgcn_exp2f((Elem<T>::get(raw[v], j) - base) * 1.44269504f);
  part = wave_reduce(part, 0.f, [](float p, float q) { return p + q; });
  if (lane == 0) sh_sum[wave] = part;
  // of a thread's values, those that may be among the n best: none of most threads'
  if (top >= least) {
    uint64_t mine = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      uint32_t some = 0;                      // the last value in the lowest bit
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float y = Elem<T>::get(raw[v], j);
        some = 2 * some + (y >= least ? 1u : 0u);
      }
      mine |= (uint64_t)some << (E * v);
    }
    for (; mine; mine &= mine - 1) {
      const int e = __builtin_ctzll(mine), v = e / E, j = E - 1 - e % E;
      const int i = atomicAdd(&sh_count, 1);
      if (i < kList) list_t[i] = (v * kBeamThreads + tid) * E + j;
    }
  }
  __syncthreads();
  const int64_t p = (int64_t)row * a.chunks + blockIdx.x;
  if (tid == 0) {
    a.part_max[p] = base;
    a.part_sum[p] = ((double)sh_sum[0] + sh_sum[1]) + ((double)sh_sum[2] + sh_sum[3]);
  }
  int count = sh_count;
  if (count > kList) {
    // exactly n: the n-th largest value, and how far among its equals
    auto at_least = [&](uint32_t key) {
      int c = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < E; ++j) c += ordered(Elem<T>::get(raw[v], j)) >= key;
      return block_sum(c, sh_n);
    };
    uint32_t key = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t c = key | 1u << b;
      if (at_least(c) >= n) key = c;
    }
    const float edge = unordered(key);
    const int need = n - at_least(key + 1);
    int last = 0;                             // of the equals, those before it are less than need
    for (int b = 30; b >= 0; --b) {
      const int c = last | 1 << b;
      if (c >= kSize) continue;
      int k = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < E; ++j)
          k += Elem<T>::get(raw[v], j) == edge && (v * kBeamThreads + tid) * E + j < c;
      if (block_sum(k, sh_n) < need) last = c;
    }
    __syncthreads();
    if (tid == 0) sh_count = 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float y = Elem<T>::get(raw[v], j);
        const int t = (v * kBeamThreads + tid) * E + j;
        if (y > -INFINITY && (y > edge || (y == edge && t <= last))) {
          const int i = atomicAdd(&sh_count, 1);
          if (i < kList) list_t[i] = t;
        }
      }
    __syncthreads();
    count = min(sh_count, kList);
  }
  // one number a value: better ones are larger, and of equals those before
  for (int i = tid; i < count; i += kBeamThreads) {
    const int t = list_t[i];
    list[i] = (uint64_t)ordered(Elem<T>::read(x + t)) << 32 | (uint32_t)~t;
  }
  __syncthreads();
  const int lists = a.K * a.chunks;
  const int64_t col = (int64_t)(row / a.K) * n * lists + row % a.K * a.chunks + blockIdx.x;
  float* cx = a.cand_x + col;
  int* ct = a.cand_t + col;
  // ranked by counting, four threads a value
  for (int i0 = 0; i0 < count; i0 += kBeamThreads / 4) {
    const int i = i0 + tid / 4;
    const uint64_t mine = list[min(i, count - 1)];
    int rank = 0;
#pragma unroll 4
    for (int k = tid & 3; k < count; k += 4) rank += list[k] > mine;
    rank += __shfl_xor(rank, 1, 64);
    rank += __shfl_xor(rank, 2, 64);
    if (i < count && rank < n && (tid & 3) == 0) {
      cx[rank * lists] = unordered((uint32_t)(mine >> 32));
      ct[rank * lists] = first + (int)~(uint32_t)mine;
    }
  }
  for (int i = count + tid; i < n; i += kBeamThreads) {
    cx[i * lists] = -INFINITY;
    ct[i * lists] = 0;
  }
}

// The n best of request blockIdx.x from its rows' chunks.
template <typename T>
__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(SelectArgs a) {
  __shared__ double base[64];                // s_k - lse_k; -inf: the row offers nothing
  __shared__ __attribute__((aligned(16))) uint32_t sh_key[kBeamThreads];
  __shared__ int sh_n[kBeamWaves], sh_count, sh_close;
  __shared__ double list_x[kJoinList], sh_edge;
  __shared__ int64_t list_i[kJoinList];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x, n = a.n, C = a.chunks;
  if (tid == 0) sh_count = sh_close = 0;
  // candidate i of the request: of list i % (K C), that is of a row's chunk, the (i / (K C))th.
  // The lists lie side by side, from their best on; eight a thread are on their way at once,
  // the first of them before the rows' sums.
  constexpr int U = 8, kBatch = U * kBeamThreads;
  const int lists = a.K * C, all = lists * n;
  const float* cx = a.cand_x + (int64_t)b * all;
  const int* ct = a.cand_t + (int64_t)b * all;
  float x[U];
  int t0[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * kBeamThreads + tid;
    x[u] = i < all ? cx[i] : -INFINITY;
    t0[u] = i < all ? ct[i] : 0;
  }
  // the rows' sums, a row to the first power of two of lanes that holds its chunks
  const int wide = C > 32 ? 64 : C > 1 ? 2 << (31 - __builtin_clz(C - 1)) : 1;
  const int per_wave = 64 / wide, c1 = lane & (wide - 1);
  for (int k0 = wave * per_wave; k0 < a.K; k0 += kBeamWaves * per_wave) {
    const int k = min(k0 + lane / wide, a.K - 1);
    const int64_t p = ((int64_t)b * a.K + k) * C;
    const float score = a.scores[b * a.K + k];
    // against the row's largest (a chunk of -inf has 0 for it and for a sum)
    float top = -INFINITY;
    double s = 0.0;
    for (int c = c1; c < C + c1; c += wide) {
      const double part = c < C ? a.part_sum[p + c] : 0.0;
      const float max_c = c < C ? a.part_max[p + c] : 0.f;
      const float at = part != 0.0 ? max_c : -INFINITY;
      float m = at;
      for (int d = wide / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
      if (m > top) {
        s *= exp((double)top - (double)m);
        top = m;
      }
      if (part != 0.0) s += part * exp((double)at - (double)top);
    }
    for (int d = wide / 2; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if (c1 == 0 && k0 + lane / wide < a.K) {
      const double x = (double)score - ((double)top + log(s));
      base[k] = fabsf(score) < INFINITY && fabs(x) < INFINITY ? x : -INFINITY;
    }
  }
  __syncthreads();
  auto sum = [&](int list, float v) {
    const double s = base[list / C];
    return v == -INFINITY || s == -INFINITY ? -INFINITY : s + (double)v;
  };
  const int hop = kBeamThreads % lists;
  auto next = [&](int l) { return l + hop < lists ? l + hop : l + hop - lists; };
  int at[U];                                 // the eight's lists
#pragma unroll
  for (int u = 0; u < U; ++u) at[u] = u ? next(at[u - 1]) : tid % lists;
  // a bound: up to 16, the n-th largest of the threads' maxima; beyond (where one row may hold
  // most of the best, several a thread: 4 x 16 rows, n = 32: 21 -> 16 us) of each wave's 512
  // values the n-th largest, to eight bits of its mantissa
  double y0[U], top = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    y0[u] = sum(at[u], x[u]);
    top = fmax(top, y0[u]);
  }
  uint32_t bound = 0;
  if (n <= 16) {
    sh_key[tid] = (uint32_t)(ordered(top) >> 32);
    __syncthreads();
    bound = nth_key<24>(sh_key, n);
  } else {
    uint32_t key[U];
#pragma unroll
    for (int u = 0; u < U; ++u) key[u] = (uint32_t)(ordered(y0[u]) >> 32);
#pragma unroll 1
    for (int bit = 31; bit >= 12; --bit) {
      const uint32_t c = bound | 1u << bit;
      int have = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        have += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[u] >= c));
      if (have >= n) bound = c;
    }
    if (lane == 0) sh_key[wave] = bound;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) bound = max(bound, sh_key[w]);
  }
  const double least = unordered(max((uint64_t)bound << 32, ordered(-(double)INFINITY)));
  // whether another logit of the list's row may give the same sum
  auto close = [&](int list, float v, double y) {
    const double s = base[list / C];
    return s + (double)unordered(ordered(v) + 1) == y || s + (double)unordered(ordered(v) - 1) == y;
  };
  auto keep = [&](double y, int64_t t) {
    const int i = atomicAdd(&sh_count, 1);
    if (i < kJoinList) {
      list_x[i] = y;
      list_i[i] = t;
    }
  };
  bool any = false;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (y0[u] >= least && y0[u] > -INFINITY) {
      any = true;
      if (close(at[u], x[u], y0[u])) sh_close = 1;
      keep(y0[u], (int64_t)(at[u] / C) << 32 | t0[u]);
    }
  // on until none of the lists has one left (a sweep holds one of each)
  const int sweep = (lists + kBatch - 1) / kBatch * kBatch;
  auto value = [&](int i) { return sum(i % lists, cx[i]); };
  auto index = [&](int i) { return (int64_t)(i % lists / C) << 32 | ct[i]; };   // (row, token)
  for (int i0 = kBatch; i0 < all; i0 += kBatch) {
    if (i0 % sweep == 0) {
      if (!__syncthreads_or(any)) break;
      any = false;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kBeamThreads + tid;
      x[u] = i < all ? cx[i] : -INFINITY;
    }
    int l = next(at[U - 1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = l;
      l = next(l);
      const double y = sum(at[u], x[u]);
      if (y >= least && y > -INFINITY) {
        any = true;
        if (close(at[u], x[u], y)) sh_close = 1;
        keep(y, index(i0 + u * kBeamThreads + tid));
      }
    }
  }
  __syncthreads();
  int count = sh_count;
  if (count > kJoinList) {
    auto counted = [&](auto wanted) {
      int c = 0;
      for (int i = tid; i < all; i += kBeamThreads) c += wanted(value(i), i);
      return block_sum(c, sh_n);
    };
    uint64_t key = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t c = key | 1ull << bit;
      if (counted([&](double y, int) { return ordered(y) >= c; }) >= n) key = c;
    }
    const double edge = unordered(key);
    const int need = n - counted([&](double y, int) { return ordered(y) > key; });
    int64_t last = 0;
    for (int bit = 37; bit >= 0; --bit) {
      const int64_t c = last | 1ll << bit;
      if (counted([&](double y, int i) { return y == edge && index(i) < c; }) < need) last = c;
    }
    __syncthreads();
    if (tid == 0) sh_count = 0;
    __syncthreads();
    for (int i = tid; i < all; i += kBeamThreads) {
      const double y = value(i);
      if (y > edge || (y == edge && index(i) <= last)) keep(y, index(i));
    }
    __syncthreads();
    count = min(sh_count, kJoinList);
  }
  const int64_t o = (int64_t)b * n;
  for (int i0 = 0; i0 < count; i0 += kBeamThreads / 4) {
    const int i = i0 + tid / 4;
    const double y = list_x[min(i, count - 1)];
    const int64_t t = list_i[min(i, count - 1)];
    int rank = 0;
#pragma unroll 4
    for (int k = tid & 3; k < count; k += 4) {
      const double z = list_x[k];
      rank += z > y || (z == y && list_i[k] < t);
    }
    rank += __shfl_xor(rank, 1, 64);
    rank += __shfl_xor(rank, 2, 64);
    if (i < count && rank < n && (tid & 3) == 0) {
      if (rank == n - 1) sh_edge = y;
      // (never -inf, which stands for no candidate)
      a.out_scores[o + rank] = (float)fmin(fmax(y, -(double)FLT_MAX), (double)FLT_MAX);
      a.out_tokens[o + rank] = t & 0xffffffff;
      a.out_parents[o + rank] = (int32_t)(t >> 32);
    }
  }
  for (int i = count + tid; i < n; i += kBeamThreads) {
    a.out_scores[o + i] = -INFINITY;
    a.out_tokens[o + i] = -1;
    a.out_parents[o + i] = -1;
  }

  // A chunk's n best are its largest logits.  Where 64 bits do not tell sums of different logits
  // apart (a score or lse past some 2^29 times the logits' spacing, logits next to zero), a chunk
  // may have left out a lower token of the n-th best sum; all larger sums are there.  Then the
  // lowest indexes of that sum are looked for in the logits, in the chunks that it is in.
  if (!sh_close || count < n) return;         // (uniform: nobody writes either any more)
  __syncthreads();
  const double edge = sh_edge;
  if (tid == 0) sh_close = 0;
  __syncthreads();
  for (int l = tid; l < lists; l += kBeamThreads) {
    const float v = cx[(n - 1) * lists + l];
    const double y = sum(l, v);
    if (v > -INFINITY && y == edge && close(l, v, y)) {
      const int i = atomicAdd(&sh_close, 1);
      if (i < kBeamThreads) sh_key[i] = l;
    }
  }
  __syncthreads();
  // whether one of those chunks has more of that sum than its n best: mostly not (n = 1 and a row
  // whose largest logit is 0: 64 x 4 rows of 131,072 22.8 -> 25.7 us; all 4 x 32,000 logits one sum,
  // so that the joining finds more than its list holds too: 39 us)
  const int full = sh_close;
  bool more = full > kBeamThreads;
  for (int i = 0; i < full && !more; ++i) {
    const int l = sh_key[i], t0 = l % C * a.size, size = min(a.size, a.V - t0);
    const double s = base[l / C];
    const T* x = reinterpret_cast<const T*>(a.logits) + b * a.b_stride + l / C * a.k_stride + t0;
    constexpr int E = Elem<T>::kPer;
    int hidden = tid < n && sum(l, cx[tid * lists + l]) == edge ? -1 : 0;
#pragma unroll 4
    for (int t = tid * E; t < size; t += kBeamThreads * E) {
      if (t + E <= size) {
        const u32x4 w = reinterpret_cast<const Any16*>(x + t)->v;
#pragma unroll
        for (int j = 0; j < E; ++j) hidden += s + (double)Elem<T>::get(w, j) == edge;
      } else {
        for (int j = t; j < size; ++j) hidden += s + (double)Elem<T>::read(x + j) == edge;
      }
    }
    more = block_sum(hidden, sh_n) > 0;
  }
  if (!more) return;
  int above = 0;
  for (int i = tid; i < count; i += kBeamThreads) above += list_x[i] > edge;
  const int first = block_sum(above, sh_n), need = n - first;
  int have = 0;
  for (int l = -1; have < need;) {
    if (tid == 0) sh_count = lists;
    __syncthreads();
    for (int i = tid; i < count; i += kBeamThreads) {
      const int in = (int)(list_i[i] >> 32) * C + (int)((uint32_t)list_i[i] / (uint32_t)a.size);
      if (list_x[i] == edge && in > l) atomicMin(&sh_count, in);
    }
    __syncthreads();
    l = sh_count;                             // the next of those chunks
    if (l >= lists) break;
    const int k = l / C, t0 = l % C * a.size;
    const double s = base[k];
    const T* row = reinterpret_cast<const T*>(a.logits) + b * a.b_stride + k * a.k_stride + t0;
    const int size = min(a.size, a.V - t0);
    for (int v0 = 0; v0 < size && have < need; v0 += kBatch) {
      uint64_t hits[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = v0 + u * kBeamThreads + tid;
        const float v = t < size ? Elem<T>::read(row + t) : -INFINITY;
        hits[u] = __builtin_amdgcn_ballot_w64(v > -INFINITY && s + (double)v == edge);
        if (lane == 0) sh_key[u * kBeamWaves + wave] = __builtin_popcountll(hits[u]);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
        for (int w = 0; w < kBeamWaves; ++w) {
          const int r = have + __builtin_popcountll(hits[u] & ((1ull << lane) - 1));
          if (w == wave && (hits[u] >> lane & 1) && r < need) {
            a.out_tokens[o + first + r] = t0 + v0 + u * kBeamThreads + tid;
            a.out_parents[o + first + r] = k;
          }
          have += sh_key[u * kBeamWaves + w];
        }
      __syncthreads();                        // (sh_key has been read)
    }
  }
}

// Chunks of a row: 64 bytes a thread (128 in fp32), so that the joining has few lists, or, where
// there are few logits, 16 (32), so that a chunk is done sooner.  A call in a graph, with the one
// and with the other: 4 rows of 32,000 bf16 logits 9.2 us, 8.6; a row of 128,000 9.2, 8.9; 4 rows
// of 152,064 10.2, 10.8; 8 rows 11.3, 16.9; 64 rows and 64 beams 46, 205.  (32 and 128 bytes:
// 256 rows of 131,072 take 22.6 and 24.7 us against 22.)
struct SelectPlan {
  int nv, chunks, size;
  int64_t rows, bytes;
};
SelectPlan select_plan(int B, int K, int V, int n, int es) {
  SelectPlan p{};
  p.rows = (int64_t)B * K;
  const int per = kBeamThreads * 16 / es;
  p.nv = es / 2 * (p.rows * ((V - 1) / 2048 + 1) > 128 ? 4 : 1);
  p.size = p.nv * per;
  p.chunks = (V - 1) / p.size + 1;
  p.bytes = p.rows * p.chunks * (12 + 8 * (int64_t)n);
  return p;
}
bool select_ok(int B, int K, int V, int n) {
  return B >= 0 && K >= 1 && K <= HELM_BEAMS_MAX && V >= 1 && n >= 1 && n <= HELM_BEAMS_MAX &&
         (int64_t)B * K <= 65535 &&
         (int64_t)K * ((V - 1) / 1024 + 1) * n <= 0x7fffffff;
}

template <typename T> void launch_select(const SelectArgs& a, const SelectPlan& p, hipStream_t st) {
  const dim3 grid(p.chunks, (uint32_t)p.rows);
  constexpr int S = sizeof(T) / 2;
  if (p.nv == S) hipLaunchKernelGGL((beam_scan_kernel<T, S>), grid, dim3(kBeamThreads), 0, st, a);
  else hipLaunchKernelGGL((beam_scan_kernel<T, 4 * S>), grid, dim3(kBeamThreads), 0, st, a);
  hipLaunchKernelGGL((beam_join_kernel<T>), dim3(a.B), dim3(kBeamThreads), 0, st, a);
}

// ---- tables ----------------------------------------------------------------------------
//
// Row j of a request goes on from p_j = parents[j] (j itself where that is no row).  Full
// pages are shared by name: new[j][c] = old[p_j][c].  A part-filled page is a row's own, since
// its next token goes there: the keeper of parent p (p itself if it is its own child, else its
// lowest child) keeps the page, and p's other children take, in ascending order, the
// part-filled pages of the rows that no row goes on from.  There are as many of those as of
// other children, no page is both read and written, and nothing is taken from a free list.
//
// The first launch, a workgroup per request and 128 columns, a column a thread, writes the
// tables (in place too: a column's old entries are in LDS before its new ones are stored),
// which page is copied where, and its columns' pages that no row names any more; the second
// copies the pages' tokens in all layers' pools and joins the lists of released pages, in the
// order of requests, columns and rows.
constexpr int kCols = 128;
constexpr int kPools = 128;                  // a launch's

struct BeamTableArgs {
  const int32_t* parents;
  int B, K;
  const int32_t* table;
  int64_t stride;
  int width, chunks;
  const int32_t* lens;
  int page;
  const int32_t* shared;                     // may be null: none
  int32_t* out;
  int64_t out_stride;
  int32_t* copies;                           // [B K][2]
  int32_t* lists;                            // [B][chunks][K kCols]
  int32_t* counts;                           // [B][chunks]
  int32_t* released;
  int32_t* n_released;
};

// The i-th set bit of x (there are more than i).
__device__ __forceinline__ int nth_bit(uint64_t x, int i) {
  for (; i > 0; --i) x &= x - 1;
  return __builtin_ctzll(x);
}

__global__ __launch_bounds__(kCols) void beam_tables_kernel(BeamTableArgs a) {
  extern __shared__ int32_t old[];           // [K][kCols], a column its thread's own
  __shared__ int sh_first[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.y, K = a.K, chunk = blockIdx.x;
  const int col = chunk * kCols + tid;
  const int32_t* rows = a.table + (int64_t)b * K * a.stride;
  int32_t* outs = a.out + (int64_t)b * K * a.out_stride;
  const bool in = col < a.width;
  int p = lane < K ? a.parents[(int64_t)b * K + lane] : -1;   // row `lane` goes on from it
  const int len = max(0, a.lens[(int64_t)b * K]);
  const int shared = a.shared ? max(0, a.shared[b]) : 0;
  for (int k0 = 0; k0 < K; k0 += 8) {        // (eight loads on their way at once)
    int32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = in && k0 + i < K ? rows[(k0 + i) * a.stride + col] : -1;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < K) old[(k0 + i) * kCols + tid] = x[i];
  }
  const int full = len / a.page;             // columns of full pages
  const bool part = len % a.page != 0;
  // which row's page row `lane` has in the part-filled page's column (each wave for itself)
  if (p < 0 || p >= K) p = lane;
  uint64_t kids = 0;                         // of row `lane`
  for (int k = 0; k < K; ++k) {
    const uint64_t x = __builtin_amdgcn_ballot_w64(lane < K && p == k);
    if (lane == k) kids = x;
  }
  const int keeper = kids >> lane & 1 ? lane : kids ? __builtin_ctzll(kids) : -1;
  const bool extra = lane < K && __shfl(keeper, p, 64) != lane;
  const uint64_t dead = __builtin_amdgcn_ballot_w64(lane < K && !kids);
  const uint64_t extras = __builtin_amdgcn_ballot_w64(extra);
  int tail = p;
  if (extra) tail = nth_bit(dead, __builtin_popcountll(extras & ((1ull << lane) - 1)));
  // (in place, the shared columns, the same in every row, stay as they are)
  if (in && !(a.out == a.table && col < shared)) {
#pragma unroll 4
    for (int k = 0; k < K; ++k) {
      const int par_k = __builtin_amdgcn_readlane(p, k);
      const int tail_k = __builtin_amdgcn_readlane(tail, k);
      const int from = col < full ? par_k : col == full && part ? tail_k : k;
      outs[k * a.out_stride + col] = old[from * kCols + tid];
    }
  }
  // which page is copied where, by the thread that holds the column (or the last there is)
  if (col == min(full, max(1, a.width) - 1))
    for (int k = 0; k < K; ++k) {
      const int par_k = __builtin_amdgcn_readlane(p, k);
      const int tail_k = __builtin_amdgcn_readlane(tail, k);
      const bool moved = part && full < a.width && tail_k != par_k;
      a.copies[2 * ((int64_t)b * K + k)] = moved ? old[par_k * kCols + tid] : -1;
      a.copies[2 * ((int64_t)b * K + k) + 1] = moved ? old[tail_k * kCols + tid] : -1;
    }

  // pages of full columns that only rows without a child name, each once
  uint64_t gone = 0;
  if (in && col >= shared && col < full)
    for (uint64_t d = dead; d; d &= d - 1) {
      const int k = __builtin_ctzll(d);
      const int slot = old[k * kCols + tid];
      bool held = slot < 0;
      for (int i0 = 0; i0 < K; i0 += 8) {
#pragma unroll
        for (int i = i0; i < i0 + 8; ++i)
          held |= i < K && (i < k || !(dead >> i & 1)) && old[min(i, K - 1) * kCols + tid] == slot;
      }
      if (!held) gone |= 1ull << k;
    }
  const int mine = __builtin_popcountll(gone);
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(incl, d, 64);
    if (lane >= d) incl += x;
  }
  if (lane == 63) sh_first[wave] = incl;
  __syncthreads();
  int at = incl - mine + (wave ? sh_first[0] : 0);
  const int64_t l = (int64_t)b * a.chunks + chunk;
  int32_t* list = a.lists + l * K * kCols;
  for (; gone; gone &= gone - 1) list[at++] = old[__builtin_ctzll(gone) * kCols + tid];
  if (tid == 0) a.counts[l] = sh_first[0] + sh_first[1];
}

struct BeamPools {
  int n, segs, unit_tokens, parts;
  int n_slots;
  int64_t slot, seg;                         // bytes between slots, between a slot's segments
  int64_t unit;                              // bytes of unit_tokens tokens of a segment
  char* at[kPools];
};

// Workgroups x < joins: each its share of the lists of released pages, behind those before.
// The rest: page blockIdx.x - joins of the copies, in pool blockIdx.y, part blockIdx.z.
template <typename W>
__global__ __launch_bounds__(kBeamThreads) void beam_copy_kernel(BeamTableArgs a, BeamPools p,
                                                             int joins) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < joins) {
    if (blockIdx.y || blockIdx.z) return;
    __shared__ int sh[kBeamWaves];
    const int n = a.B * a.chunks, per = (n + joins - 1) / joins;
    const int l0 = min(n, (int)blockIdx.x * per), l1 = min(n, l0 + per);
    int before = 0;
    for (int l = tid; l < l0; l += kBeamThreads) before += a.counts[l];
    int at = block_sum(before, sh);
    for (int l = l0; l < l1; ++l) {
      const int c = a.counts[l];
      for (int i = tid; i < c; i += kBeamThreads)
        a.released[at + i] = a.lists[(int64_t)l * a.K * kCols + i];
      at += c;
    }
    if ((int)blockIdx.x == joins - 1 && tid == 0) *a.n_released = at;
    return;
  }
  const int row = blockIdx.x - joins;
  const int src = a.copies[2 * row], dst = a.copies[2 * row + 1];
  if (src == dst || (uint32_t)src >= (uint32_t)p.n_slots || (uint32_t)dst >= (uint32_t)p.n_slots)
    return;
  const int used = max(0, a.lens[row / a.K * a.K]) % a.page;
  // (a page's tokens stay within 2^31 words: checked on the host)
  const uint32_t words = (uint32_t)((used + p.unit_tokens - 1) / p.unit_tokens * p.unit /
                                    (int64_t)sizeof(W));
  const char* s = p.at[blockIdx.y] + src * p.slot;
  char* d = p.at[blockIdx.y] + dst * p.slot;
  const uint32_t all = words * p.segs;
  constexpr int U = 8;
  for (uint32_t i0 = blockIdx.z * kBeamThreads * U; i0 < all; i0 += p.parts * kBeamThreads * U) {
    W x[U];
    int64_t off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = min(i0 + u * kBeamThreads + tid, all - 1);
      off[u] = i / words * p.seg + (int64_t)(i % words) * sizeof(W);
      x[u] = *reinterpret_cast<const W*>(s + off[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kBeamThreads + tid < all) *reinterpret_cast<W*>(d + off[u]) = x[u];
  }
}

bool tables_ok(int B, int K, int width) {
  return B >= 0 && K >= 1 && K <= HELM_BEAMS_MAX && (int64_t)B * K <= 65535 && width >= 0 &&
         (int64_t)B * K * width <= 0x7fffffff;
}
int table_chunks(int width) { return std::max(1, (width + kCols - 1) / kCols); }

}  // namespace

extern "C" size_t helm_beam_select_workspace_bytes(int B, int K, int V, int n, int dtype) {
  if (!select_ok(B, K, V, n)) return 0;
  return (size_t)select_plan(B, K, V, n, dtype == HELM_F32 ? 4 : 2).bytes;
}

extern "C" int helm_beam_select(const void* logits, int64_t b_stride, int64_t k_stride, int dtype,
                                const float* scores, int B, int K, int V, int n,
                                float* out_scores, int64_t* out_tokens, int32_t* out_parents,
                                void* workspace, size_t ws_bytes, void* stream) {
  using namespace helm;
  if (dtype != HELM_F16 && dtype != HELM_BF16 && dtype != HELM_F32)
    return report_error(HELM_E_UNSUPPORTED, "logits are float16, bfloat16 or float32");
  if (!select_ok(B, K, V, n) || b_stride < 0 || k_stride < 0)
    return report_error(HELM_E_INVALID, "bad beam selection shape (1 to " +
                                            std::to_string(HELM_BEAMS_MAX) +
                                            " beams and candidates, at most 65535 rows)");
  if (B == 0) return HELM_OK;
  if (!logits || !scores || !out_scores || !out_tokens || !out_parents)
    return report_error(HELM_E_INVALID, "null pointer argument");
  const int es = dtype == HELM_F32 ? 4 : 2;
  if (reinterpret_cast<uint64_t>(logits) % es)
    return report_error(HELM_E_INVALID, "logits must be aligned to their elements");
  const SelectPlan p = select_plan(B, K, V, n, es);
  if (!workspace || ws_bytes < (size_t)p.bytes || (reinterpret_cast<uint64_t>(workspace) & 7))
    return report_error(HELM_E_WORKSPACE,
                        "workspace too small or unaligned: need " + std::to_string(p.bytes));
  SelectArgs a{};
  a.logits = logits;
  a.b_stride = b_stride;
  a.k_stride = k_stride;
  a.scores = scores;
  a.B = B;
  a.K = K;
  a.V = V;
  a.n = n;
  a.chunks = p.chunks;
  a.size = p.size;
  const int64_t parts = p.rows * p.chunks;
  a.part_sum = static_cast<double*>(workspace);
  a.part_max = reinterpret_cast<float*>(a.part_sum + parts);
  a.cand_x = a.part_max + parts;
  a.cand_t = reinterpret_cast<int*>(a.cand_x + parts * n);
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_parents = out_parents;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HELM_F32) launch_select<float>(a, p, st);
  else if (dtype == HELM_BF16) launch_select<bf16_t>(a, p, st);
  else launch_select<f16_t>(a, p, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return report_error((int)e, std::string("beam selection launch: ") + hipGetErrorString(e));
  return HELM_OK;
}

extern "C" size_t helm_beam_tables_workspace_bytes(int B, int K, int table_width) {
  if (!tables_ok(B, K, table_width)) return 0;
  return (size_t)B * table_chunks(table_width) * ((size_t)K * kCols + 1) * sizeof(int32_t);
}

extern "C" int helm_beam_tables(const int32_t* parents, int B, int K, const int32_t* page_table,
                                int64_t table_stride, int table_width, const int32_t* seq_lens,
                                int page_size, const int32_t* shared_pages, int32_t* new_table,
                                int64_t new_stride, int32_t* copies, int32_t* released,
                                int32_t* n_released, const void* const* pools, int n_pools,
                                int64_t n_slots, int64_t slot_bytes, int segments,
                                int64_t segment_bytes, int unit_tokens, int64_t unit_bytes,
                                void* workspace, size_t ws_bytes, void* stream) {
  using namespace helm;
  if (!tables_ok(B, K, table_width) || page_size < 1 || table_stride < table_width ||
      new_stride < table_width)
    return report_error(HELM_E_INVALID, "bad beam table shape (1 to " +
                                            std::to_string(HELM_BEAMS_MAX) +
                                            " beams, at most 65535 rows, page_size >= 1)");
  if (n_pools < 0 || (n_pools && (!pools || n_slots < 0 || n_slots > 0x7fffffff || slot_bytes < 0 ||
                                  segments < 1 || segment_bytes < 0 || unit_tokens < 1 ||
                                  unit_bytes < 1)))
    return report_error(HELM_E_INVALID, "bad pool shape");
  const int64_t units = n_pools ? ((int64_t)page_size + unit_tokens - 1) / unit_tokens : 1;
  const int64_t part = n_pools ? units * unit_bytes : 0;     // of a segment
  if (n_pools && (segments > 0x7fffffff / unit_bytes / units || segment_bytes < part ||
                  (n_slots > 1 && slot_bytes < part)))
    return report_error(HELM_E_INVALID, "a page's segments overlap or pass 2^31 bytes");
  for (int i = 0; i < n_pools; ++i)
    if (!pools[i] && n_slots) return report_error(HELM_E_INVALID, "null pool");
  if (B == 0 && !n_released) return report_error(HELM_E_INVALID, "null pointer argument");
  if (B && (!parents || !seq_lens || !copies || !n_released ||
            (table_width && (!page_table || !new_table || !released))))
    return report_error(HELM_E_INVALID, "null pointer argument");
  const size_t need = helm_beam_tables_workspace_bytes(B, K, table_width);
  if (need && (!workspace || ws_bytes < need || (reinterpret_cast<uint64_t>(workspace) & 3)))
    return report_error(HELM_E_WORKSPACE,
                        "workspace too small or unaligned: need " + std::to_string(need));
  const int64_t R = (int64_t)B * K;
  const bool in_place = new_table == page_table && new_stride == table_stride;
  // what is read; what is written
  auto rows = [&](const int32_t* t, int64_t stride) {
    return stride == table_width ? range(t, R * table_width) : range(t, table_width, R, stride);
  };
  const Range r[] = {rows(page_table, table_stride), range(parents, R),
                     range(seq_lens, R), range(shared_pages, shared_pages ? B : 0),
                     rows(new_table, new_stride), range(copies, 2 * R),
                     range(released, R * table_width), range(n_released, 1)};
  constexpr int kOut = 4, kRanges = 8;
  // (overlap takes one row of its first operand: the table's rows one by one)
  auto meet = [](const Range& x, const Range& y) {
    for (int64_t i = 0; i < x.rows; ++i)
      if (overlap({x.at + (uintptr_t)(i * x.step), 1, x.bytes, x.bytes}, y)) return true;
    return false;
  };
  for (int i = kOut; i < kRanges; ++i)
    for (int j = 0; j < i; ++j) {
      if (in_place && i == kOut && j == 0) continue;
      if (j == 0 || j == kOut ? meet(r[i], r[j]) : meet(r[j], r[i]))
        return report_error(HELM_E_INVALID, "an output lies over another operand (new_table may "
                                            "be page_table itself, nothing else)");
    }
  // the pools are written: no operand may lie in one (its parts are looked at where its whole
  // stretch of memory is touched)
  for (int i = 0; i < n_pools && n_slots; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(pools[i]);
    const int64_t all = (n_slots - 1) * slot_bytes + (segments - 1) * segment_bytes + part;
    for (const Range& x : r) {
      if (!x.rows || !x.bytes) continue;
      const int64_t len = (x.rows - 1) * x.step + x.bytes;
      if (!overlap({x.at, 1, len, len}, {at, 1, all, all})) continue;
      for (int64_t j = 0; j < segments; ++j)
        if (meet(x, {at + (uintptr_t)(j * segment_bytes), n_slots, part,
                     n_slots > 1 ? slot_bytes : part}))
          return report_error(HELM_E_INVALID, "an operand lies over a pool's pages");
    }
  }
  BeamTableArgs a{};
  a.parents = parents;
  a.B = B;
  a.K = K;
  a.table = page_table;
  a.stride = table_stride;
  a.width = table_width;
  a.chunks = table_chunks(table_width);
  a.lens = seq_lens;
  a.page = page_size;
  a.shared = shared_pages;
  a.out = new_table;
  a.out_stride = new_stride;
  a.copies = copies;
  a.lists = static_cast<int32_t*>(workspace);
  a.counts = a.lists + (size_t)B * a.chunks * K * kCols;
  a.released = released;
  a.n_released = n_released;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (B)
    hipLaunchKernelGGL(beam_tables_kernel, dim3(a.chunks, B), dim3(kCols),
                       K * kCols * sizeof(int32_t), st, a);
  // 16 bytes a lane where every page's segments allow it; workgroups of 32 KB or more
  BeamPools p{};
  p.n_slots = (int)n_slots;
  p.segs = segments;
  p.unit_tokens = unit_tokens;
  p.slot = slot_bytes;
  p.seg = segment_bytes;
  p.unit = unit_bytes;
  p.parts = (int)std::min<int64_t>(64, std::max<int64_t>(1, units * unit_bytes * segments >> 16));
  int joins = (int)std::max<int64_t>(1, std::min<int64_t>(64, (int64_t)B * a.chunks));
  if (B == 0) n_pools = 0;
  for (int i0 = 0; i0 == 0 || i0 < n_pools; i0 += kPools) {
    p.n = std::min(kPools, n_pools - i0);
    uint64_t bits = (uint64_t)slot_bytes | (uint64_t)segment_bytes | (uint64_t)unit_bytes;
    for (int i = 0; i < p.n; ++i) {
      p.at[i] = static_cast<char*>(const_cast<void*>(pools[i0 + i]));
      bits |= reinterpret_cast<uint64_t>(pools[i0 + i]);
    }
    const dim3 grid((uint32_t)(joins + (p.n ? R : 0)), std::max(1, p.n), p.n ? p.parts : 1);
    if (bits % 16 == 0)
      hipLaunchKernelGGL((beam_copy_kernel<u32x4>), grid, dim3(kBeamThreads), 0, st, a, p, joins);
    else
      hipLaunchKernelGGL((beam_copy_kernel<uint8_t>), grid, dim3(kBeamThreads), 0, st, a, p, joins);
    joins = 0;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return report_error((int)e, std::string("beam tables launch: ") + hipGetErrorString(e));
  return HELM_OK;
}
