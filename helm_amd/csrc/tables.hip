// A serving step's request lengths into block tables, slots, positions and
// offsets (helm_batch_tables).
//
// Sequence b holds c = cached[b] tokens and gets n = new[b] more.  With pages of
// P tokens it owns ceil(c / P) pages already and takes
//   need_b = ceil((c + n) / P) - ceil(c / P)
// further ones from the free list, in sequence order, from where the sequences
// before it stopped (sum of their needs).  Token i of the packed step belongs
// to the sequence with cu[b] <= i < cu[b + 1], cu the running sum of n; its
// position is p = c + i - cu[b], its slot table[b][p / P] * P + p % P.
//
// One launch.  Every workgroup sums all B lengths itself (two running sums in
// LDS, 8 bytes a sequence) and then fills its own share of the tokens and of
// the pages: B is small against the tokens, and a sum in one workgroup that the
// others wait for would cost a second launch.  Entries of the table that this
// call writes are never read by it: a token on a new page takes its slot from
// the free list.  The lengths are read until the last workgroup ends, so no
// output may lie over an input; seq_lens alone may be cached_lens itself (a loop's
// lengths, kept in place), and is then written by a second launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "helm_amd.h"

namespace helm {
int report_error(int code, const std::string& msg);
}

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct TablesArgs {
  const int32_t* new_lens;
  const int32_t* cached_lens;
  int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* free_slots;
  int n_free;
  int page;
  int B;
  int max_tokens;
  int32_t* cu;
  int64_t* positions;
  int64_t* slots;
  int32_t* seq_lens;
  int32_t* taken;
};

__device__ __forceinline__ int clamp_i32(int64_t x) {
  return static_cast<int>(x < 0x7fffffff ? x : 0x7fffffff);
}

// One sequence's lengths (negative ones count as zero) and its pages.
struct Seq {
  int cached, total, old_pages, need;
};
__device__ __forceinline__ Seq load_seq(const TablesArgs& a, int b) {
  Seq s;
  s.cached = max(0, a.cached_lens[b]);
  const int n = max(0, a.new_lens[b]);
  s.total = clamp_i32((int64_t)s.cached + n);
  const unsigned P = a.page;
  s.old_pages = ((unsigned)s.cached + P - 1) / P;
  s.need = (int)(((unsigned)s.total + P - 1) / P) - s.old_pages;
  return s;
}

// Last index b of the ascending run x[0 .. n) with x[b] <= v (x[0] <= v).
__device__ __forceinline__ int last_at_most(const int* x, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void batch_tables_kernel(TablesArgs a) {
  extern __shared__ int lds[];
  int* cu = lds;                 // [B + 1] first token of each sequence
  int* pg = lds + a.B + 1;       // [B + 1] first new page of each sequence
  __shared__ int64_t part[2][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  // running sums: each thread sums its run of sequences, the runs are summed
  // across the workgroup, then each thread writes its run's prefixes
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int64_t tok = 0, pages = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    tok += s.total - s.cached;
    pages += s.need;
  }
  int64_t tok_in = tok, pages_in = pages;      // inclusive over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t t = __shfl_up(tok_in, d, 64), p = __shfl_up(pages_in, d, 64);
    if (lane >= d) {
      tok_in += t;
      pages_in += p;
    }
  }
  if (lane == 63) {
    part[0][wave] = tok_in;
    part[1][wave] = pages_in;
  }
  __syncthreads();
  int64_t t0 = tok_in - tok, p0 = pages_in - pages;
  for (int w = 0; w < wave; ++w) {
    t0 += part[0][w];
    p0 += part[1][w];
  }
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    cu[b] = clamp_i32(t0);
    pg[b] = clamp_i32(p0);
    if (blockIdx.x == 0 && a.seq_lens) a.seq_lens[b] = s.total;
    t0 += s.total - s.cached;
    p0 += s.need;
  }
  if (tid == kThreads - 1) {
    cu[a.B] = clamp_i32(t0);
    pg[a.B] = clamp_i32(p0);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.B; b += kThreads) a.cu[b] = cu[b];
    if (tid == 0) *a.taken = pg[a.B];
  }

  const int gtid = blockIdx.x * kThreads + tid, gsize = gridDim.x * kThreads;
  const unsigned P = a.page;
  // the pages taken, into their rows
  const int n_pages = pg[a.B];
  for (int64_t j = gtid; j < n_pages; j += gsize) {
    const int b = last_at_most(pg, a.B, (int)j);
    const int64_t col = (int64_t)((unsigned)max(0, a.cached_lens[b]) + P - 1) / P + (j - pg[b]);
    if (col < a.width)
      a.table[b * a.table_stride + col] = j < a.n_free ? a.free_slots[j] : -1;
  }
  // the tokens
  const int n_tok = cu[a.B];
  for (int64_t i = gtid; i < a.max_tokens; i += gsize) {
    int64_t pos = 0, slot = -1;
    if (i < n_tok) {
      const int b = last_at_most(cu, a.B, (int)i);
      const int cached = max(0, a.cached_lens[b]);
      pos = (int64_t)cached + (i - cu[b]);
      const int col = (int)((unsigned)pos / P);
      const int old_pages = (int)(((unsigned)cached + P - 1) / P);
      int page = -1;
      if (col < a.width) {
        if (col < old_pages) {
          page = a.table[b * a.table_stride + col];
        } else {
          const int64_t j = (int64_t)pg[b] + (col - old_pages);
          if (j < a.n_free) page = a.free_slots[j];
        }
      }
      if (page >= 0) slot = (int64_t)page * P + ((unsigned)pos % P);
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

// lens[b] += new_lens[b], as load_seq adds them, once the tables are done.
__global__ __launch_bounds__(kThreads) void add_lens_kernel(TablesArgs a, int32_t* lens) {
  const int b = blockIdx.x * kThreads + threadIdx.x;
  if (b < a.B) lens[b] = load_seq(a, b).total;
}

// `rows` rows of `bytes` bytes, `step` (>= bytes) apart.
struct Range {
  uintptr_t at;
  int64_t rows, bytes, step;
};
template <typename T>
Range range(const T* p, int64_t n, int64_t rows = 1, int64_t stride = 0) {
  const int64_t e = sizeof(T);
  return {reinterpret_cast<uintptr_t>(p), rows, n * e, (rows > 1 ? stride : n) * e};
}
// Whether a byte of x (one row) is one of y's.
bool overlap(const Range& x, const Range& y) {
  if (!x.bytes || !y.bytes || !y.rows || x.at + x.bytes <= y.at) return false;
  if (x.at < y.at + y.bytes) return true;
  const int64_t row = (int64_t)(x.at - y.at) / y.step;      // the last that starts at or before x
  if (row >= y.rows) return false;
  const int64_t in = (int64_t)(x.at - y.at) - row * y.step;
  return in < y.bytes || (row + 1 < y.rows && in + x.bytes > y.step);
}

}  // namespace

extern "C" int helm_batch_tables(const int32_t* new_lens, const int32_t* cached_lens, int B,
                                 int32_t* page_table, int64_t table_stride, int table_width,
                                 const int32_t* free_slots, int n_free, int page_size,
                                 int max_tokens, int32_t* cu_seqlens, int64_t* positions,
                                 int64_t* slot_map, int32_t* seq_lens, int32_t* pages_taken,
                                 void* stream) {
  if (B < 1 || B > HELM_TABLES_MAX_SEQS || page_size < 1 || table_width < 0 || n_free < 0 ||
      max_tokens < 0 || table_stride < table_width)
    return helm::report_error(HELM_E_INVALID, "bad batch table shape (1 to " +
                                                  std::to_string(HELM_TABLES_MAX_SEQS) +
                                                  " sequences, page_size >= 1)");
  if (!new_lens || !cached_lens || (!page_table && table_width) || (!free_slots && n_free) ||
      !cu_seqlens || !seq_lens || !pages_taken || (max_tokens && (!positions || !slot_map)))
    return helm::report_error(HELM_E_INVALID, "null pointer argument");
  TablesArgs a{new_lens, cached_lens, page_table, table_stride, table_width, free_slots, n_free,
               page_size, B, max_tokens, cu_seqlens, positions, slot_map, seq_lens, pages_taken};
  // the table (read and written), what is only read, what is only written
  const bool in_place = seq_lens == cached_lens;
  const Range r[] = {range(page_table, table_width, B, table_stride),
                     range(new_lens, B), range(cached_lens, B), range(free_slots, n_free),
                     range(cu_seqlens, B + 1), range(positions, max_tokens),
                     range(slot_map, max_tokens), range(seq_lens, B), range(pages_taken, 1)};
  constexpr int kIn = 1, kCached = 2, kOut = 4, kLens = 7, kRanges = 9;
  for (int i = kIn; i < kRanges; ++i)
    for (int j = 0; j < std::min(i, i < kOut ? kIn : kRanges); ++j)
      if (overlap(r[i], r[j]) && !(in_place && i == kLens && j == kCached))
        return helm::report_error(HELM_E_INVALID,
                                  "an output lies over another operand (seq_lens may be "
                                  "cached_lens itself, nothing else)");
  if (in_place) a.seq_lens = nullptr;
  const int grid = std::max(1, std::min(256, (max_tokens + 2 * kThreads - 1) / (2 * kThreads)));
  hipLaunchKernelGGL(batch_tables_kernel, dim3(grid), dim3(kThreads), 2 * (B + 1) * sizeof(int),
                     reinterpret_cast<hipStream_t>(stream), a);
  if (in_place)
    hipLaunchKernelGGL(add_lens_kernel, dim3((B + kThreads - 1) / kThreads), dim3(kThreads), 0,
                       reinterpret_cast<hipStream_t>(stream), a, seq_lens);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return helm::report_error((int)e, std::string("batch tables launch: ") + hipGetErrorString(e));
  return HELM_OK;
}
