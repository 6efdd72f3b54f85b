// Decode attention of sequences that share their first pages (helm_prefix_decode_attn): row
// (r, h, s) of a sequence of len tokens stands at position p = len - S + s and gets
// softmax(cap(q . K^T scale)) . V over its tokens j <= p (and j > p - window).
//
// A group's shared pages are walked once for the rows of all its sequences, a sequence's
// own pages for its own S G rows a KV head; every walk leaves partial sums (m, l, o) of its
// rows over its tokens, and a second kernel joins a row's:
//   out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i,  M = max m_i.
// Bound by memory up to some 400 rows a KV head (4 D operations a row and token against
// 4 D bytes a token), by the matrix cores beyond.
//
// Work: a KV head's walks, the groups' row tiles first, then the sequences', lie end to end on
// one line, a step of 32 tokens weighing what it costs, and each of the head's workgroups takes
// an equal stretch of it, whatever the lengths are: the launch depends on none.  Every
// workgroup sums the lengths up for itself.  A piece of a walk on workgroup w leaves its
// partials at slot (walk + w), of which no two pieces are alike, as both only grow along the line.
//
// A walk has 32 rows and 32 x 32 matrix tiles, with the operands' layouts of prompt.h: lane
// l = 32 hh + jr owns row jr, the two lanes of a row hold its scores, maximum, sum and output.
// The four waves of the workgroup deal its steps out among them, each through K and V buffers
// of its own, one step ahead, with no barrier in the walk, and join their sums in LDS.
// Weights enter P . V in two 16-bit parts (~2^-17 of the weight; f16 taken times 2^9).
//
// Hidden tokens (past a row's position or out of its window, past a sequence's end, in pages
// that the pool does not have) take no part whatever they hold: their scores are overwritten,
// and an infinity or NaN in V shows as NaN in an output, upon which the wave walks again with V's
// infinities and NaN taken out of the products and added where a row sees them (careful).
#pragma once

#include <type_traits>

#include "attn_chunk32.h"
#include "prompt.h"

namespace helm {

constexpr int kPfThreads = 256;
constexpr int kPfWaves = kPfThreads / 64;
constexpr int kPfRows = 32;          // of a walk, and of a slot of the groups' partials
constexpr int kPfStep = 32;          // tokens of a step
// a workgroup's least stretch: a step for each wave
constexpr int kPfLeast = kPfWaves;

struct PfParams {
  const char *q, *k, *v;
  char* out;
  int64_t slot, head;                // bytes between slots, between a slot's KV heads
  int n_slots;
  const int32_t* table;
  int64_t table_stride;
  int max_pages, page, bpp;          // bpp: 16-token blocks of a page
  const int32_t *lens, *starts, *shared;
  int n_groups, R, Hq, Hkv, G, S;
  int wgs;                           // workgroups of a KV head
  int own_tiles, own_rows;           // walks of a sequence's own pages; rows of their slots
  int group_slots, own_slots;        // slots of a KV head's partials
  float scale;                       // >= 0 (a negative one's sign is taken into q)
  uint32_t q_sign;
  float softcap;
  int window;                        // <= 0: off
  // workspace
  struct PfSeq* seqs;                // [R], for the joining kernel
  float *group_ml, *group_o, *own_ml, *own_o;
};

// Where the partials of sequence r's rows are: the line's stretches [at, at + tiles * each).
struct PfSeq {
  int row0;                          // its first row among its group's
  int group_at, group_each, group_slot;   // each: a tile's length, 0: no walk
  int own_at, own_each;
  int stretch;                       // of a workgroup
  int pad;
};

// What sequence r sees: tokens [first, end) of its table, of them `shared` in its group's pages.
struct PfView {
  int first, end;
};
__device__ __forceinline__ int pf_room(const PfParams& p) { return p.max_pages * p.page; }
__device__ __forceinline__ PfView pf_view(const PfParams& p, int len) {
  const int end = min(max(len, 0), pf_room(p));
  const int first = p.window > 0 ? max(0, end - p.S + 1 - p.window) : 0;
  return {min(first, end) & ~15, end};
}
// Tokens in the shared pages of group g.
__device__ __forceinline__ int pf_shared(const PfParams& p, int pages) {
  return min(max(pages, 0), p.max_pages) * p.page;
}
__device__ __forceinline__ int pf_steps(int first, int end) {
  return end > first ? (end - first + kPfStep - 1) / kPfStep : 0;
}

// LDS of the start, where K and V are later: the groups' tables and sums.
constexpr int kPfMaxGroups = 1024;
struct PfStart {
  int starts[kPfMaxGroups + 1];
  int shared[kPfMaxGroups];          // tokens
  int lo[kPfMaxGroups], hi[kPfMaxGroups];
  int at[kPfMaxGroups], slot[kPfMaxGroups];
};

// A walk's rows and tokens.
struct PfWalk {
  int seq0, rows;                    // rows of it and those of its entity behind it
  int row0;                          // its first among its entity's
  int first, end;                    // tokens
};

template <typename T, int D, bool kCap>
struct PfBody {
  static constexpr int NK = D / 16, NE = D / 32, CPR = D / 8;
  static constexpr int kRow = 2 * D, kBlk = kBlockTok * kRow;
  static constexpr int kBlkLoads = kBlk / 1024;
  static constexpr int kShift = std::is_same<T, f16_t>::value ? 9 : 0;
  using Ops = MfmaOps<T>;
  using M32 = Mfma32<T>;
  typedef mf_u32x4 Buf[kPfWaves][2][kBlk / 16];     // [wave][block of the step][chunk]
};

// Steps [i0, i1) of walk w of KV head hk; partials of its row r to ml[2 r], o[r D].
template <typename T, int D, bool kCap>
__device__ __forceinline__ void pf_walk(const PfParams& p, const PfWalk& w, int hk, int i0, int i1,
                                        float* ml, float* part,
                                        typename PfBody<T, D, kCap>::Buf& ldsk,
                                        typename PfBody<T, D, kCap>::Buf& ldsv) {
  using Body = PfBody<T, D, kCap>;
  using Ops = typename Body::Ops;
  using M32 = typename Body::M32;
  constexpr int NK = Body::NK, NE = Body::NE, CPR = Body::CPR, kRow = Body::kRow;
  constexpr int kBlk = Body::kBlk, kBlkLoads = Body::kBlkLoads, kShift = Body::kShift;
  constexpr int kOwnLoads = 2 * kBlkLoads;          // of a step's K or V
  constexpr float kSlack = chunk_slack(kShift);
  __shared__ float tops[kPfWaves][kPfRows], sums[kPfWaves][kPfRows];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, jr = lane & 31, hh = lane >> 5;

  // ---- row jr: its sequence, head and position; what it sees
  const int nrows = min(kPfRows, w.rows);
  const bool row_ok = jr < nrows;
  const int row = w.row0 + (row_ok ? jr : 0);
  const int sg = p.S * p.G;
  const int seq = w.seq0 + row / sg, s_row = row % sg / p.G, hq = hk * p.G + row % p.G;
  const int len = min(max(p.lens[seq], 0), pf_room(p));
  const int last = row_ok ? min(len - p.S + s_row, w.end - 1) : -1;
  const int from = p.window > 0 ? max(0, len - p.S + s_row - p.window + 1) : 0;
  // the rows' first last and last first tokens: steps between need no test
  int all_to = row_ok ? last : 0x7fffffff, all_from = row_ok ? from : 0;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    all_to = min(all_to, __shfl_xor(all_to, d, 64));
    all_from = max(all_from, __shfl_xor(all_from, d, 64));
  }
  all_to = __builtin_amdgcn_readfirstlane(all_to);
  all_from = __builtin_amdgcn_readfirstlane(all_from);
  mf_u32x4 qop[NK];
  {
    const char* qp = p.q + (((int64_t)seq * p.Hq + hq) * p.S + s_row) * kRow;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const mf_u32x4 x = *reinterpret_cast<const mf_u32x4*>(qp + 16 * (2 * i + hh));
      qop[i] = row_ok ? x ^ p.q_sign : mf_u32x4{0u, 0u, 0u, 0u};
    }
  }

  // ---- pages: lane 2 k + u holds block u of the wave's step win + k
  const int64_t trow = (int64_t)w.seq0 * p.table_stride;
  struct Window {
    int slot, in;                    // the block's slot (-1: none) and its place in the page
  };
  auto window = [&](int k0) -> Window {
    const int step = i0 + wave + kPfWaves * (k0 + (lane >> 1));
    const int block = (w.first >> 4) + 2 * step + (lane & 1);
    const int page = block / p.bpp;
    return {step < i1 && page < p.max_pages ? p.table[trow + page] : -1, block - page * p.bpp};
  };
  constexpr int kWin = 32;
  Window win, win_next;
  int win0;

  const char* kb = p.k + hk * p.head;
  const char* vb = p.v + hk * p.head;
  // the loads of the wave's step k, K or V, straight into LDS; tokens past the walk's end and
  // pages that are not there come in as zeros
  auto dma = [&](int k, const char* base, mf_u32x4 (*dst)[kBlk / 16]) {
    const int step = i0 + wave + kPfWaves * k;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int slot = __builtin_amdgcn_readlane(win.slot, (2 * (k - win0) + u) & 63);
      const int in = __builtin_amdgcn_readlane(win.in, (2 * (k - win0) + u) & 63);
      const int nt = min(max(w.end - (w.first + kPfStep * step + 16 * u), 0), kBlockTok);
      const bool there = step < i1 && (uint32_t)slot < (uint32_t)p.n_slots;
      const auto rs = make_rsrc(base + (there ? slot : 0) * p.slot + (int64_t)(there ? in : 0) * kBlk,
                                there ? nt * kRow : 0);
#pragma unroll
      for (int l = 0; l < kBlkLoads; ++l) {
        const int t = (64 / CPR) * l + lane / CPR;
        buf_load16_lds(rs, &dst[u][64 * l], t * kRow + 16 * ((lane % CPR) ^ swz<D>(t)));
      }
    }
  };
  auto gone_blocks = [&](int k) {
    int gone = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if ((uint32_t)__builtin_amdgcn_readlane(win.slot, (2 * (k - win0) + u) & 63) >=
          (uint32_t)p.n_slots)
        gone |= 1 << u;
    return gone;
  };
  // (every LDS read so far has returned)
  auto reads_done = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // all loads into LDS but the youngest kOwnLoads have landed
  auto older_landed = [&] {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOwnLoads) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- a step's operands in LDS (prompt.h)
  const int g_a = jr >> 3, h_a = (jr >> 2) & 1, t_a = jr & 3;
  const int tau = 16 * (g_a >> 1) + 8 * h_a + 4 * (g_a & 1) + t_a;
  const int kblk = tau >> 4, ktok = tau & 15, nl = lane & 15;
  const int k_off = kblk * kBlk + ktok * kRow + 16 * (hh ^ swz<D>(ktok));
  const int v_tok0 = 8 * hh + (nl >> 2);
  const int v_off = v_tok0 * kRow + 16 * ((2 * (jr >> 4) + ((nl & 3) >> 1)) ^ swz<D>(v_tok0)) +
                    8 * (nl & 1);
  auto k_operand = [&](const char* kk, int i) {
    return *reinterpret_cast<const mf_u32x4*>(kk + (k_off ^ (32 * i)));
  };
  auto v_operand = [&](const char* vv, int u, int z, int e) {
    return ld_tr16(vv + (v_off ^ (64 * e) ^ (16 * z)) + u * kBlk + 4 * kRow * z);
  };

  const float scale2 = p.scale * kLog2E;
  const float inv_cap = kCap ? 1.f / p.softcap : 0.f, cap2 = p.softcap * kLog2E;
  const float mul = kCap ? 1.f : scale2;             // logits in base-2 units
  float m, lsum;
  mf_f32x16 o[NE];

  auto step = [&](auto careful, int k) {
    const int tok0 = w.first + kPfStep * (i0 + wave + kPfWaves * k);
    const int gone = gone_blocks(k);
    const char* kk = reinterpret_cast<const char*>(&ldsk[wave][0][0]);
    const char* vv = reinterpret_cast<const char*>(&ldsv[wave][0][0]);
    older_landed();                                  // K
    mf_f32x16 sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NK; ++i) sc = M32::mma(k_operand(kk, i), qop[i], sc);
    reads_done();
    if (k + 1 == win0 + kWin) {
      win = win_next;
      win0 += kWin;
      win_next = window(win0 + kWin);
    }
    dma(k + 1, kb, ldsk[wave]);                      // (past the last: nothing, zeros)
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = sc[r];
    if constexpr (kCap) softcap_scores<16>(x, p.scale * inv_cap, cap2);
    if (gone || tok0 + 31 > all_to || tok0 < all_from) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int t = tok0 + 16 * (r >> 3) + 8 * hh + (r & 7);
        if (t > last || t < from || (gone >> (r >> 3) & 1)) x[r] = -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top *= mul;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0, 0)) {
      float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
      if constexpr (kShift) mn = ceilf(mn);          // (so that m - kShift is exact)
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      lsum *= f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        if constexpr (careful.value) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[e][r] = scale_finite(o[e][r], f);
        } else {
          o[e] *= f;
        }
      }
    }
    const float base = m == -INFINITY ? 0.f : m - kShift;
    uint32_t hi[8], lo[8];
    uint32_t some[8];                                // careful: 1 where the row sees the token
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w0 = __builtin_amdgcn_exp2f(fmaf(x[2 * i], mul, -base));
      const float w1 = __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], mul, -base));
      Ops::split2(w0, w1, hi[i], lo[i]);
      lsum += w0 + w1;
      if constexpr (careful.value) {
        const uint32_t one = Ops::ones8()[0];
        some[i] = (x[2 * i] != -INFINITY ? one & 0xffffu : 0u) |
                  (x[2 * i + 1] != -INFINITY ? one & 0xffff0000u : 0u);
      }
    }
    older_landed();                                  // V
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const mf_u32x4 ph{hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]};
      const mf_u32x4 pl{lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]};
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const uint2 a0 = v_operand(vv, u, 0, e);
        const uint2 a1 = v_operand(vv, u, 1, e);
        mf_u32x4 vop{a0.x, a0.y, a1.x, a1.y};
        if constexpr (careful.value) {
          const mf_u32x4 sop{some[4 * u], some[4 * u + 1], some[4 * u + 2], some[4 * u + 3]};
          careful_v<T>(vop, sop, o[e]);
        }
        o[e] = M32::mma(vop, ph, o[e]);
        o[e] = M32::mma(vop, pl, o[e]);
      }
    }
    reads_done();
    dma(k + 1, vb, ldsv[wave]);
  };
  const int steps = i0 + wave < i1 ? (i1 - i0 - wave - 1) / kPfWaves + 1 : 0;
  auto walk = [&](auto careful) {
    m = -INFINITY;
    lsum = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[e][r] = 0.f;
    win = window(0);
    win_next = window(kWin);
    win0 = 0;
    if (steps) {
      dma(0, kb, ldsk[wave]);
      __builtin_amdgcn_sched_barrier(0);             // (K's loads are the older ones)
      dma(0, vb, ldsv[wave]);
    }
    for (int k = 0; k < steps; ++k) step(careful, k);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (no load is on its way any more)
  };
  walk(std::false_type{});
  bool odd = false;
#pragma unroll
  for (int e = 0; e < NE; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = odd || o[e][r] != o[e][r];
  if (__builtin_amdgcn_ballot_w64(odd && row_ok)) walk(std::true_type{});

  // ---- the waves' sums joined, through LDS where K (the first half of the dims) and V were
  lsum += __shfl_xor(lsum, 32, 64);
  if (hh == 0) tops[wave][jr] = m;
  __syncthreads();
  float top = tops[0][jr];
#pragma unroll
  for (int i = 1; i < kPfWaves; ++i) top = fmaxf(top, tops[i][jr]);
  const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
  if (hh == 0) sums[wave][jr] = lsum * f;
  auto at = [&](int i, int c, int h, int r) {
    return reinterpret_cast<mf_f32x4*>(c < CPR / 2 ? &ldsk[0][0][0] : &ldsv[0][0][0]) + 4 * D * i +
           64 * (c % (CPR / 2)) + 32 * h + (r ^ c % 16);
  };
#pragma unroll
  for (int c = 0; c < CPR; ++c) {
    mf_f32x4 x;
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = scale_finite(o[c / 4][4 * (c % 4) + t], f);
    *at(wave, c, hh, jr) = x;
  }
  __syncthreads();
  for (int i = tid; i < nrows * CPR; i += kPfThreads) {
    const int r = i / CPR, c = i % CPR;
    mf_f32x4 a{0.f, 0.f, 0.f, 0.f}, b{0.f, 0.f, 0.f, 0.f};
    float l = 0.f, mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPfWaves; ++j) {
      l += sums[j][r];
      mx = fmaxf(mx, tops[j][r]);
      a += *at(j, c, 0, r);
      b += *at(j, c, 1, r);
    }
    mf_f32x4* dst = reinterpret_cast<mf_f32x4*>(part + (int64_t)r * D + 8 * c);
    dst[0] = a;
    dst[1] = b;
    if (c == 0) *reinterpret_cast<float2*>(ml + 2 * r) = make_float2(mx, l);
  }
  __syncthreads();                                   // (the next walk fills the buffers)
}

template <typename T, int D, bool kCap>
__global__ __launch_bounds__(kPfThreads, D == 256 ? 1 : 2) void prefix_attn_kernel(PfParams p) {
  using Body = PfBody<T, D, kCap>;
  typedef typename Body::Buf Buf;
  // K and V of the waves' steps; before that, the start's tables
  __shared__ union Lds {
    __device__ Lds() {}
    Buf buf;
    PfStart start;
  } lds;
  __shared__ Buf ldsv;
  static_assert(sizeof(PfStart) <= 32768, "the start's tables");
  extern __shared__ int own_first[];                 // [R] a sequence's first own token
  __shared__ int sh_sum[kPfWaves + 1], sh_found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hk = blockIdx.x % p.Hkv, wg = blockIdx.x / p.Hkv;
  PfStart& st = lds.start;

  // ---- the line: lengths of the groups' walks, then of the sequences'
  for (int g = tid; g <= p.n_groups; g += kPfThreads)
    st.starts[g] = min(max(p.starts[g], 0), p.R);
  for (int g = tid; g < p.n_groups; g += kPfThreads) {
    st.shared[g] = pf_shared(p, p.shared[g]);
    st.lo[g] = 0x7fffffff;
    st.hi[g] = 0;
  }
  __syncthreads();
  auto group_of = [&](int r) {                       // -1: none
    int lo = 0, hi = p.n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (st.starts[mid] <= r) lo = mid;
      else hi = mid;
    }
    return p.n_groups && st.starts[lo] <= r && r < st.starts[lo + 1] ? lo : -1;
  };
  for (int r = tid; r < p.R; r += kPfThreads) {
    const PfView v = pf_view(p, p.lens[r]);
    const int g = group_of(r), sh = g < 0 ? 0 : st.shared[g];
    if (g >= 0) {
      atomicMin(&st.lo[g], v.first);
      atomicMax(&st.hi[g], min(v.end, sh));
    }
    own_first[r] = max(sh, v.first);
  }
  __syncthreads();
  auto group_walk = [&](int g) { return pf_steps(st.lo[g], st.hi[g]); };
  auto group_rows = [&](int g) { return max(0, st.starts[g + 1] - st.starts[g]) * p.S * p.G; };
  auto own_walk = [&](int r) { return pf_steps(own_first[r], pf_view(p, p.lens[r]).end); };
  const int E = p.n_groups + p.R;
  auto length = [&](int e) {
    return e < p.n_groups ? (group_rows(e) + kPfRows - 1) / kPfRows * group_walk(e)
                          : p.own_tiles * own_walk(e - p.n_groups);
  };
  // running sums: each thread sums a run of entities, of lengths and of groups' slots
  const int per = (E + kPfThreads - 1) / kPfThreads;
  const int e0 = min(E, tid * per), e1 = min(E, e0 + per);
  int sum = 0, slots = 0;
  for (int e = e0; e < e1; ++e) {
    sum += length(e);
    if (e < p.n_groups) slots += (group_rows(e) + kPfRows - 1) / kPfRows;
  }
  int at = sum, slot = slots;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(at, d, 64), y = __shfl_up(slot, d, 64);
    if (lane >= d) {
      at += x;
      slot += y;
    }
  }
  __shared__ int sh_slot[kPfWaves];
  if (lane == 63) {
    sh_sum[wave] = at;
    sh_slot[wave] = slot;
  }
  __syncthreads();
  at -= sum;
  slot -= slots;
  int total = 0;
  for (int i = 0; i < kPfWaves; ++i) {
    if (i < wave) {
      at += sh_sum[i];
      slot += sh_slot[i];
    }
    total += sh_sum[i];
  }
  const int stretch = max(kPfLeast, (total + p.wgs - 1) / p.wgs);
  const int a = wg * stretch, b = min(a + stretch, total);
  if (tid == 0) sh_found[0] = -1;
  __syncthreads();
  for (int e = e0, x = at, y = slot; e < e1; ++e) {
    const int n = length(e);
    if (blockIdx.x == 0 && e < p.n_groups) {
      st.at[e] = x;
      st.slot[e] = y;
    }
    if (blockIdx.x == 0 && e >= p.n_groups) {
      PfSeq& q = p.seqs[e - p.n_groups];
      q.own_at = x;
      q.own_each = p.own_tiles ? n / p.own_tiles : 0;
      q.stretch = stretch;
    }
    if (a >= x && a < x + n) {
      sh_found[0] = e;
      sh_found[1] = x;
      sh_found[2] = y;
    }
    x += n;
    if (e < p.n_groups) y += (group_rows(e) + kPfRows - 1) / kPfRows;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int r = tid; r < p.R; r += kPfThreads) {
      const int g = group_of(r);
      PfSeq& q = p.seqs[r];
      q.row0 = g < 0 ? 0 : (r - st.starts[g]) * p.S * p.G;
      q.group_at = g < 0 ? 0 : st.at[g];
      q.group_slot = g < 0 ? 0 : st.slot[g];
      q.group_each = g < 0 ? 0 : group_walk(g);
    }
  if (a >= b) return;
  int e = __builtin_amdgcn_readfirstlane(sh_found[0]);
  int x = __builtin_amdgcn_readfirstlane(sh_found[1]);
  int y = __builtin_amdgcn_readfirstlane(sh_found[2]);
  __syncthreads();                                   // (the walks' buffers may be written)
  if (e < 0) return;

  // ---- the workgroup's stretch [a, b), walk by walk
  for (; e < E && x < b; ++e) {
    PfWalk w;
    int tiles, rows;
    if (e < p.n_groups) {
      // (the group's numbers again, from memory: the tables in LDS are gone)
      w.seq0 = min(max(p.starts[e], 0), p.R);
      const int n = max(0, min(max(p.starts[e + 1], 0), p.R) - w.seq0);
      const int sh = pf_shared(p, p.shared[e]);
      rows = n * p.S * p.G;
      tiles = (rows + kPfRows - 1) / kPfRows;
      int lo = 0x7fffffff, hi = 0;
      for (int i = lane; i < n; i += 64) {
        const PfView v = pf_view(p, p.lens[w.seq0 + i]);
        lo = min(lo, v.first);
        hi = max(hi, min(v.end, sh));
      }
#pragma unroll
      for (int d = 32; d; d >>= 1) {
        lo = min(lo, __shfl_xor(lo, d, 64));
        hi = max(hi, __shfl_xor(hi, d, 64));
      }
      w.first = __builtin_amdgcn_readfirstlane(lo);
      w.end = __builtin_amdgcn_readfirstlane(hi);
    } else {
      w.seq0 = e - p.n_groups;
      w.first = own_first[w.seq0];
      w.end = pf_view(p, p.lens[w.seq0]).end;
      rows = p.S * p.G;
      tiles = p.own_tiles;
    }
    const int steps = pf_steps(w.first, w.end), n = tiles * steps;
    if (steps)
      for (int t = max(0, (a - x) / steps); t < tiles && x + t * steps < b; ++t) {
        const int from = x + t * steps;
        const int i0 = max(a - from, 0), i1 = min(b - from, steps);
        w.row0 = kPfRows * t;
        w.rows = rows - w.row0;
        float *ml, *o;
        if (e < p.n_groups) {
          const int s = y + t + wg;
          if (s >= p.group_slots) continue;          // (starts that do not ascend)
          const int64_t at = ((int64_t)hk * p.group_slots + s) * kPfRows;
          ml = p.group_ml + 2 * at;
          o = p.group_o + at * D;
        } else {
          const int64_t at =
              ((int64_t)hk * p.own_slots + w.seq0 * p.own_tiles + t + wg) * p.own_rows;
          ml = p.own_ml + 2 * at;
          o = p.own_o + at * D;
        }
        if (i0 < i1) pf_walk<T, D, kCap>(p, w, hk, i0, i1, ml, o, lds.buf, ldsv);
      }
    x += n;
    if (e < p.n_groups) y += tiles;
  }
}

// Row blockIdx.x of the output, (r, hq, s), from its walks' partials.
template <typename T, int D>
__global__ __launch_bounds__(kPfThreads) void prefix_join_kernel(PfParams p) {
  constexpr int C = D / 4, N = kPfThreads / C, U = 4;
  __shared__ float4 sh_o[N][C];
  __shared__ float2 sh_ml[N];
  using Ops = MfmaOps<T>;
  const int s = blockIdx.x % p.S, hq = blockIdx.x / p.S % p.Hq, r = blockIdx.x / p.S / p.Hq;
  const int hk = hq / p.G, row = s * p.G + hq % p.G;
  const PfSeq q = p.seqs[r];
  // the pieces of a walk at [at, at + each) of the line: on workgroups at / stretch and on
  auto pieces = [&](int from, int each, int& w0) {
    w0 = from / q.stretch;
    return each > 0 ? (from + each - 1) / q.stretch - w0 + 1 : 0;
  };
  const int grow = q.row0 + row, gt = grow / kPfRows, ot = row / kPfRows;
  int w0, v0;
  int n_group = pieces(q.group_at + gt * q.group_each, q.group_each, w0);
  const int n_own = pieces(q.own_at + ot * q.own_each, q.own_each, v0);
  const int g0 = q.group_slot + gt + w0, o0 = r * p.own_tiles + ot + v0;
  n_group = min(n_group, max(0, p.group_slots - g0));
  const int n = n_group + n_own;
  const int c = threadIdx.x % C, g = threadIdx.x / C;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = g; i0 < n; i0 += U * N) {
    float2 ml[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * N, n - 1);
      if (i < n_group) {
        const int64_t at = ((int64_t)hk * p.group_slots + g0 + i) * kPfRows + grow % kPfRows;
        ml[u] = reinterpret_cast<const float2*>(p.group_ml)[at];
        v[u] = reinterpret_cast<const float4*>(p.group_o)[at * C + c];
      } else {
        const int64_t at = ((int64_t)hk * p.own_slots + o0 + i - n_group) * p.own_rows + row % kPfRows;
        ml[u] = reinterpret_cast<const float2*>(p.own_ml)[at];
        v[u] = reinterpret_cast<const float4*>(p.own_o)[at * C + c];
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * N < n) mn = fmaxf(mn, ml[u].x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - base);
    l *= f;
    acc = make_float4(scale_finite(acc.x, f), scale_finite(acc.y, f), scale_finite(acc.z, f),
                      scale_finite(acc.w, f));
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * N < n) {
        const float x = __builtin_amdgcn_exp2f(ml[u].x - base);
        l += x * ml[u].y;
        acc.x += scale_finite(v[u].x, x);
        acc.y += scale_finite(v[u].y, x);
        acc.z += scale_finite(v[u].z, x);
        acc.w += scale_finite(v[u].w, x);
      }
  }
  sh_o[g][c] = acc;
  if (c == 0) sh_ml[g] = make_float2(m, l);
  __syncthreads();
  if (g > 0) return;
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, sh_ml[i].x);
  const float base = mx == -INFINITY ? 0.f : mx;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 x = sh_ml[i];
    const float f = __builtin_amdgcn_exp2f(x.x - base);
    sum += f * x.y;
    const float4 v = sh_o[i][c];
    acc.x += scale_finite(v.x, f);
    acc.y += scale_finite(v.y, f);
    acc.z += scale_finite(v.z, f);
    acc.w += scale_finite(v.w, f);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(p.out + ((int64_t)blockIdx.x * D + 4 * c) * 2) =
      make_uint2(Ops::pk(acc.x * inv, acc.y * inv), Ops::pk(acc.z * inv, acc.w * inv));
}

template <typename T, int D>
hipError_t launch_prefix_dim(const PfParams& p, hipStream_t st) {
  const dim3 grid((uint32_t)(p.Hkv * p.wgs));
  const size_t dyn = sizeof(int) * (size_t)p.R;
  if (p.softcap > 0.f)
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, true>), grid, dim3(kPfThreads), dyn, st, p);
  else
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, false>), grid, dim3(kPfThreads), dyn, st, p);
  hipLaunchKernelGGL((prefix_join_kernel<T, D>), dim3((uint32_t)(p.R * p.Hq * p.S)),
                     dim3(kPfThreads), 0, st, p);
  return hipGetLastError();
}

// One per element type, each in a source of its own (prefix_bf16.hip, prefix_f16.hip).
hipError_t launch_prefix_bf16(const PfParams& p, int D, hipStream_t st);
hipError_t launch_prefix_f16(const PfParams& p, int D, hipStream_t st);

template <typename T>
hipError_t launch_prefix_type(const PfParams& p, int D, hipStream_t st) {
  if (D == 64) return launch_prefix_dim<T, 64>(p, st);
  if (D == 128) return launch_prefix_dim<T, 128>(p, st);
  return launch_prefix_dim<T, 256>(p, st);
}

}  // namespace helm
