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
// Work: a workgroup a CU, each with a KV head.  A head's walks over shared pages lie end to
// end on one line of steps of 32 tokens, and each of the head's workgroups takes an equal
// stretch of it; the walks over own pages on another, shared out among the head's waves.  So
// any lengths are spread evenly, and the launch depends on none: every workgroup sums them up
// for itself.  A piece of a walk leaves its partials at slot (walk + workgroup or wave), of which
// no two pieces are alike, as both only grow along the line.
//
// 32 x 32 matrix tiles, with the operands' layouts of prompt.h: lane l = 32 hh + jr owns row
// jr, the two lanes of a row hold its scores, maximum, sum and output.  Three forms of a walk:
//   own     a wave by itself: K and V of a step go straight into LDS buffers of its own, one
//           step ahead; no barrier;
//   dealt   up to 32 rows of a group: the workgroup's waves deal the steps of its stretch
//           out among them, each as above, and join their sums in LDS;
//   wide    more rows: each wave owns 32 of them, all share each stage of K and V (two stage
//           buffers, one barrier a stage), which so are read once for up to 32 rows a wave.
// Weights enter P . V in two 16-bit parts (~2^-17 of the weight), in wide walks, where the
// matrix cores have the most to do, rounded once (2^-8 of it in bf16, 2^-11 in f16, and the
// row's sum adds the rounded ones); f16 weights are taken times 2^9.
//
// Hidden tokens (past a row's position or out of its window, past a sequence's end, in pages
// that the pool does not have) take no part whatever they hold: their scores are overwritten,
// and an infinity or NaN in V shows as NaN in an output, upon which the walk is done again with
// V's infinities and NaN taken for zeros in LDS (careful), and they are added to the partials of
// the rows that see them.
#pragma once

#include <type_traits>

#include "attn_chunk32.h"
#include "prompt.h"

namespace helm {

constexpr int kPfRows = 32;          // of a wave, and of a slot of the groups' partials
constexpr int kPfStep = 32;          // tokens of a step
constexpr int kPfOwnLeast = 4;       // a wave's least stretch of the own walks
constexpr int kPfJoinThreads = 256;
// Waves of a workgroup: K and V buffers of 64 D bytes each a wave, 128 KB in all (64 at D = 64).
constexpr int pf_waves(int D) { return D == 256 ? 4 : 8; }

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

// Where the partials of sequence r's rows are: walk t is steps [at + t each, at + (t + 1) each)
// of its line.
struct PfSeq {
  int row0;                          // its first row among its group's
  int tile_rows;                     // rows of its group's walks
  int group_at, group_each, group_slot, group_stretch;
  int own_at, own_each, own_stretch;
  int pad[3];
};

// What a sequence of len tokens sees: [first, end) of its table, first a block's.
struct PfView {
  int first, end;
};
__device__ __forceinline__ int pf_room(const PfParams& p) { return p.max_pages * p.page; }
__device__ __forceinline__ PfView pf_view(const PfParams& p, int len) {
  const int end = min(max(len, 0), pf_room(p));
  const int first = p.window > 0 ? max(0, end - p.S + 1 - p.window) : 0;
  return {min(first, end) & ~15, end};
}
// Tokens in the shared pages of a group.
__device__ __forceinline__ int pf_shared(const PfParams& p, int pages) {
  return min(max(pages, 0), p.max_pages) * p.page;
}
__device__ __forceinline__ int pf_steps(int first, int end) {
  return end > first ? (end - first + kPfStep - 1) / kPfStep : 0;
}
// A group in LDS: its first sequence, the tokens in its shared pages, and of those the ones that
// any of its sequences sees, [lo, hi).
struct PfGroup {
  int start, shared, lo, hi;
};
// where the groups' walks and slots start (for the joining kernel), before K and V come there
struct PfAt {
  int at[HELM_PREFIX_MAX_GROUPS], slot[HELM_PREFIX_MAX_GROUPS];
};

template <typename T, int D>
struct PfBuf {
  static constexpr int kChunks = 2 * D;                // 16-byte chunks of a block
  // a wave's K (or V) of a step; or, over all waves, a stage of 16 tokens a wave, K and then V
  typedef mf_u32x4 type[pf_waves(D)][2][kChunks];
};

// A walk's piece: rows [row0, row0 + rows) of sequences seq0 .. (S G rows each), steps [i0, i1)
// of tokens [first, end).
struct PfPiece {
  int seq0, row0, rows, first, end, i0, i1;
};

// What a wave holds: 32 query rows, what they see, their sums.
template <typename T, int D> struct PfRowsOf {
  static constexpr int NK = D / 16, NE = D / 32;
  mf_u32x4 q[NK];
  int last, from;                    // row jr's last and first visible token
  int all_to, all_from;              // every row sees the tokens between
  bool ok;
  float m, lsum;
  mf_f32x16 o[NE];
};

// Row i of a piece: its sequence, query position and head; what it sees.
struct PfRow {
  int seq, s, g, last, from;
};
__device__ __forceinline__ PfRow pf_row(const PfParams& p, const PfPiece& w, int i,
                                        const int* ends) {
  const unsigned row = w.row0 + i, sg = p.S * p.G;
  PfRow r;
  r.seq = w.seq0 + row / sg;
  r.s = row % sg / (unsigned)p.G;
  r.g = row % (unsigned)p.G;
  const int at = ends[r.seq] - p.S + r.s;
  r.last = min(at, w.end - 1);
  r.from = p.window > 0 ? max(0, at - p.window + 1) : 0;
  return r;
}
// The loads of the wave's rows first .., as they are in memory; pf_fix_q makes operands of them.
template <typename T, int D>
__device__ __forceinline__ void pf_load_rows(const PfParams& p, const PfPiece& w, int first, int hk,
                                             const int* ends, PfRowsOf<T, D>& s) {
  const int lane = threadIdx.x & 63, jr = lane & 31, hh = lane >> 5;
  s.ok = first + jr < w.rows;
  const PfRow r = pf_row(p, w, s.ok ? first + jr : 0, ends);
  const char* qp = p.q + (((int64_t)r.seq * p.Hq + hk * p.G + r.g) * p.S + r.s) * (2 * D);
#pragma unroll
  for (int i = 0; i < PfRowsOf<T, D>::NK; ++i)
    s.q[i] = *reinterpret_cast<const mf_u32x4*>(qp + 16 * (2 * i + hh));
  s.last = s.ok ? r.last : -1;
  s.from = r.from;
  int to = s.ok ? s.last : 0x7fffffff, from = s.ok ? s.from : 0;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    to = min(to, __shfl_xor(to, d, 64));
    from = max(from, __shfl_xor(from, d, 64));
  }
  s.all_to = __builtin_amdgcn_readfirstlane(to);
  s.all_from = __builtin_amdgcn_readfirstlane(from);
}
template <typename T, int D>
__device__ __forceinline__ void pf_fix_q(const PfParams& p, PfRowsOf<T, D>& s) {
#pragma unroll
  for (int i = 0; i < PfRowsOf<T, D>::NK; ++i)
    s.q[i] = s.ok ? s.q[i] ^ p.q_sign : mf_u32x4{0u, 0u, 0u, 0u};
}

template <typename T, int D> __device__ __forceinline__ void pf_zero(PfRowsOf<T, D>& s) {
  s.m = -INFINITY;
  s.lsum = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) s.o[e][r] = 0.f;
}
template <typename T, int D> __device__ __forceinline__ bool pf_odd(const PfRowsOf<T, D>& s) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = odd || s.o[e][r] != s.o[e][r];
  return odd && s.ok;
}

// 32 tokens from tok0 on, whose K and V blocks (16 tokens each) are in LDS at kk and vv.  gone:
// bit u, block u is not there.  after_k(): K has been read; before_v(): V is wanted.
template <typename T, int D, bool kCap, int kParts, typename FK, typename FV>
__device__ __forceinline__ void pf_step(const PfParams& p, PfRowsOf<T, D>& s, int tok0, int gone,
                                        const char* kk, const char* vv, FK after_k, FV before_v) {
  constexpr int NK = D / 16, NE = D / 32, kRow = 2 * D, kBlk = kBlockTok * kRow;
  constexpr int kShift = std::is_same<T, f16_t>::value ? 9 : 0;
  constexpr float kSlack = chunk_slack(kShift);
  using Ops = MfmaOps<T>;
  using M32 = Mfma32<T>;
  const int lane = threadIdx.x & 63, jr = lane & 31, hh = lane >> 5;
  // the operands in LDS (prompt.h); their offsets are worked out anew each step, in few registers
  const int g_a = jr >> 3, h_a = (jr >> 2) & 1, t_a = jr & 3;
  const int tau = 16 * (g_a >> 1) + 8 * h_a + 4 * (g_a & 1) + t_a;
  const int ktok = tau & 15, nl = lane & 15;
  int k_off = (tau >> 4) * kBlk + ktok * kRow + 16 * (hh ^ swz<D>(ktok));
  const int v_tok0 = 8 * hh + (nl >> 2);
  int v_off = v_tok0 * kRow + 16 * ((2 * (jr >> 4) + ((nl & 3) >> 1)) ^ swz<D>(v_tok0)) +
              8 * (nl & 1);
  asm volatile("" : "+v"(k_off), "+v"(v_off));
  mf_f32x16 sc;
#pragma unroll
  for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    sc = M32::mma(*reinterpret_cast<const mf_u32x4*>(kk + (k_off ^ (32 * i))), s.q[i], sc);
    if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);      // (few operands ahead)
  }
  after_k();
  const float scale2 = p.scale * kLog2E;
  const float mul = kCap ? 1.f : scale2;                     // logits in base-2 units
  float x[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = sc[r];
  if constexpr (kCap) softcap_scores<16>(x, p.scale * (1.f / p.softcap), p.softcap * kLog2E);
  if (gone || tok0 + 31 > s.all_to || tok0 < s.all_from) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int t = tok0 + 16 * (r >> 3) + 8 * hh + (r & 7);
      if (t > s.last || t < s.from || (gone >> (r >> 3) & 1)) x[r] = -INFINITY;
    }
  }
  float top = x[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
  top *= mul;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > s.m + kSlack) != 0, 0)) {
    float mn = fmaxf(s.m, fmaxf(top, __shfl_xor(top, 32, 64)));
    if constexpr (kShift) mn = ceilf(mn);                    // (so that m - kShift is exact)
    const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s.m - mn);
    s.m = mn;
    s.lsum *= f;
#pragma unroll
    for (int e = 0; e < NE; ++e) s.o[e] *= f;
  }
  const float base = s.m == -INFINITY ? 0.f : s.m - kShift;
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w0 = __builtin_amdgcn_exp2f(fmaf(x[2 * i], mul, -base));
    const float w1 = __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], mul, -base));
    if constexpr (kParts == 2) {
      Ops::split2(w0, w1, hi[i], lo[i]);
      s.lsum += w0 + w1;
    } else {
      hi[i] = Ops::pk(w0, w1);
      s.lsum = dot2<T>(hi[i], Ops::ones8()[0], s.lsum);
    }
  }
  before_v();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const mf_u32x4 ph{hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]};
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const char* at = vv + u * kBlk;
      const uint2 a0 = ld_tr16(at + (v_off ^ (64 * e)));
      const uint2 a1 = ld_tr16(at + (v_off ^ (64 * e) ^ 16) + 4 * kRow);
      const mf_u32x4 vop{a0.x, a0.y, a1.x, a1.y};
      s.o[e] = M32::mma(vop, ph, s.o[e]);
      if constexpr (kParts == 2) {
        const mf_u32x4 pl{lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]};
        s.o[e] = M32::mma(vop, pl, s.o[e]);
      }
      if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// A block of 16 tokens of a piece: where its rows of a KV head are, from the pool's start, and
// how many of them are tokens of the piece.
struct PfBlock {
  int64_t at;
  int nt;
};
__device__ __forceinline__ PfBlock pf_block(const PfParams& p, const PfPiece& w, int hk, int slot,
                                            int in, int tok, int block_bytes) {
  const bool there = (uint32_t)slot < (uint32_t)p.n_slots;
  return {hk * p.head + (there ? slot : 0) * p.slot + (int64_t)(there ? in : 0) * block_bytes,
          there ? min(max(w.end - tok, 0), kBlockTok) : 0};
}
// 16 tokens of K or V from global memory straight into LDS at dst, nt of them there, the rest
// zeros; chunks swizzled as attn_chunk32.h says.
template <int D>
__device__ __forceinline__ void pf_dma(const char* block, int nt, mf_u32x4* dst) {
  constexpr int CPR = D / 8, kRow = 2 * D, kLoads = kBlockTok * kRow / 1024;
  const int lane = threadIdx.x & 63;
  const auto rs = make_rsrc(block, nt * kRow);
#pragma unroll
  for (int l = 0; l < kLoads; ++l) {
    const int t = (64 / CPR) * l + lane / CPR;
    buf_load16_lds(rs, dst + 64 * l, t * kRow + 16 * ((lane % CPR) ^ swz<D>(t)));
  }
}

// V's infinities and NaN in n chunks of LDS, taken for zeros.
template <typename T> __device__ __forceinline__ void pf_clean(mf_u32x4* v, int n) {
  for (int i = threadIdx.x & 63; i < n; i += 64) {
    mf_u32x4 x = v[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] &= ~nonfinite_halves<T>(x[j]);
    v[i] = x;
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
// ... and added to the partials of the piece's rows that see them: worker id of n (the lanes of
// a wave, or the workgroup's) has two dims of every (n / (D / 2))th row.
template <typename T, int D>
__device__ __forceinline__ void pf_add_special(const PfParams& p, const PfPiece& w, int hk,
                                            const int* ends, float* part, int id, int n) {
  constexpr int kRow = 2 * D, kBlk = kBlockTok * kRow, kPairs = D / 2;
  const int every = max(1, n / kPairs);
  for (int item = id; item < kPairs * every; item += n) {
    const int pair = item % kPairs, r0 = item / kPairs;
    for (int b = 2 * w.i0; b < 2 * w.i1; ++b) {
      const int block = (w.first >> 4) + b, page = block / p.bpp;
      if (page >= p.max_pages) break;
      const int slot = p.table[(int64_t)w.seq0 * p.table_stride + page];
      const PfBlock k = pf_block(p, w, hk, slot, block - page * p.bpp, 16 * block, kBlk);
      for (int t = 0; t < k.nt; ++t) {
        const uint32_t v =
            *reinterpret_cast<const uint32_t*>(p.v + k.at + t * kRow + 4 * pair);
        const uint32_t bad = nonfinite_halves<T>(v);
        if (!bad) continue;
        for (int r = r0; r < w.rows; r += every) {
          const PfRow row = pf_row(p, w, r, ends);
          if (16 * block + t > row.last || 16 * block + t < row.from) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint16_t x = v >> 16 * h;
            if (bad >> 16 * h & 1)
              part[(int64_t)r * D + 2 * pair + h] += std::is_same<T, bf16_t>::value
                                                         ? __uint_as_float((uint32_t)x << 16)
                                                         : (float)__builtin_bit_cast(_Float16, x);
          }
        }
      }
    }
  }
}

// A wave's walk through K and V buffers of its own: steps first, first + stride, ... of the piece.
// Returns whether it was a careful one.
template <typename T, int D, bool kCap>
__device__ __forceinline__ bool pf_walk_alone(const PfParams& p, const PfPiece& w, int first,
                                              int stride, int hk, const int* ends,
                                              PfRowsOf<T, D>& s, mf_u32x4 (*lk)[2 * D],
                                              mf_u32x4 (*lv)[2 * D]) {
  constexpr int kBlk = kBlockTok * 2 * D;
  constexpr int kOwnLoads = 2 * kBlk / 1024;           // of a step's K or V
  constexpr int kWin = 32;
  const int lane = threadIdx.x & 63;
  const int steps = first < w.i1 ? (w.i1 - first - 1) / stride + 1 : 0;
  // lane 2 k + u holds block u of the wave's step win0 + k: its slot (-1: none), its place there
  struct Window {
    int slot, in;
  };
  const int32_t* trow = p.table + (int64_t)w.seq0 * p.table_stride;
  auto window = [&](int k0) -> Window {
    const int k = k0 + (lane >> 1);
    const int block = (w.first >> 4) + 2 * (first + stride * k) + (lane & 1);
    const int page = (unsigned)block / (unsigned)p.bpp;
    return {k < steps && page < p.max_pages ? trow[page] : -1, block - page * p.bpp};
  };
  Window win = window(0), next{-1, 0};
  int win0 = 0;
  auto slot_of = [&](int k, int u) {
    return __builtin_amdgcn_readlane(win.slot, (2 * (k - win0) + u) & 63);
  };
  auto dma = [&](int k, const char* pool, mf_u32x4 (*dst)[2 * D]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int in = __builtin_amdgcn_readlane(win.in, (2 * (k - win0) + u) & 63);
      const int tok = w.first + kPfStep * (first + stride * k) + 16 * u;
      const PfBlock b = pf_block(p, w, hk, k < steps ? slot_of(k, u) : -1, in, tok, kBlk);
      pf_dma<D>(pool + b.at, b.nt, dst[u]);
    }
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
  pf_load_rows(p, w, 0, hk, ends, s);
  for (bool careful = false;; careful = true) {
    pf_zero(s);
    if (careful) {
      win = window(0);
      win0 = 0;
    }
    if (steps) {
      dma(0, p.k, lk);
      __builtin_amdgcn_sched_barrier(0);               // (K's loads are the older ones)
      dma(0, p.v, lv);
    }
    if (steps > kWin) next = window(kWin);
    if (!careful) pf_fix_q(p, s);
    for (int k = 0; k < steps; ++k) {
      int gone = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if ((uint32_t)slot_of(k, u) >= (uint32_t)p.n_slots) gone |= 1 << u;
      older_landed();                                  // K
      pf_step<T, D, kCap, 2>(
          p, s, w.first + kPfStep * (first + stride * k), gone,
          reinterpret_cast<const char*>(lk), reinterpret_cast<const char*>(lv),
          [&] {
            reads_done();
            if (k + 1 == win0 + kWin) {
              win = next;
              win0 += kWin;
              next = window(win0 + kWin);
            }
            dma(k + 1, p.k, lk);                       // (past the last: nothing, zeros)
          },
          [&] {
            older_landed();                            // V
            if (careful) pf_clean<T>(&lv[0][0], 4 * D);
          });
      reads_done();
      dma(k + 1, p.v, lv);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load is on its way any more)
    if (careful || !__builtin_amdgcn_ballot_w64(pf_odd(s))) return careful;
  }
}

// All waves' walk through the stages of a piece, 32 rows a wave.
template <typename T, int D, bool kCap>
__device__ __forceinline__ bool pf_walk_wide(const PfParams& p, const PfPiece& w, int hk,
                                             const int* ends, PfRowsOf<T, D>& s,
                                             typename PfBuf<T, D>::type& lds0,
                                             typename PfBuf<T, D>::type& lds1) {
  constexpr int NW = pf_waves(D), kSteps = NW / 2, kBlk = kBlockTok * 2 * D, kChunks = 2 * D;
  __shared__ int sh_gone[2][NW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool wave_rows = kPfRows * wave < w.rows;
  const int stages = (w.i1 - w.i0 + kSteps - 1) / kSteps;
  const int32_t* trow = p.table + (int64_t)w.seq0 * p.table_stride;
  // lane i holds the slot of this wave's block (of the stage's NW) of stage win0 + i
  struct Window {
    int slot, in;
  };
  auto window = [&](int s0) -> Window {
    const int block = (w.first >> 4) + 2 * w.i0 + NW * (s0 + lane) + wave;
    const int page = (unsigned)block / (unsigned)p.bpp;
    return {s0 + lane < stages && page < p.max_pages ? trow[page] : -1, block - page * p.bpp};
  };
  Window win = window(0), next{-1, 0};
  int win0 = 0;
  auto dma = [&](int st, typename PfBuf<T, D>::type& dst) {
    if (st == win0 + 64) {
      win = next;
      win0 += 64;
      next = window(win0 + 64);
    }
    const int slot = __builtin_amdgcn_readlane(win.slot, (st - win0) & 63);
    const int in = __builtin_amdgcn_readlane(win.in, (st - win0) & 63);
    const PfBlock b =
        pf_block(p, w, hk, slot, in, w.first + kPfStep * w.i0 + 16 * (NW * st + wave), kBlk);
    mf_u32x4* k = &dst[0][0][0] + wave * kChunks;
    pf_dma<D>(p.k + b.at, b.nt, k);
    pf_dma<D>(p.v + b.at, b.nt, k + NW * kChunks);
    if (lane == 0) sh_gone[st & 1][wave] = (uint32_t)slot >= (uint32_t)p.n_slots;
  };
  pf_load_rows(p, w, wave_rows ? kPfRows * wave : 0, hk, ends, s);
  for (bool careful = false;; careful = true) {
    pf_zero(s);
    if (careful) {
      win = window(0);
      win0 = 0;
    }
    dma(0, lds0);
    if (stages > 64) next = window(64);
    if (!careful) pf_fix_q(p, s);
    auto stage = [&](int st, typename PfBuf<T, D>::type& cur, typename PfBuf<T, D>::type& nxt) {
      // the stage is in LDS (this wave's loads done, then everyone's), and every wave is
      // done with the other buffer, which the next stage's loads fill
      __builtin_amdgcn_s_waitcnt(0x0F70);              // vmcnt(0)
      if (careful) pf_clean<T>(&cur[0][0][0] + (NW + wave) * kChunks, kChunks);
      __syncthreads();
      const uint64_t gone = __builtin_amdgcn_ballot_w64(lane < NW && sh_gone[st & 1][lane % NW]);
      if (st + 1 < stages) dma(st + 1, nxt);
      if (!wave_rows) return;
#pragma unroll 1
      for (int j = 0; j < kSteps && w.i0 + kSteps * st + j < w.i1; ++j) {
        const char* kk = reinterpret_cast<const char*>(&cur[0][0][0]) + 2 * j * kBlk;
        pf_step<T, D, kCap, 1>(p, s, w.first + kPfStep * (w.i0 + kSteps * st + j),
                               (int)(gone >> (2 * j)) & 3, kk, kk + NW * kBlk, [] {}, [] {});
      }
    };
    for (int st = 0; st < stages; st += 2) {
      stage(st, lds0, lds1);
      if (st + 1 < stages) stage(st + 1, lds1, lds0);
    }
    // (the barrier also ends every wave's reads of the buffers)
    if (!__syncthreads_or(wave_rows && pf_odd(s)) || careful) return careful;
  }
}

// A wave's sums to their slot: row jr's dims 32 e + 8 g + 4 hh .. + 3 are register 4 g .. of o[e].
template <typename T, int D>
__device__ __forceinline__ void pf_store(const PfRowsOf<T, D>& s, float* ml, float* part) {
  const int lane = threadIdx.x & 63, jr = lane & 31, hh = lane >> 5;
  const float l = s.lsum + __shfl_xor(s.lsum, 32, 64);
  if (!s.ok) return;
  if (hh == 0) *reinterpret_cast<float2*>(ml + 2 * jr) = make_float2(s.m, l);
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(part + jr * D + 32 * e + 8 * g + 4 * hh) =
          make_float4(s.o[e][4 * g], s.o[e][4 * g + 1], s.o[e][4 * g + 2], s.o[e][4 * g + 3]);
}

// The waves' sums over the same rows joined, through LDS where K (the first half of the dims)
// and V were (prompt_join's layout), and to their slot.
template <typename T, int D>
__device__ __forceinline__ void pf_store_joined(const PfRowsOf<T, D>& s, int nrows, float* ml,
                                                float* part, typename PfBuf<T, D>::type& ldsk,
                                                typename PfBuf<T, D>::type& ldsv) {
  constexpr int NW = pf_waves(D), CPR = D / 8;
  __shared__ float tops[NW][kPfRows], sums[NW][kPfRows];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, jr = lane & 31, hh = lane >> 5;
  const float lsum = s.lsum + __shfl_xor(s.lsum, 32, 64);
  if (hh == 0) tops[wave][jr] = s.m;
  __syncthreads();
  float top = tops[0][jr];
#pragma unroll
  for (int i = 1; i < NW; ++i) top = fmaxf(top, tops[i][jr]);
  const float f = s.m == top ? 1.f : __builtin_amdgcn_exp2f(s.m - top);
  if (hh == 0) sums[wave][jr] = lsum * f;
  auto at = [&](int i, int c, int h, int r) {
    return reinterpret_cast<mf_f32x4*>(c < CPR / 2 ? &ldsk[0][0][0] : &ldsv[0][0][0]) + 4 * D * i +
           64 * (c % (CPR / 2)) + 32 * h + (r ^ c % 16);
  };
#pragma unroll
  for (int c = 0; c < CPR; ++c) {
    mf_f32x4 x;
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = scale_finite(s.o[c / 4][4 * (c % 4) + t], f);
    *at(wave, c, hh, jr) = x;
    if (c % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  for (int i = tid; i < nrows * CPR; i += 64 * NW) {
    const int r = i / CPR, c = i % CPR;
    mf_f32x4 a{0.f, 0.f, 0.f, 0.f}, b{0.f, 0.f, 0.f, 0.f};
    float l = 0.f, mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < NW; ++j) {
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
  __syncthreads();                                     // (the next walk fills the buffers)
}

template <typename T, int D, bool kCap>
__global__ __launch_bounds__(64 * pf_waves(D), D == 256 ? 1 : 2)
void prefix_attn_kernel(PfParams p) {
  constexpr int NW = pf_waves(D), kThreads = 64 * NW;
  typedef typename PfBuf<T, D>::type Buf;
  __shared__ union Lds {
    __device__ Lds() {}
    Buf buf;
    PfAt at;
  } lds;
  __shared__ Buf ldsv;
  extern __shared__ PfGroup groups[];                  // [n_groups + 1], then int [R]:
  int* ends = reinterpret_cast<int*>(groups + p.n_groups + 1);   // the sequences' tokens
  __shared__ int sh_sum[3][NW], sh_group[4], sh_own[NW][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % p.Hkv, wg = blockIdx.x / p.Hkv;
  // (the last workgroups take the first own walks: those that the groups' line may leave idle)
  const int wg_own = (p.wgs - 1 - wg) * NW, own_wave = wg_own + wave;
  const int n_groups = p.n_groups, sg = p.S * p.G;

  // ---- the lines: the walks' lengths, and where this workgroup's and its waves' stretches start
  const int len0 = tid < p.R ? p.lens[tid] : 0;
  for (int g = tid; g <= n_groups; g += kThreads)
    groups[g] = {min(max(p.starts ? p.starts[g] : 0, 0), p.R),
                 g < n_groups ? pf_shared(p, p.shared[g]) : 0, 0x7fffffff, 0};
  if (tid < NW) sh_own[tid][0] = -1;
  if (tid == 0) sh_group[0] = -1;
  __syncthreads();
  auto group_of = [&](int r) {                         // -1: none
    int lo = 0, hi = n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (groups[mid].start <= r) lo = mid;
      else hi = mid;
    }
    return n_groups && groups[lo].start <= r && r < groups[lo + 1].start ? lo : -1;
  };
  for (int r = tid; r < p.R; r += kThreads) {
    const PfView v = pf_view(p, r == tid ? len0 : p.lens[r]);
    ends[r] = v.end;
    const int g = group_of(r);
    if (g >= 0) {
      atomicMin(&groups[g].lo, v.first);
      atomicMax(&groups[g].hi, min(v.end, groups[g].shared));
    }
  }
  __syncthreads();
  auto group_rows = [&](int g) { return max(0, groups[g + 1].start - groups[g].start) * sg; };
  auto group_tiles = [&](int rows) {
    return rows <= kPfRows ? (rows > 0) : (rows + kPfRows * NW - 1) / (kPfRows * NW);
  };
  auto group_steps = [&](int g) { return pf_steps(groups[g].lo, groups[g].hi); };
  // the first of sequence r's tokens that its own walk has, g its group or -1
  auto own_first = [&](int r, int g) {
    return max(g < 0 ? 0 : groups[g].shared, pf_view(p, ends[r]).first);
  };
  auto own_steps = [&](int r, int g) { return pf_steps(own_first(r, g), ends[r]); };
  // each thread sums a run of groups, of lengths and of slots, and a run of sequences
  const int gper = (n_groups + kThreads - 1) / kThreads, rper = (p.R + kThreads - 1) / kThreads;
  const int g0 = min(n_groups, tid * gper), g1 = min(n_groups, g0 + gper);
  const int r0 = min(p.R, tid * rper), r1 = min(p.R, r0 + rper);
  int sum[3] = {0, 0, 0}, before[3], total[3] = {0, 0, 0};
  for (int g = g0; g < g1; ++g) {
    const int rows = group_rows(g);
    sum[0] += group_tiles(rows) * group_steps(g);
    sum[1] += (rows + kPfRows - 1) / kPfRows;
  }
  for (int r = r0; r < r1; ++r) sum[2] += p.own_tiles * own_steps(r, group_of(r));
#pragma unroll
  for (int i = 0; i < 3; ++i) before[i] = sum[i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int t = __shfl_up(before[i], d, 64);
      if (lane >= d) before[i] += t;
    }
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < 3; ++i) sh_sum[i][wave] = before[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    before[i] -= sum[i];
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const int x = sh_sum[i][v];
      if (v < wave) before[i] += x;
      total[i] += x;
    }
  }
  const int group_total = __builtin_amdgcn_readfirstlane(total[0]);
  const int own_total = __builtin_amdgcn_readfirstlane(total[2]);
  // (whole stages, and a step for each wave at least)
  const int stretch =
      max(2, ((group_total + p.wgs - 1) / p.wgs + NW / 2 - 1) / (NW / 2)) * (NW / 2);
  const int own_stretch = max(kPfOwnLeast, (own_total + p.wgs * NW - 1) / (p.wgs * NW));
  const int a = wg * stretch, b = min(a + stretch, group_total);
  for (int g = g0, x = before[0], y = before[1]; g < g1; ++g) {
    const int rows = group_rows(g), n = group_tiles(rows) * group_steps(g);
    if (blockIdx.x == 0) {
      lds.at.at[g] = x;
      lds.at.slot[g] = y;
    }
    if (a >= x && a < x + n) {
      sh_group[0] = g;
      sh_group[1] = x;
      sh_group[2] = y;
    }
    x += n;
    y += (rows + kPfRows - 1) / kPfRows;
  }
  for (int r = r0, x = before[2]; r < r1; ++r) {
    const int n = own_steps(r, group_of(r)), end = x + p.own_tiles * n;
    if (blockIdx.x == 0) {
      PfSeq& q = p.seqs[r];
      q.own_at = x;
      q.own_each = n;
      q.own_stretch = own_stretch;
      q.group_stretch = stretch;
    }
    // the waves whose stretches start in it
    for (int i = max(0, (x + own_stretch - 1) / own_stretch - wg_own);
         i < NW && (wg_own + i) * own_stretch < end; ++i) {
      sh_own[i][0] = r;
      sh_own[i][1] = x;
    }
    x = end;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int r = tid; r < p.R; r += kThreads) {
      const int g = group_of(r);
      PfSeq& q = p.seqs[r];
      q.row0 = g < 0 ? 0 : (r - groups[g].start) * sg;
      q.tile_rows = g < 0 || group_rows(g) <= kPfRows ? kPfRows : kPfRows * NW;
      q.group_at = g < 0 ? 0 : lds.at.at[g];
      q.group_slot = g < 0 ? 0 : lds.at.slot[g];
      q.group_each = g < 0 ? 0 : group_steps(g);
    }
    __syncthreads();                                   // (the walks' buffers may be written)
  }

  // ---- the workgroup's stretch [a, b) of the groups' line, walk by walk, then each wave's of
  // the own walks, without a barrier
  int g = __builtin_amdgcn_readfirstlane(sh_group[0]);
  int gx = __builtin_amdgcn_readfirstlane(sh_group[1]);
  int gslot = __builtin_amdgcn_readfirstlane(sh_group[2]);
  int r = __builtin_amdgcn_readfirstlane(sh_own[wave][0]);
  int rx = __builtin_amdgcn_readfirstlane(sh_own[wave][1]);
  const int oa = own_wave * own_stretch, ob = min(oa + own_stretch, own_total);
  int rg = r < 0 ? -1 : __builtin_amdgcn_readfirstlane(group_of(r));
  int t = -1;                                          // the walk's number in its group, sequence
  bool own = g < 0;
  PfRowsOf<T, D> s;
  for (;;) {
    // the next piece: its rows, steps and slot
    PfPiece w;
    int tiles, steps, rows, tile, x, to;
    if (!own) {
      if (g >= n_groups || gx >= b) {
        own = true;
        t = -1;
        continue;
      }
      w.seq0 = __builtin_amdgcn_readfirstlane(groups[g].start);
      w.first = __builtin_amdgcn_readfirstlane(groups[g].lo);
      w.end = __builtin_amdgcn_readfirstlane(groups[g].hi);
      rows = __builtin_amdgcn_readfirstlane(group_rows(g));
      tile = rows <= kPfRows ? kPfRows : kPfRows * NW;
      tiles = group_tiles(rows);
      x = gx;
      to = b;
    } else {
      if (r < 0 || r >= p.R || rx >= ob) break;
      w.seq0 = r;
      w.first = __builtin_amdgcn_readfirstlane(own_first(r, rg));
      w.end = __builtin_amdgcn_readfirstlane(ends[r]);
      rows = sg;
      tile = kPfRows;
      tiles = p.own_tiles;
      x = rx;
      to = ob;
    }
    const int from0 = own ? oa : a;
    steps = pf_steps(w.first, w.end);
    t = t < 0 ? (steps ? max(0, (from0 - x) / steps) : tiles) : t + 1;
    if (t >= tiles || x + t * steps >= to) {           // the next group, sequence
      if (!own) {
        gx += tiles * steps;
        gslot += (rows + kPfRows - 1) / kPfRows;
        ++g;
      } else {
        rx += tiles * steps;
        ++r;
        if (r < p.R) rg = __builtin_amdgcn_readfirstlane(group_of(r));
      }
      t = -1;
      continue;
    }
    x += t * steps;
    w.i0 = max(from0 - x, 0);
    w.i1 = min(to - x, steps);
    w.row0 = tile * t;
    w.rows = min(rows - w.row0, tile);
    if (w.i0 >= w.i1) continue;
    const bool wide = tile > kPfRows;
    float *ml, *part;
    if (own) {
      const int64_t at = ((int64_t)hk * p.own_slots + r * p.own_tiles + t + own_wave) * p.own_rows;
      ml = p.own_ml + 2 * at;
      part = p.own_o + at * D;
    } else {
      const int slot = gslot + t * (tile / kPfRows) + NW * wg;
      // (starts that do not ascend may have more rows than there are)
      if (slot + (w.rows + kPfRows - 1) / kPfRows > p.group_slots) continue;
      const int64_t at = ((int64_t)hk * p.group_slots + slot) * kPfRows;
      ml = p.group_ml + 2 * at;
      part = p.group_o + at * D;
    }
    bool careful;
    if (wide) {
      careful = pf_walk_wide<T, D, kCap>(p, w, hk, ends, s, lds.buf, ldsv);
      if (kPfRows * wave < w.rows)
        pf_store(s, ml + 2 * kPfRows * wave, part + (int64_t)kPfRows * wave * D);
      if (careful) __syncthreads();                    // (all rows are stored)
    } else {
      careful = pf_walk_alone<T, D, kCap>(p, w, own ? w.i0 : w.i0 + wave, own ? 1 : NW, hk, ends,
                                          s, lds.buf[wave], ldsv[wave]);
      if (own) {
        pf_store(s, ml, part);
      } else {
        pf_store_joined(s, w.rows, ml, part, lds.buf, ldsv);
        careful = __syncthreads_or(careful);
      }
    }
    if (careful)
      pf_add_special<T, D>(p, w, hk, ends, part, own ? lane : tid, own ? 64 : kThreads);
  }
}

// Row blockIdx.x of the output, (r, hq, s), from its walks' partials.
template <typename T, int D>
__global__ __launch_bounds__(kPfJoinThreads) void prefix_join_kernel(PfParams p) {
  constexpr int NW = pf_waves(D), C = D / 4, N = kPfJoinThreads / C, U = 4;
  __shared__ float4 sh_o[N][C];
  __shared__ float2 sh_ml[N];
  using Ops = MfmaOps<T>;
  const int s = blockIdx.x % p.S, hq = blockIdx.x / p.S % p.Hq, r = blockIdx.x / p.S / p.Hq;
  const int hk = hq / p.G, row = s * p.G + hq % p.G;
  const PfSeq q = p.seqs[r];
  // the pieces of a walk at [at, at + each) of a line: on stretches at / stretch and on
  auto pieces = [](int from, int each, int stretch, int& first) {
    first = each > 0 ? from / stretch : 0;
    return each > 0 ? (from + each - 1) / stretch - first + 1 : 0;
  };
  const int grow = q.row0 + row, gt = grow / q.tile_rows, ot = row / kPfRows;
  int w0, v0;
  int n_group = pieces(q.group_at + gt * q.group_each, q.group_each, q.group_stretch, w0);
  const int n_own = pieces(q.own_at + ot * q.own_each, q.own_each, q.own_stretch, v0);
  const int g0 = q.group_slot + grow / kPfRows + NW * w0, o0 = r * p.own_tiles + ot + v0;
  n_group = min(n_group, max(0, (p.group_slots - g0 + NW - 1) / NW));
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
        const int64_t at = ((int64_t)hk * p.group_slots + g0 + NW * i) * kPfRows + grow % kPfRows;
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
  const size_t dyn = sizeof(PfGroup) * (p.n_groups + 1) + sizeof(int) * (size_t)p.R;
  if (p.softcap > 0.f)
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, true>), grid, dim3(64 * pf_waves(D)), dyn, st, p);
  else
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, false>), grid, dim3(64 * pf_waves(D)), dyn, st, p);
  hipLaunchKernelGGL((prefix_join_kernel<T, D>), dim3((uint32_t)(p.R * p.Hq * p.S)),
                     dim3(kPfJoinThreads), 0, st, p);
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
