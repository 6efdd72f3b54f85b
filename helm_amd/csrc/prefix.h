// Decode attention of sequences that share their first pages (helm_prefix_decode_attn): row
// (r, h, s) of a sequence of len tokens stands at position p = len - S + s and gets
// softmax(cap(q . K^T scale)) . V over its tokens j <= p (and j > p - window).
//
// A group's shared pages are walked once for the rows of all its sequences, a sequence's
// own pages for its own S G rows a KV head; every walk leaves partial sums (m, l, o) of its
// rows over its tokens, and a second kernel joins a row's:
//   out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i,  M = max m_i.
// Bound by memory up to some 280 rows a KV head (6 D operations a row and token, the weights being
// in two parts, against 4 D bytes a token), by the matrix cores beyond.
//
// Work: a KV head's walks, the groups' (128 rows each) and then the sequences',
// lie end to end on one line of steps of 32 tokens, and each of the head's workgroups takes an
// equal stretch of it.  So any lengths are spread evenly, and the launch depends on none:
// every workgroup sums them up for itself.  A piece of a walk leaves its partials at slot
// (walk + workgroup), of which no two pieces are alike, as both only grow along the line.
// Walks of a group that has several come first on the line, each from a stretch's start on:
// so the workgroups that read the same tokens for different rows do so side by side, through
// one XCD's L2 (a KV head's workgroups are on one where 8, 16, ... heads lie round the XCDs):
// 32k tokens under 64 sequences 93 -> 88 us at that step; 6% more is read than K and V hold.
//
// A walk is that of prompt.h: 32 x 32 matrix tiles, 32 rows a wave, K and V straight from memory
// into LDS, one barrier a stage.  Few rows keep few of the waves busy; such a walk is bound by
// memory.  K and V come from HBM here, not from L2: three stages are on their way.
//
// Bound, measured at D = 128, bf16 (walks and their joining, us a call): 4 beams of 16 prompts of
// up to 4k tokens 49, 2.8 TB/s of K and V; 24 chats behind 8k shared tokens 36, of which the
// joining takes 5 and the line 3.5; 32k tokens under 64 sequences 92, of whose walks' cycles the
// matrix cores are busy 30% and LDS 12%.  From 32k to 64k tokens 64 sequences take 51 us more,
// which is 1.0 PFLOP/s with both parts' products, 32 sequences 26, which is 5.2 TB/s; some 30 us
// of a call do not grow with the tokens.
//
// Weights enter P . V in two 16-bit parts (2^-16 of the weight in bf16, 2^-22 in f16) and the row's
// sum in fp32, as in the decode kernels; f16 weights are taken times 2^9, what is under 2^-34 of
// the largest is lost.  An output is then off by its own rounding and hardly more: relative rms
// error 1.7e-3 in bf16, 2.1e-4 in f16.  (In one part: 2.3e-3 and up to 3.0e-4, for 24 chats 34 us
// against 36, 4 beams of 16 prompts 48.7 against 49.4, 32k tokens under 64 sequences 82 against 91.)
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
// What a walk costs before its first step and behind its last, in steps.  (4 beams of 16 prompts and
// 32k tokens under 64 sequences, us: with 5 49.2 and 91.6, with 4 52.0 and 90.5, with 6 49.3 and
// 92.7, with 8 51.3 and 95.1, with 12 54.1 and 99.9; with 2, where workgroups of several short walks
// end late, 61.8 and 100.)
constexpr int kPfFixed = 5;
// A workgroup's least stretch (a prompt of 2k tokens, 4 beams: 17.3 us, with 2 18.0, with 8 21.5).
constexpr int kPfLeast = 4;
constexpr int kPfJoinThreads = 256;
constexpr int kPfWaves = 4;          // of a workgroup
constexpr int kPfThreads = 64 * kPfWaves;
constexpr int kPfTile = kPfRows * kPfWaves;            // rows of a walk
// Stage buffers.  (With weights in one part; two, and three workgroups a CU: 24 chats 39.6 us, 4
// beams of 16 prompts 55, 32k tokens 88; three buffers, three workgroups 39.7, 58, 88; four and
// two 33.9, 48, 84.)
constexpr int kPfBufs = 4;
// Tokens of a stage; workgroups of a CU, which the buffers (16 KB, 32 at D = 256) leave room for.
template <int D> struct PfShape {
  static constexpr int kTok = D == 64 ? 64 : 32, kPerCu = D == 256 ? 1 : 2;
};

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

// Where the partials of sequence r's rows are: walk t is from at + t each on of the line, its
// steps (0: there is none) from kPfFixed behind that on.
struct PfSeq {
  int row0;                          // its first row among its group's
  int group_at, group_each, group_steps, group_slot;
  int own_at, own_steps;
  int stretch;                       // of a workgroup
};

// What a sequence of len >= 0 tokens sees: [first, end) of its table, first a block's.
struct PfView {
  int first, end;
};
__device__ __forceinline__ int pf_room(const PfParams& p) { return p.max_pages * p.page; }
__device__ __forceinline__ PfView pf_view(const PfParams& p, int len) {
  // (row 0's first: len - S + 1 - window, or 0)
  const int first = p.window > 0 && len - p.window >= p.S ? len - p.window - p.S + 1 : 0;
  return {first & ~15, min(len, pf_room(p))};
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

// A stage of K and V in LDS, blocks of 16 tokens.  The stage buffers are objects of their own, so
// that the compiler sees that loads into one do not touch the reads of another.
template <int D> struct PfBuf {
  static constexpr int kBlocks = PfShape<D>::kTok / kBlockTok, kChunks = 2 * D;
  typedef mf_u32x4 type[2][kBlocks][kChunks];
};
template <int D> using PfLds = typename PfBuf<D>::type;

// A walk's piece: rows [row0, row0 + rows) of sequences seq0 .. (S G rows each), steps [i0, i1)
// of tokens [first, end).
struct PfPiece {
  int seq0, row0, rows, first, end, i0, i1;
};

// What a wave holds: 32 query rows, what they see, their sums.
template <int D> struct PfRowsOf {
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
                                        const int* lens) {
  const unsigned row = w.row0 + i, sg = p.S * p.G;
  PfRow r;
  r.seq = w.seq0 + row / sg;
  r.s = row % sg / (unsigned)p.G;
  r.g = row % (unsigned)p.G;
  const int at = lens[r.seq] - p.S + r.s;
  r.last = min(at, w.end - 1);
  r.from = p.window > 0 && at >= p.window ? at - p.window + 1 : 0;
  return r;
}
// The wave's rows first ..: what they see, and the address of row jr's query.
template <int D>
__device__ __forceinline__ const char* pf_rows(const PfParams& p, const PfPiece& w, int first,
                                               int hk, const int* lens, PfRowsOf<D>& s) {
  const int jr = threadIdx.x & 31;
  s.ok = first + jr < w.rows;
  const PfRow r = pf_row(p, w, s.ok ? first + jr : 0, lens);
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
  return p.q + (((int64_t)r.seq * p.Hq + hk * p.G + r.g) * p.S + r.s) * (2 * D);
}

template <int D> __device__ __forceinline__ void pf_zero(PfRowsOf<D>& s) {
  s.m = -INFINITY;
  s.lsum = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) s.o[e][r] = 0.f;
}
template <int D> __device__ __forceinline__ bool pf_odd(const PfRowsOf<D>& s) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = odd || s.o[e][r] != s.o[e][r];
  return odd && s.ok;
}

// 32 tokens from tok0 on, whose K and V blocks (16 tokens each) are in LDS at kk and vv.  gone:
// bit u, block u is not there.
template <typename T, int D, bool kCap>
__device__ __forceinline__ void pf_step(const PfParams& p, PfRowsOf<D>& s, int tok0, int gone,
                                        const char* kk, const char* vv) {
  constexpr int NK = D / 16, NE = D / 32, kRow = 2 * D, kBlk = kBlockTok * kRow;
  constexpr int kShift = std::is_same<T, f16_t>::value ? 9 : 0;
  constexpr float kSlack = chunk_slack(kShift);
  using Ops = MfmaOps<T>;
  using M32 = Mfma32<T>;
  const int lane = threadIdx.x & 63, jr = lane & 31, hh = lane >> 5;
  // the operands in LDS (prompt.h)
  const int g_a = jr >> 3, h_a = (jr >> 2) & 1, t_a = jr & 3;
  const int tau = 16 * (g_a >> 1) + 8 * h_a + 4 * (g_a & 1) + t_a;
  const int ktok = tau & 15, nl = lane & 15;
  const int k_off = (tau >> 4) * kBlk + ktok * kRow + 16 * (hh ^ swz<D>(ktok));
  const int v_tok0 = 8 * hh + (nl >> 2);
  const int v_off = v_tok0 * kRow + 16 * ((2 * (jr >> 4) + ((nl & 3) >> 1)) ^ swz<D>(v_tok0)) +
                    8 * (nl & 1);
  mf_f32x16 sc;
#pragma unroll
  for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
  for (int i = 0; i < NK; ++i)
    sc = M32::mma(*reinterpret_cast<const mf_u32x4*>(kk + (k_off ^ (32 * i))), s.q[i], sc);
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
  float ws[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w0 = __builtin_amdgcn_exp2f(fmaf(x[2 * i], mul, -base));
    const float w1 = __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], mul, -base));
    ws[i] = w0 + w1;
    if constexpr (std::is_same<T, f16_t>::value) Ops::split2_mix(w0, w1, hi[i], lo[i]);
    else Ops::split2(w0, w1, hi[i], lo[i]);
  }
  s.lsum += ((ws[0] + ws[1]) + (ws[2] + ws[3])) + ((ws[4] + ws[5]) + (ws[6] + ws[7]));
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const mf_u32x4 pop{hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]};
    const mf_u32x4 rest{lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]};
    mf_u32x4 vop[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const char* at = vv + u * kBlk;
      const uint2 a0 = ld_tr16(at + (v_off ^ (64 * e)));
      const uint2 a1 = ld_tr16(at + (v_off ^ (64 * e) ^ 16) + 4 * kRow);
      vop[e] = mf_u32x4{a0.x, a0.y, a1.x, a1.y};
      s.o[e] = M32::mma(vop[e], pop, s.o[e]);
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) s.o[e] = M32::mma(vop[e], rest, s.o[e]);
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
// V's infinities and NaN, added to the partials of the piece's rows that see them: worker id of n
// has two dims of every (n / (D / 2))th row.
template <typename T, int D>
__device__ __forceinline__ void pf_add_special(const PfParams& p, const PfPiece& w, int hk,
                                            const int* lens, float* part, int id, int n) {
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
          const PfRow row = pf_row(p, w, r, lens);
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

// The workgroup's walk through the stages of a piece, 32 rows a wave.  Returns whether it was
// done again, with V's infinities and NaN taken for zeros.
template <typename T, int D, bool kCap>
__device__ __forceinline__ bool pf_walk(const PfParams& p, const PfPiece& w, int hk,
                                        const int* lens, PfRowsOf<D>& s, PfLds<D>& lds0,
                                        PfLds<D>& lds1, PfLds<D>& lds2, PfLds<D>& lds3) {
  using Buf = PfLds<D>;
  constexpr int NW = kPfWaves, NB = kPfBufs;
  constexpr int SB = PfBuf<D>::kBlocks, kSteps = SB / 2;
  constexpr int CPR = D / 8, kRow = 2 * D, kBlk = kBlockTok * kRow, kBlkLoads = kBlk / 1024;
  constexpr int kLoads = 2 * SB * kBlkLoads / NW;      // a wave's, of one block
  constexpr int kAhead = (NB - 2) * kLoads;            // those of the stages behind the present one
  constexpr int NK = D / 16;
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool wave_rows = kPfRows * wave < w.rows;
  const int stages = (w.i1 - w.i0 + kSteps - 1) / kSteps;
  const int tok0 = w.first + kPfStep * w.i0;
  const int32_t* trow = p.table + (int64_t)w.seq0 * p.table_stride;
  // load i of the stage's is part i % kBlkLoads of a block's K, its V, the next block's, ...
  const int my_blk = wave * kLoads / kBlkLoads / 2;
  // lane SB k + u holds the slot of block u of stage win0 + k (-1: none), its place there
  constexpr int kWin = 64 / SB;
  struct Window {
    int slot, in;
  };
  auto window = [&](int s0) -> Window {
    const int st = s0 + lane / SB;
    const int block = (tok0 >> 4) + SB * st + lane % SB;
    const int page = (unsigned)block / (unsigned)p.bpp;
    return {st < stages && page < p.max_pages ? trow[page] : -1, block - page * p.bpp};
  };
  Window win = window(0), next{-1, 0};
  int win0 = 0;
  uint32_t gone = 0;                                   // a byte a stage: its blocks not there
  // (past the last stage: nothing, zeros, so that every stage waits for the same)
  auto dma = [&](int st, Buf& dst) {
    if (st == win0 + kWin) {
      win = next;
      win0 += kWin;
      next = window(win0 + kWin);
    }
    uint32_t g = 0;
#pragma unroll
    for (int u = 0; u < SB; ++u)
      if ((uint32_t)__builtin_amdgcn_readlane(win.slot, SB * (st - win0) + u) >=
          (uint32_t)p.n_slots)
        g |= 1u << u;
    gone = gone >> 8 | g << 24;
    const int slot = __builtin_amdgcn_readlane(win.slot, SB * (st - win0) + my_blk);
    const int in = __builtin_amdgcn_readlane(win.in, SB * (st - win0) + my_blk);
    const PfBlock b = pf_block(p, w, hk, slot, in, tok0 + 16 * (SB * st + my_blk), kBlk);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = wave * kLoads + k, is_v = i / kBlkLoads % 2, u = i % kBlkLoads;
      const int t = (64 / CPR) * u + lane / CPR;
      // (tokens past the piece's and pages that are not there: zeros)
      buf_load16_lds(make_rsrc((is_v ? p.v : p.k) + b.at, b.nt * kRow), &dst[is_v][my_blk][64 * u],
                     t * kRow + 16 * ((lane % CPR) ^ swz<D>(t)));
    }
  };
  // careful: infinities and NaN in what this wave has loaded of V, taken for zeros
  auto clean = [&](Buf& buf) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = wave * kLoads + k, is_v = i / kBlkLoads % 2, u = i % kBlkLoads;
      if (!is_v) continue;
      mf_u32x4& v = buf[1][my_blk][64 * u + lane];
      mf_u32x4 x = v;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] &= ~nonfinite_halves<T>(x[j]);
      v = x;
    }
  };
  const char* qp = pf_rows<D>(p, w, wave_rows ? kPfRows * wave : 0, hk, lens, s);
#pragma unroll
  for (int i = 0; i < NK; ++i) s.q[i] = *reinterpret_cast<const mf_u32x4*>(qp + 16 * (2 * i + hh));
  auto start = [&] {
    dma(0, lds0);
    __builtin_amdgcn_sched_barrier(0);                 // (in this order)
    dma(1, lds1);
    __builtin_amdgcn_sched_barrier(0);
    dma(2, lds2);
    if (stages > kWin) next = window(kWin);
  };
  start();
#pragma unroll
  for (int i = 0; i < NK; ++i) s.q[i] = s.ok ? s.q[i] ^ p.q_sign : mf_u32x4{0u, 0u, 0u, 0u};
  for (bool careful = false;; careful = true) {
    pf_zero(s);
    auto stage = [&](int st, Buf& cur, Buf& nxt) {
      // the stage is in LDS (this wave's loads done, all but those of the NB - 2 stages behind
      // it, then everyone's), and every wave is done with the buffer of the stage before,
      // which loads of a later one fill (a plain barrier would wait for all loads)
      if (careful) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAhead) : "memory");
        clean(cur);
      }
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAhead) : "memory");
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t there = gone >> (32 - 8 * (NB - 1));          // this stage's
      dma(st + NB - 1, nxt);
      if (!wave_rows) return;
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        if (j == 0 || w.i0 + kSteps * st + j < w.i1)
          pf_step<T, D, kCap>(p, s, tok0 + kPfStep * (kSteps * st + j), there >> (2 * j) & 3,
                              reinterpret_cast<const char*>(&cur[0][2 * j][0]),
                              reinterpret_cast<const char*>(&cur[1][2 * j][0]));
    };
    // (left from within: a round's end always has the same loads on their way)
    for (int st = 0;; st += NB) {
      stage(st, lds0, lds3);
      if (st + 1 >= stages) break;
      stage(st + 1, lds1, lds0);
      if (st + 2 >= stages) break;
      stage(st + 2, lds2, lds1);
      if (st + 3 >= stages) break;
      stage(st + 3, lds3, lds2);
      if (st + NB >= stages) break;
    }
    // (no load is on its way any more, and the barrier ends every wave's reads of the buffers)
    __builtin_amdgcn_s_waitcnt(0x0F70);
    if (!__syncthreads_or(wave_rows && pf_odd(s)) || careful) return careful;
    win = window(0);
    win0 = 0;
    start();
  }
}

// A wave's sums to their slot: row jr's dims 32 e + 8 g + 4 hh .. + 3 are register 4 g .. of o[e].
// (Through LDS, in whole lines, with weights in one part: 32k tokens under 64 sequences 81 -> 83 us,
// 4 beams of 16 prompts 48 -> 52.)
template <int D>
__device__ __forceinline__ void pf_store(const PfRowsOf<D>& s, float* ml, float* part) {
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

// Running sums of N numbers over the workgroup's threads before this one, and in all.
template <int NW, int N>
__device__ __forceinline__ void pf_scan(const int (&x)[N], int (&before)[N], int (&all)[N],
                                        int (*sh)[NW]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) before[i] = x[i];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = __shfl_up(before[i], d, 64);
      if (lane >= d) before[i] += t;
    }
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) sh[i][wave] = before[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    before[i] -= x[i];
    all[i] = 0;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      if (v < wave) before[i] += sh[i][v];
      all[i] += sh[i][v];
    }
  }
}

template <typename T, int D, bool kCap>
__global__ __launch_bounds__(kPfThreads, PfShape<D>::kPerCu)
void prefix_attn_kernel(PfParams p) {
  constexpr int NW = kPfWaves, kThreads = kPfThreads, kTile = kPfTile;
  __shared__ union Lds {
    __device__ Lds() {}
    PfLds<D> buf;
    PfAt at;
  } lds0;
  __shared__ PfLds<D> lds1, lds2, lds3;
  extern __shared__ PfGroup groups[];                  // [n_groups + 1], then int [R]:
  int* lens = reinterpret_cast<int*>(groups + p.n_groups + 1);   // the sequences' tokens
  __shared__ int sh_sum[5][NW], sh_found[4], sh_down;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % p.Hkv, wg = blockIdx.x / p.Hkv;
  const int sg = p.S * p.G;
  int n_groups = p.n_groups;

  // ---- the line: the walks' lengths, and where this workgroup's stretch starts
  const int len0 = tid < p.R ? p.lens[tid] : 0;
  for (int g = tid; g <= n_groups; g += kThreads)
    groups[g] = {n_groups ? min(max(p.starts[g], 0), p.R) : 0,
                 g < n_groups ? pf_shared(p, p.shared[g]) : 0, 0x7fffffff, 0};
  if (tid == 0) sh_down = 0;
  __syncthreads();
  for (int g = tid; g < n_groups; g += kThreads)
    if (groups[g].start > groups[g + 1].start) sh_down = 1;
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
    const int len = max(r == tid ? len0 : p.lens[r], 0);
    const PfView v = pf_view(p, len);
    lens[r] = len;
    const int g = group_of(r);
    const int end = g < 0 ? 0 : min(v.end, groups[g].shared);
    if (v.first < end) {                               // (it sees some of the shared tokens)
      atomicMin(&groups[g].lo, v.first);
      atomicMax(&groups[g].hi, end);
    }
  }
  __syncthreads();
  // (starts that do not ascend: no groups, as the line's length would have no bound)
  if (sh_down) n_groups = 0;
  const int E = n_groups + p.R;
  if (tid == 0) sh_found[0] = E;
  // entity e, a group or a sequence: its rows and tokens
  struct Entity {
    int seq0, rows, first, end;
  };
  auto entity = [&](int e) -> Entity {
    if (e < n_groups) {
      const PfGroup g = groups[e];
      return {g.start, max(0, groups[e + 1].start - g.start) * sg, g.lo, g.hi};
    }
    const int r = e - n_groups, g = group_of(r);
    const PfView v = pf_view(p, lens[r]);
    return {r, sg, max(g < 0 ? 0 : groups[g].shared, v.first), v.end};
  };
  auto tiles_of = [&](int rows) { return (rows + kTile - 1) / kTile; };
  auto slots_of = [&](int e, int rows) {
    return e < n_groups ? (rows + kPfRows - 1) / kPfRows : 0;
  };
  auto several = [&](int e, int rows) { return e < n_groups && rows > kTile; };
  // each thread sums a run of entities: lengths, walks and slots of the groups of several
  // walks, lengths and slots of the others
  const int per = (E + kThreads - 1) / kThreads;
  const int e0 = min(E, tid * per), e1 = min(E, e0 + per);
  constexpr int N = 5;
  int sum[N] = {}, at[N], total[N];
  const Entity mine = e0 < e1 ? entity(e0) : Entity{0, 0, 0, 0};       // (mostly its only one)
  auto entity_of_run = [&](int e) { return e == e0 ? mine : entity(e); };
  for (int e = e0; e < e1; ++e) {
    const Entity n = entity_of_run(e);
    const int steps = pf_steps(n.first, n.end), tiles = tiles_of(n.rows);
    const int len = steps ? tiles * (steps + kPfFixed) : 0;
    if (several(e, n.rows)) {
      sum[0] += len;
      sum[1] += tiles;
      sum[2] += slots_of(e, n.rows);
    } else {
      sum[3] += len;
      sum[4] += slots_of(e, n.rows);
    }
  }
  pf_scan<NW, N>(sum, at, total, sh_sum);
  // whether a stretch's start is worth it: half a stretch a walk is left unused
  const bool align = total[1] > 0 && 2 * total[1] <= p.wgs;
  const int room = p.wgs - (align ? total[1] : 0);
  const int stretch = max(kPfLeast, (total[0] + total[3] + room - 1) / room);
  auto each_of = [&](bool multi, int steps) {
    const int n = steps ? steps + kPfFixed : 0;
    return multi && align ? (n + stretch - 1) / stretch * stretch : n;
  };
  if (align) {
    int len[1] = {0}, to[1], all[1];
    for (int e = e0; e < e1; ++e) {
      const Entity n = entity_of_run(e);
      if (several(e, n.rows)) len[0] += tiles_of(n.rows) * each_of(true, pf_steps(n.first, n.end));
    }
    __syncthreads();                                   // (sh_sum has been read)
    pf_scan<NW, 1>(len, to, all, sh_sum);
    at[0] = to[0];
    total[0] = all[0];
  }
  const int end_all = __builtin_amdgcn_readfirstlane(total[0] + total[3]);
  const int a = wg * stretch, b = min(a + stretch, end_all);
  at[3] += total[0];
  at[4] += total[2];
  for (int e = e0; e < e1; ++e) {
    const Entity n = entity_of_run(e);
    const bool multi = several(e, n.rows);
    const int steps = pf_steps(n.first, n.end), tiles = tiles_of(n.rows);
    const int each = each_of(multi, steps);
    int &x = at[multi ? 0 : 3], &y = at[multi ? 2 : 4];
    if (a >= x && a < x + tiles * each) {
      sh_found[0] = e;
      sh_found[1] = x;
      sh_found[2] = y;
    }
    if (blockIdx.x == 0) {
      if (e < n_groups) {
        lds0.at.at[e] = x;
        lds0.at.slot[e] = y;
      } else {
        PfSeq& q = p.seqs[e - n_groups];
        q.own_at = x;
        q.own_steps = steps;
        q.stretch = stretch;
      }
    }
    x += tiles * each;
    y += slots_of(e, n.rows);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int r = tid; r < p.R; r += kThreads) {
      const int g = group_of(r);
      const Entity n = g < 0 ? Entity{0, 0, 0, 0} : entity(g);
      const int steps = pf_steps(n.first, n.end);
      PfSeq& q = p.seqs[r];
      q.row0 = g < 0 ? 0 : (r - n.seq0) * sg;
      q.group_at = g < 0 ? 0 : lds0.at.at[g];
      q.group_slot = g < 0 ? 0 : lds0.at.slot[g];
      q.group_each = each_of(several(g < 0 ? E : g, n.rows), steps);
      q.group_steps = steps;
    }
    __syncthreads();                                   // (the walks' buffers may be written)
  }

  // ---- the workgroup's stretch [a, b) of the line, walk by walk
  int e = __builtin_amdgcn_readfirstlane(sh_found[0]);
  int x = __builtin_amdgcn_readfirstlane(sh_found[1]);
  int y = __builtin_amdgcn_readfirstlane(sh_found[2]);
  auto rows_at = [&](int i) {
    return i < n_groups ? max(0, groups[i + 1].start - groups[i].start) * sg : sg;
  };
  bool multi = e < E && several(e, rows_at(e));
  PfRowsOf<D> s;
  for (int t = -1; e < E && x < b;) {
    const Entity n = entity(e);
    PfPiece w;
    w.seq0 = __builtin_amdgcn_readfirstlane(n.seq0);
    w.first = __builtin_amdgcn_readfirstlane(n.first);
    w.end = __builtin_amdgcn_readfirstlane(n.end);
    const int rows = __builtin_amdgcn_readfirstlane(n.rows);
    const int tiles = tiles_of(rows), steps = pf_steps(w.first, w.end);
    const int each = each_of(multi, steps);
    t = t < 0 ? (each ? max(0, (a - x) / each) : tiles) : t + 1;
    if (t >= tiles || x + t * each >= b) {             // the next group of its kind, sequence
      x += tiles * each;
      y += slots_of(e, rows);
      for (++e; e < n_groups && several(e, rows_at(e)) != multi;) ++e;
      if (multi && e >= n_groups) {                    // (no more of several walks)
        multi = false;
        for (e = 0; e < n_groups && several(e, rows_at(e));) ++e;
      }
      t = -1;
      continue;
    }
    const int from = x + t * each + kPfFixed;
    w.i0 = max(a - from, 0);
    w.i1 = min(b - from, steps);
    if (w.i0 >= w.i1) continue;
    w.row0 = kTile * t;
    w.rows = min(rows - w.row0, kTile);
    float *ml, *part;
    if (e < n_groups) {
      const int to = y + t * NW + NW * wg;
      const int64_t at = ((int64_t)hk * p.group_slots + to) * kPfRows;
      ml = p.group_ml + 2 * at;
      part = p.group_o + at * D;
    } else {
      const int64_t at = ((int64_t)hk * p.own_slots + w.seq0 * p.own_tiles + t + wg) * p.own_rows;
      ml = p.own_ml + 2 * at;
      part = p.own_o + at * D;
    }
    const bool careful = pf_walk<T, D, kCap>(p, w, hk, lens, s, lds0.buf, lds1, lds2, lds3);
    if (kPfRows * wave < w.rows)
      pf_store(s, ml + 2 * kPfRows * wave, part + (int64_t)kPfRows * wave * D);
    if (careful) {
      __syncthreads();                                 // (all rows are stored)
      pf_add_special<T, D>(p, w, hk, lens, part, tid, kThreads);
    }
  }
}

// Row blockIdx.x of the output, (r, hq, s), from its walks' partials.
template <typename T, int D>
__global__ __launch_bounds__(kPfJoinThreads) void prefix_join_kernel(PfParams p) {
  constexpr int NW = kPfWaves, kTile = kPfTile;
  constexpr int C = D / 4, N = kPfJoinThreads / C, U = 4;
  __shared__ float4 sh_o[N][C];
  __shared__ float2 sh_ml[N];
  using Ops = MfmaOps<T>;
  const int s = blockIdx.x % p.S, hq = blockIdx.x / p.S % p.Hq, r = blockIdx.x / p.S / p.Hq;
  const int hk = hq / p.G, row = s * p.G + hq % p.G;
  const PfSeq q = p.seqs[r];
  // the pieces of a walk whose steps start kPfFixed behind `at` on the line
  auto pieces = [&](int at, int steps, int& first) {
    first = (at + kPfFixed) / q.stretch;
    return steps > 0 ? (at + kPfFixed + steps - 1) / q.stretch - first + 1 : 0;
  };
  const int grow = q.row0 + row, gt = grow / kTile, ot = row / kTile;
  int w0, v0;
  const int n_group = pieces(q.group_at + gt * q.group_each, q.group_steps, w0);
  const int own_each = q.own_steps > 0 ? q.own_steps + kPfFixed : 0;
  const int n_own = pieces(q.own_at + ot * own_each, q.own_steps, v0);
  const int g0 = q.group_slot + grow / kPfRows + NW * w0, o0 = r * p.own_tiles + ot + v0;
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
        const int64_t at =
            ((int64_t)hk * p.own_slots + o0 + i - n_group) * p.own_rows + row % kTile;
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
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, true>), grid, dim3(kPfThreads), dyn, st, p);
  else
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, false>), grid, dim3(kPfThreads), dyn, st, p);
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
