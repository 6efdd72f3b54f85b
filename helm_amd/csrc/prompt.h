// Causal attention of packed whole prompts on 32 x 32 matrix-core tiles
// (helm_prompt_attn): row i of a sequence gets softmax(cap(q . K^T scale)) . V
// over the sequence's rows j <= i (and j > i - window).
//
// Bound by the matrix cores: 4 D operations a visible (row, head) pair against
// 8 bytes a row and head dim.  A workgroup owns 128 rows of one query head, a wave
// 32 of them (D = 256: 256 rows; few tiles: 32 rows in all, PromptSplit); it walks the
// keys in stages, whose K and V go straight from memory into LDS (two stage buffers,
// one barrier a stage), and computes 32 tokens a step.  Lane l = 32 hh + jr owns query row jr:
//   S^T = K Q^T  (v_mfma_f32_32x32x16): A is K of token tau(jr), B query row jr; with
//         tau(8g + 4h + t) = 16 (g >> 1) + 8h + 4 (g & 1) + t the lane gets row jr's
//         scores of tokens 8 hh .. 8 hh + 7 of both 16-token blocks of the step,
//   O^T += V^T P^T: which are the tokens that B wants of it; A is V by LDS
//         transpose reads.  O register 4g + t of dim group e is dim
//         32 e + 8 g + 4 hh + t of row jr.
// So a row's scores, maximum, sum and output sit in the two lanes (*, jr).  The
// running maximum is refreshed only when a score passes it by 2^8 (f16: 2^6) in weight.
// Weights are rounded once to the 16-bit type, by half a step: 2^-8 (bf16) or 2^-11 (f16) of
// the weight at most, at random, and the row's sum adds the rounded ones.  f16 weights are
// taken times 2^9; those below 2^-23 of the running maximum's fall under the type's normal
// range and are off by 2^-34 of that at most.  An output's relative rms error is 2.0e-3 to
// 2.1e-3 in bf16 and 2.2e-4 to 2.6e-4 in f16, against 1.6e-3 and 1.9e-4 to 2.0e-4 where weights
// stay in fp32 (its own rounding); the low parts of the weights would be a second product
// of P . V, half as much matrix work again.
//
// Hidden tokens take no part whatever they hold: their scores are overwritten,
// and an infinity or NaN in V (which would turn a weight of zero into NaN) shows
// as NaN in an output, upon which the workgroup walks again with V's infinities
// and NaN taken out of the products and added where a row sees them (careful).
#pragma once

#include <type_traits>

#include "attn_chunk32.h"

namespace helm {

// Tokens of a stage, waves of a workgroup, waves a SIMD holds, whether the upper half of
// the query operand stays in LDS, and whether a step works its LDS offsets out anew.
// The query operand and the output of 32 rows take 48, 96 or 192 registers: with the
// query's half in LDS and stages of 32 tokens three waves fit a SIMD at D = 128 and two at
// 256, where one wave's products wait for its own softmax.  bf16, 32 / 8 heads,
// us: D = 128, 16,384 tokens 2,012 -> 1,954, ragged to 2,033 130 -> 120, 14 of 512
// (40 heads) 77 -> 67; D = 256, 10,180 tokens of four prompts, 16 / 8 heads, soft-capped,
// 1,024 window 322 -> 223.  D = 64 is no faster for it (8,192 tokens 315; stages of 32 326,
// four waves a SIMD by force 309 to 502).
template <int D> struct PromptShape {
  static constexpr int kTok = D == 64 ? 64 : 32, kWaves = D == 256 ? 8 : 4;
  static constexpr int kPerSimd = D == 128 ? 3 : 2;
  static constexpr bool kQLds = D != 64, kAnew = D == 256;
};

struct PromptParams {
  const char *q, *k, *v;
  char* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;   // bytes
  const int32_t* cu;
  int B, N, Hq, Hkv, G;
  int tiles;           // grid's row tiles: at least the sequences' together
  float scale;         // >= 0 (a negative one's sign is taken into q)
  uint32_t q_sign;     // xor on packed q pairs
  float softcap;
  int window;          // <= 0: off
  int zero_rest;
};

// Few row tiles: the longest walk of one wave would be the launch's time.  There a workgroup
// owns 32 rows: its waves deal the steps of their walk out among them, each through K and V
// buffers of its own (no barrier in the walk), and join their sums at the end.  Every
// workgroup then loads K and V for 32 rows, not 128 or 256, so this is for launches that
// leave CUs idle: up to 512 such tiles (times heads), which are resident together (one a
// CU, two rounds, at D = 256; up to 640 at D = 64, three a CU), or 1,280 where the sequences
// are 2,048 tokens on average and an extra round's start and join are small beside the
// walks.  The host knows N and B alone: a padded N counts as rows, and one long prompt
// among short ones as their average.
// bf16, us without and with, D = 64 / 128 / 256:
//   8 / 2 heads, 1,200 tokens            20.8 -> 11.7, 29.7 -> 16.7, 67 -> 28
//   8 / 2 heads, 4,800 (1,208 tiles)     69 -> 46,     103 -> 80,    241 -> 185
//   32 / 8 heads, 600 (640)              13.3 -> 10.0, 19.3 -> 18.2, 37 -> 39
// and beyond, where it loses:
//   8 / 2 heads, 4 of 1,200 (1,232)      22.0 -> 21.4, 32.9 -> 37.0, 72 -> 86
//   32 / 8 heads, 4 of 150 (736)         6.7 -> 7.6,   9.3 -> 14.1,  18 -> 30
// Eight waves for four, 8 / 2 heads, 2,400 tokens: D = 64 19.8 -> 24.8, 128 28 -> 39.
template <int D> struct PromptSplit {
  static constexpr int kWaves = 4, kPerSimd = D == 256 ? 1 : 2;
  static constexpr int kTiles = D == 64 ? 640 : 512, kTilesLong = 1280;
};
template <int D> bool prompt_splits(const PromptParams& p) {
  const int64_t wgs = ((int64_t)(p.N + 31) / 32 + p.B) * p.Hq;
  return wgs <= (p.N / 2048 >= p.B ? PromptSplit<D>::kTilesLong : PromptSplit<D>::kTiles);
}

// Sequence b's rows, clamped to the tensors.
struct PromptSeq {
  int first, len;
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int b) {
  const int s = min(max(p.cu[b], 0), p.N);
  const int e = min(max(p.cu[b + 1], s), p.N);
  return {s, e - s};
}

__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return __builtin_amdgcn_readlane(x, 63);
}

// Row tile j (of `rows` rows) of the packed batch: its sequence and its first row in it.
// b < 0: past the last tile, row = its number there.
struct PromptTile {
  int b, first, len, row;
};
// Up to 256 sequences: the tiles that lie furthest into their sequences, whose walks are
// the longest, come first over the whole batch, so that the last workgroups to run
// are short ones.  F(l) = sum of max(0, tiles_b - l) counts the tiles at l or further;
// tile j is at the l with F(l + 1) <= j < F(l), in the (j - F(l + 1))th sequence that
// has one there.
__device__ __forceinline__ PromptTile prompt_tile_longest(const PromptParams& p, int j, int rows,
                                                          int lane) {
  constexpr int K = 4;
  PromptSeq s[K];
  int nt[K], top = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    s[i] = {0, 0};
    if (64 * i + lane < p.B) s[i] = prompt_seq(p, 64 * i + lane);
    nt[i] = (s[i].len + rows - 1) / rows;
    top = max(top, nt[i]);
  }
  auto from = [&](int l) {
    int x = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) x += max(0, nt[i] - l);
    return wave_sum(x);
  };
  const int all = from(0);
  if (j >= all) return {-1, 0, 0, j - all};
  int lo = 0, hi = 1;                       // F(lo) > j >= F(hi), once hi is doubled up to it
  int below = from(1);
  while (below > j) {
    lo = hi;
    hi *= 2;
    below = from(hi);
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, f = from(mid);
    if (f > j) {
      lo = mid;
    } else {
      hi = mid;
      below = f;
    }
  }
  int nth = j - below;
  PromptTile t{-1, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const uint64_t has = __builtin_amdgcn_ballot_w64(nt[i] > lo);
    const int n = __builtin_popcountll(has);
    if (t.b < 0 && nth < n) {
      const int rank = __builtin_popcountll(has & ((1ull << lane) - 1));
      const uint64_t hit = __builtin_amdgcn_ballot_w64(nt[i] > lo && rank == nth);
      const int at = __builtin_ctzll(hit);
      t = {64 * i + at, __builtin_amdgcn_readlane(s[i].first, at),
           __builtin_amdgcn_readlane(s[i].len, at), lo * rows};
    }
    nth -= n;
  }
  return t;
}
// Any number: sequence by sequence, the later rows of each first.
__device__ __forceinline__ PromptTile prompt_tile_in_order(const PromptParams& p, int j, int rows,
                                                           int lane) {
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    PromptSeq s{0, 0};
    if (b0 + lane < p.B) s = prompt_seq(p, b0 + lane);
    const int nt = (s.len + rows - 1) / rows;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(incl, d, 64);
      if (lane >= d) incl += t;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + incl > j);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int first = __builtin_amdgcn_readlane(s.first, at);
      const int len = __builtin_amdgcn_readlane(s.len, at);
      const int t = base + __builtin_amdgcn_readlane(incl, at) - 1 - j;   // from the last
      return {b0 + at, first, len, t * rows};
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return {-1, 0, 0, j - base};
}

// Rows of CH 16-byte chunks in LDS (half a query row, an output row on its way out): chunk
// c of row r sits at slot c ^ out_swz(r), so that 16 lanes that read one chunk of 16 rows,
// or write one, meet every bank group once (rows of 128 bytes: two share 256).
template <int CH> __device__ __forceinline__ int out_swz(int r) {
  return CH == 8 ? (r >> 1) & 7 : r & (CH - 1);
}

template <typename T> __device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
  uint32_t r = 0;
  if ((w & kExp) == kExp) r |= 0xffffu;
  if ((w >> 16 & kExp) == kExp) r |= 0xffff0000u;
  return r;
}

// x f, but an infinity or NaN (a visible one, which counts at any weight) stays what it is where
// f is zero.
__device__ __forceinline__ float scale_finite(float x, float f) {
  return fabsf(x) < INFINITY ? x * f : x;
}

// Joins the waves' sums over 32 rows: a wave's part counts exp2(m - M) of itself, M the
// largest of the row's maxima.  Wave w's sums go where its K (the row's first half) and
// its V were, 64 D bytes each: dims 32 e + 8 g + 4 hh .. + 3 of row r (chunk c = 4 e + g)
// at 16-byte slot 64 c + 32 hh + (r ^ c % 16), so that writes (a chunk's rows) and reads
// (a row's chunks) both meet every bank group.
template <typename T, int D, int NW>
__device__ __forceinline__ void prompt_join(const PromptParams& p, float m, float lsum,
                                            mf_f32x16 (&o)[D / 32], mf_u32x4* kbuf, mf_u32x4* vbuf,
                                            const PromptTile& tl, int hq) {
  constexpr int CPR = D / 8;
  __shared__ float tops[NW][32], sums[NW][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, jr = lane & 31, hh = lane >> 5;
  lsum += __shfl_xor(lsum, 32, 64);
  if (hh == 0) tops[wave][jr] = m;
  __syncthreads();
  float top = tops[0][jr];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = fmaxf(top, tops[w][jr]);
  const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
  if (hh == 0) sums[wave][jr] = lsum * f;
  auto at = [&](int w, int c, int h, int r) {
    return reinterpret_cast<mf_f32x4*>(c < CPR / 2 ? kbuf : vbuf) + 4 * D * w +
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
  for (int i = threadIdx.x; i < 32 * CPR; i += 64 * NW) {
    const int r = i / CPR, c = i % CPR;
    if (tl.row + r >= tl.len) break;
    float l = 0.f;
    mf_f32x4 a{0.f, 0.f, 0.f, 0.f}, b{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      l += sums[w][r];
      a += *at(w, c, 0, r);
      b += *at(w, c, 1, r);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    using Ops = MfmaOps<T>;
    *reinterpret_cast<mf_u32x4*>(p.out + (int64_t)(tl.first + tl.row + r) * p.o_tok +
                                 hq * p.o_head + 16 * c) =
        mf_u32x4{Ops::pk(a[0] * inv, a[1] * inv), Ops::pk(a[2] * inv, a[3] * inv),
                 Ops::pk(b[0] * inv, b[1] * inv), Ops::pk(b[2] * inv, b[3] * inv)};
  }
}

template <typename T, int D, bool kCap, bool kWindow, bool kSplit>
__device__ __forceinline__ void prompt_body(const PromptParams& p) {
  constexpr int NW = kSplit ? PromptSplit<D>::kWaves : PromptShape<D>::kWaves;
  constexpr int kRows = kSplit ? 32 : 32 * NW;       // query rows of the workgroup
  constexpr int kTok = kSplit ? 32 : PromptShape<D>::kTok, SB = kTok / kBlockTok;
  constexpr int NK = D / 16, NE = D / 32, CPR = D / 8;
  constexpr int kRow = 2 * D, kBlk = kBlockTok * kRow;
  constexpr int kShift = std::is_same<T, f16_t>::value ? 9 : 0;
  constexpr float kSlack = chunk_slack(kShift);
  constexpr int kBlkLoads = kBlk / 1024;
  // 16-byte-a-lane loads of a wave and stage: neighbours of one block of K or V, or two
  constexpr int kLoads = 2 * SB * kBlkLoads / NW;
  constexpr bool kQLds = PromptShape<D>::kQLds && !kSplit;
  constexpr bool kAnew = PromptShape<D>::kAnew && !kSplit;
  constexpr int QC = CPR / 2;                // 16-byte chunks of half a query row
  constexpr int NQ = kQLds ? NK / 2 : NK;
  using Ops = MfmaOps<T>;
  using M32 = Mfma32<T>;
  typedef mf_u32x4 StageBuf[2][SB][kBlk / 16];
  __shared__ StageBuf lds0, lds1;
  __shared__ mf_u32x4 ldsk[kSplit ? NW : 1][SB][kBlk / 16], ldsv[kSplit ? NW : 1][SB][kBlk / 16];
  __shared__ mf_u32x4 ldsq[kQLds ? NW * 32 * QC : 1];   // [wave][row][slot]

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, jr = lane & 31, hh = lane >> 5;
  // the query heads of a KV head lie Hkv apart, which for 8 KV heads (2, 4) keeps each on
  // one XCD (its share), whose L2 then reads its K and V once for all of them
  const int hk = blockIdx.x % p.Hq % p.Hkv, hq = hk * p.G + blockIdx.x % p.Hq / p.Hkv;
  const PromptTile tl = p.B <= 256 ? prompt_tile_longest(p, blockIdx.x / p.Hq, kRows, lane)
                                   : prompt_tile_in_order(p, blockIdx.x / p.Hq, kRows, lane);
  if (tl.b < 0) {
    if (!p.zero_rest) return;
    // (the workgroups past the last tile share out the rows outside every sequence)
    const int r0 = min(max(p.cu[0], 0), p.N), r1 = min(max(p.cu[p.B], r0), p.N);
    const int spare = p.tiles - (blockIdx.x / p.Hq - tl.row);
    for (int64_t i = (int64_t)tl.row * NW + wave; i < p.N - (r1 - r0); i += (int64_t)spare * NW) {
      const int64_t r = i < r0 ? i : i + (r1 - r0);
      if (lane < CPR)
        *reinterpret_cast<mf_u32x4*>(p.out + r * p.o_tok + hq * p.o_head + 16 * lane) =
            mf_u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
  const int row_w = kSplit ? tl.row : tl.row + 32 * wave;    // the wave's first row
  const int row = row_w + jr;
  const bool row_ok = row < tl.len;
  const bool wave_rows = row_w < tl.len;
  const int row_last = min(row_w + 31, tl.len - 1);
  const int end = min(tl.row + kRows, tl.len);     // keys: [0, end)
  const int win = kWindow ? p.window : 0;
  const int st0 = kWindow ? max(0, tl.row - win + 1) / kTok : 0;
  const int st1 = (end + kTok - 1) / kTok;

  const float scale2 = p.scale * kLog2E;
  const float inv_cap = kCap ? 1.f / p.softcap : 0.f, cap2 = p.softcap * kLog2E;

  const char* kb = p.k + tl.first * p.k_tok + hk * p.k_head;
  const char* vb = p.v + tl.first * p.v_tok + hk * p.v_head;
  // this wave's loads of a stage straight into LDS: load i of the stage's is part u of
  // i / kBlkLoads, a block's K, then its V, then the next block's; lane l of it fetches the
  // chunk that the swizzle (attn_chunk32.h) keeps in slot 64 u + l; tokens past the
  // sequence's end come in as zeros
  auto dma_stage = [&](int st, StageBuf& dst) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = wave * kLoads + k, kb_v = i / kBlkLoads, u = i % kBlkLoads;
      const int blk = kb_v / 2, is_v = kb_v % 2;                       // (uniform)
      const int tok0 = st * kTok + blk * kBlockTok;
      const int nt = min(max(tl.len - tok0, 0), kBlockTok);
      const int64_t stride = is_v ? p.v_tok : p.k_tok;
      const auto rs = make_rsrc((is_v ? vb : kb) + tok0 * stride,
                                nt ? (nt - 1) * (int)stride + kRow : 0);
      const int t = (64 / CPR) * u + lane / CPR;
      buf_load16_lds(rs, &dst[is_v][blk][64 * u],
                     t * (int)stride + 16 * ((lane % CPR) ^ swz<D>(t)));
    }
  };

  // split: the wave's own loads of stage st's K (0) or V (1) alone
  constexpr int kOwnLoads = SB * kBlkLoads;
  auto dma_own = [&](int st, int is_v) {
#pragma unroll
    for (int blk = 0; blk < SB; ++blk) {
      const int tok0 = st * kTok + blk * kBlockTok;
      const int nt = min(max(tl.len - tok0, 0), kBlockTok);
      const int64_t stride = is_v ? p.v_tok : p.k_tok;
      const auto rs = make_rsrc((is_v ? vb : kb) + tok0 * stride,
                                nt ? (nt - 1) * (int)stride + kRow : 0);
#pragma unroll
      for (int u = 0; u < kBlkLoads; ++u) {
        const int t = (64 / CPR) * u + lane / CPR;
        buf_load16_lds(rs, &(is_v ? ldsv : ldsk)[wave][blk][64 * u],
                       t * (int)stride + 16 * ((lane % CPR) ^ swz<D>(t)));
      }
    }
  };
  // (wave barrier of memory: every LDS read so far has returned)
  auto reads_done = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // all loads into LDS but the youngest kOwnLoads have landed
  auto older_landed = [&] {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOwnLoads) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  if constexpr (!kSplit) dma_stage(st0, lds0);      // (on its way before the query rows)
  mf_u32x4 qop[NQ];
  mf_u32x4* qs = &ldsq[kQLds ? (wave * 32 + jr) * QC : 0];
  {
    const char* qp = p.q + (int64_t)(tl.first + (row_ok ? row : 0)) * p.q_tok + hq * p.q_head;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const mf_u32x4 w = *reinterpret_cast<const mf_u32x4*>(qp + 16 * (2 * i + hh));
      const mf_u32x4 x = row_ok ? w ^ p.q_sign : mf_u32x4{0u, 0u, 0u, 0u};
      if (i < NQ) qop[i < NQ ? i : 0] = x;
      else qs[(2 * (i - NQ) + hh) ^ out_swz<QC>(jr)] = x;     // (read by this wave alone)
    }
  }
  const int g_a = jr >> 3, h_a = (jr >> 2) & 1, t_a = jr & 3;
  const int tau = 16 * (g_a >> 1) + 8 * h_a + 4 * (g_a & 1) + t_a;
  const int kblk = tau >> 4, ktok = tau & 15;
  const int nl = lane & 15;
  // Byte offsets of a step's operands in its stage buffer: the swizzle is an XOR below the
  // row's size, so every operand lies at one offset XOR a constant.  (D = 256 does that
  // anew for each read: kept in registers, 24 offsets pushed others to memory.)
  const int k_off = kblk * kBlk + ktok * kRow + 16 * (hh ^ swz<D>(ktok));
  const int v_tok0 = 8 * hh + (nl >> 2);
  const int v_off = v_tok0 * kRow + 16 * ((2 * (jr >> 4) + ((nl & 3) >> 1)) ^ swz<D>(v_tok0)) +
                    8 * (nl & 1);
  const int q_off = 16 * (hh ^ out_swz<QC>(jr));
  auto anew = [](int off) {
    if constexpr (kAnew) asm volatile("" : "+v"(off));
    return off;
  };
  // (from the first of the step's two blocks of K or V)
  auto k_operand = [&](const mf_u32x4* kk, int i, int off) {
    return *reinterpret_cast<const mf_u32x4*>(reinterpret_cast<const char*>(kk) + (off ^ (32 * i)));
  };
  auto v_operand = [&](const mf_u32x4* vv, int u, int z, int e, int off) {
    // token v_tok0 + 4 z: the row four further, whose swizzle differs by z's bit
    return ld_tr16(reinterpret_cast<const char*>(vv) + (off ^ (64 * e) ^ (16 * z)) + u * kBlk +
                   4 * kRow * z);
  };

  float m, lsum;
  mf_f32x16 o[NE];

  auto step = [&](auto careful, int tok0, const mf_u32x4* kk, const mf_u32x4* vv) {
    if constexpr (kSplit) older_landed();      // K
    mf_f32x16 sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
    const int ko = anew(k_off), qo = anew(q_off);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const mf_u32x4 q = i < NQ ? qop[i < NQ ? i : 0]
                                : *reinterpret_cast<const mf_u32x4*>(
                                      reinterpret_cast<const char*>(qs) + (qo ^ (32 * (i - NQ))));
      sc = M32::mma(k_operand(kk, i, ko), q, sc);
      // (few operands ahead)
      if (kAnew && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kSplit) {
      reads_done();
      dma_own(tok0 / kTok + NW, 0);            // (past the sequence: zeros, never used)
    }
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = sc[r];
    if constexpr (kCap) softcap_scores<16>(x, p.scale * inv_cap, cap2);
    const float mul = kCap ? 1.f : scale2;     // logits in base-2 units
    const bool limit = tok0 + 31 > row_w || (kWindow && tok0 <= row_last - win);
    if (limit) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int t = tok0 + 16 * (r >> 3) + 8 * hh + (r & 7);
        if (t > row || (kWindow && t <= row - win)) x[r] = -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top *= mul;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0, 0)) {
      float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
      if constexpr (kShift) mn = ceilf(mn);    // (so that m - kShift is exact)
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
    uint32_t w[8];
    uint32_t some[8];                          // careful: 1 where the row sees the token
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w0 = __builtin_amdgcn_exp2f(fmaf(x[2 * i], mul, -base));
      const float w1 = __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], mul, -base));
      w[i] = Ops::pk(w0, w1);
      lsum = dot2<T>(w[i], Ops::ones8()[0], lsum);
      if constexpr (careful.value) {
        const uint32_t one = Ops::ones8()[0];
        some[i] = (x[2 * i] != -INFINITY ? one & 0xffffu : 0u) |
                  (x[2 * i + 1] != -INFINITY ? one & 0xffff0000u : 0u);
      }
    }
    if constexpr (kSplit) older_landed();      // V
    const int vo = anew(v_off);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const mf_u32x4 pop{w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]};
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const uint2 a0 = v_operand(vv, u, 0, e, vo);
        const uint2 a1 = v_operand(vv, u, 1, e, vo);
        mf_u32x4 vop{a0.x, a0.y, a1.x, a1.y};
        if constexpr (careful.value) {
          mf_u32x4 bad;
#pragma unroll
          for (int i = 0; i < 4; ++i) bad[i] = nonfinite_halves<T>(vop[i]);
          if (__builtin_amdgcn_ballot_w64((bad[0] | bad[1] | bad[2] | bad[3]) != 0u)) {
            const mf_u32x4 sop{some[4 * u], some[4 * u + 1], some[4 * u + 2], some[4 * u + 3]};
            constexpr uint32_t kMant = std::is_same<T, bf16_t>::value ? 0x7fu : 0x3ffu;
            const uint32_t one = Ops::ones8()[0];
            mf_u32x4 pos, neg, nan;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t is_nan = 0, is_neg = 0;
              if (vop[i] & kMant) is_nan |= 0xffffu;
              if (vop[i] >> 16 & kMant) is_nan |= 0xffff0000u;
              if (vop[i] & 0x8000u) is_neg |= 0xffffu;
              if (vop[i] & 0x80000000u) is_neg |= 0xffff0000u;
              nan[i] = one & bad[i] & is_nan;
              neg[i] = one & bad[i] & ~is_nan & is_neg;
              pos[i] = one & bad[i] & ~is_nan & ~is_neg;
              vop[i] &= ~bad[i];
            }
            mf_f32x16 zero;
#pragma unroll
            for (int r = 0; r < 16; ++r) zero[r] = 0.f;
            const mf_f32x16 hp = M32::mma(pos, sop, zero), hn = M32::mma(neg, sop, zero),
                            hx = M32::mma(nan, sop, zero);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              if (hp[r] != 0.f) o[e][r] += INFINITY;
              if (hn[r] != 0.f) o[e][r] -= INFINITY;
              if (hx[r] != 0.f) o[e][r] = __builtin_nanf("");
            }
          }
        }
        o[e] = M32::mma(vop, pop, o[e]);
        if (kAnew && e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto walk = [&](auto careful) {
    m = -INFINITY;
    lsum = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[e][r] = 0.f;
    // a step none of whose tokens any row of the wave sees is left out (uniform)
    auto part = [&](int st, int bp, const StageBuf& cur) {
      const int tok0 = st * kTok + bp * kBlockTok;
      if (wave_rows && tok0 <= row_last && !(kWindow && tok0 + 31 <= row_w - win))
        step(careful, tok0, &cur[0][bp][0], &cur[1][bp][0]);
    };
    if constexpr (kSplit) {
      if (st0 + wave < st1) {
        dma_own(st0 + wave, 0);
        __builtin_amdgcn_sched_barrier(0);    // (K's loads are the older ones)
        dma_own(st0 + wave, 1);
      }
      for (int st = st0 + wave; st < st1; st += NW) {
        step(careful, st * kTok, &ldsk[wave][0][0], &ldsv[wave][0][0]);
        reads_done();
        dma_own(st + NW, 1);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // (no load is on its way any more)
    } else if constexpr (careful.value) {
      for (int st = st0; st < st1; ++st) {
        __syncthreads();                    // (every wave is done with the stage before)
        dma_stage(st, lds0);
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
#pragma unroll 1
        for (int bp = 0; bp < SB; bp += 2) part(st, bp, lds0);
      }
    } else {
      auto stage = [&](int st, const StageBuf& cur, StageBuf& nxt) {
        // stage st is in LDS (this wave's loads done, then everyone's), and every wave
        // is done with the other buffer, which the next stage's loads fill
        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
        __syncthreads();
        if (st + 1 < st1) dma_stage(st + 1, nxt);
        part(st, 0, cur);
        if constexpr (SB > 2) part(st, 2, cur);
      };
      for (int st = st0; st < st1; st += 2) {
        stage(st, lds0, lds1);
        if (st + 1 < st1) stage(st + 1, lds1, lds0);
      }
    }
  };
  walk(std::false_type{});
  bool odd = false;
#pragma unroll
  for (int e = 0; e < NE; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = odd || o[e][r] != o[e][r];
  if constexpr (kSplit) {
    if (__builtin_amdgcn_ballot_w64(odd && row_ok)) walk(std::true_type{});
    prompt_join<T, D, NW>(p, m, lsum, o, &ldsk[0][0][0], &ldsv[0][0][0], tl, hq);
    return;
  }
  // (the barrier also ends every wave's reads of the buffers that a second walk fills)
  if (__syncthreads_or(odd && row_ok)) {
    walk(std::true_type{});
    __syncthreads();
  }

  // The rows leave through LDS, each wave's in a part of its own: 16 bytes a lane, whole
  // rows a store.  (Straight from the registers a row's lines went out in 16-byte pieces, which
  // bound short prompts: 14 of 512 tokens, 40 heads of 128, 89 -> 72 us.)
  const float l = lsum + __shfl_xor(lsum, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  // (with the query's half in LDS: half a row at a time, where that was)
  constexpr int kHalves = kQLds ? 2 : 1, EH = NE / kHalves, CH = CPR / kHalves;
  char* rows = kQLds ? reinterpret_cast<char*>(&ldsq[wave * 32 * QC])
                     : reinterpret_cast<char*>(&lds0[0][0][0]) + wave * (32 * kRow);
  char* op = p.out + (int64_t)(tl.first + row_w) * p.o_tok + hq * p.o_head + 16 * (lane % CH);
#pragma unroll
  for (int half = 0; half < kHalves; ++half) {
#pragma unroll
    for (int e = 0; e < EH; ++e)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const mf_f32x16& oe = o[half * EH + e];
        const int slot = (4 * e + g) ^ out_swz<CH>(jr);
        *reinterpret_cast<uint2*>(rows + jr * (16 * CH) + 16 * slot + 8 * hh) =
            make_uint2(Ops::pk(oe[4 * g] * inv, oe[4 * g + 1] * inv),
                       Ops::pk(oe[4 * g + 2] * inv, oe[4 * g + 3] * inv));
      }
#pragma unroll
    for (int i = 0; i < 32 * CH / 64; ++i) {
      const int r = (64 / CH) * i + lane / CH;
      const int slot = (lane % CH) ^ out_swz<CH>(r);
      const mf_u32x4 w = *reinterpret_cast<const mf_u32x4*>(rows + r * (16 * CH) + 16 * slot);
      if (row_w + r < tl.len)
        *reinterpret_cast<mf_u32x4*>(op + r * p.o_tok + 16 * CH * half) = w;
    }
  }
}

template <typename T, int D, bool kCap, bool kWindow>
__global__ __launch_bounds__(64 * PromptShape<D>::kWaves, PromptShape<D>::kPerSimd)
void prompt_attn_kernel(PromptParams p) {
  prompt_body<T, D, kCap, kWindow, false>(p);
}
template <typename T, int D, bool kCap, bool kWindow>
__global__ __launch_bounds__(64 * PromptSplit<D>::kWaves, PromptSplit<D>::kPerSimd)
void prompt_split_kernel(PromptParams p) {
  prompt_body<T, D, kCap, kWindow, true>(p);
}

template <typename T, int D, bool kCap, bool kWindow>
hipError_t launch_prompt_form(PromptParams p, hipStream_t st) {
  const bool split = prompt_splits<D>(p);
  const int rows = split ? 32 : 32 * PromptShape<D>::kWaves;
  p.tiles = (p.N + rows - 1) / rows + p.B;
  const dim3 grid((uint32_t)p.tiles * p.Hq);
  if (split)
    hipLaunchKernelGGL((prompt_split_kernel<T, D, kCap, kWindow>), grid,
                       dim3(64 * PromptSplit<D>::kWaves), 0, st, p);
  else
    hipLaunchKernelGGL((prompt_attn_kernel<T, D, kCap, kWindow>), grid,
                       dim3(64 * PromptShape<D>::kWaves), 0, st, p);
  return hipGetLastError();
}
template <typename T, int D>
hipError_t launch_prompt_dim(const PromptParams& p, hipStream_t st) {
  const bool cap = p.softcap > 0.f, win = p.window > 0;
  if (cap && win) return launch_prompt_form<T, D, true, true>(p, st);
  if (cap) return launch_prompt_form<T, D, true, false>(p, st);
  if (win) return launch_prompt_form<T, D, false, true>(p, st);
  return launch_prompt_form<T, D, false, false>(p, st);
}

// One per element type, each in a source of its own (prompt_bf16.hip, prompt_f16.hip).
hipError_t launch_prompt_bf16(const PromptParams& p, int D, hipStream_t st);
hipError_t launch_prompt_f16(const PromptParams& p, int D, hipStream_t st);

template <typename T>
hipError_t launch_prompt_type(const PromptParams& p, int D, hipStream_t st) {
  if (D == 64) return launch_prompt_dim<T, 64>(p, st);
  if (D == 128) return launch_prompt_dim<T, 128>(p, st);
  return launch_prompt_dim<T, 256>(p, st);
}

}  // namespace helm
