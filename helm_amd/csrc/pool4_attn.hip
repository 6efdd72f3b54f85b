// Decode attention over a pool of 4-bit pages (helm_pool4_decode_attn): for
// every sequence, KV head and query row softmax(cap(q . K^T scale) + mask) . V
// over the cached tokens, K and V as pool4.h stores them.
//
// Bound by memory: 17 D / 16 bytes a token and KV head (K and V), each read
// once.  The codes become bf16 matrix-core operands in registers (two values an
// instruction, exact), so nothing but the 4-bit page crosses memory.
//
// Work: grid.x = split, grid.y = KV head * row tiles of 16 query rows, grid.z =
// sequence; four waves.  The sequence's blocks of 32 tokens (two tiles) go round
// the waves of all splits: wave w of split s takes blocks 4 s + w + 4 splits * j.  A
// wave's first blocks so follow from the launch alone (their table entries are
// read beside the sequence's length, not after it), a sequence of any length is
// spread evenly, and a short one uses few splits.
// Lane (n, h) = (lane % 16, lane / 16):
//   S^T = K Q^T  (16 x 16 x 32, one product per tile and 32 dims): A is token n's
//         dims D/4 h + 8i .. + 7, which is word i of the lane's D/8 contiguous code
//         bytes; B is query row n at the same dims.  The lane gets row n's scores
//         of tokens 4h .. 4h + 3 of each tile: eight a block.
//   O^T += V^T P^T  (K = the block's 32 tokens): B is row n's weights, the lane's own
//         eight; A is V of those eight tokens at chunk n's dim e, e = 0 .. D/16 - 1
//         (one product each).  The lane gets row n at dims D/4 h .. + D/4 - 1.
// Row n's scores, maximum, sum and output all sit in the four lanes (n, *): no
// value moves between lanes until the split's end.  The maximum is refreshed
// (all lanes together) only when a score passes it by 2^8; weights stay below
// that and enter the product as hi + lo bf16 parts (~2^-17 of the weight).
// f16 queries enter as hi + lo parts too (exact: 11 bits in 16).
//
// Hidden tokens (past the sequence's length, past the causal limit, or under a
// mask of -inf) take no part whatever their K and V hold: their scores are
// overwritten, and where V's group stands for NaN the products take zeros there
// and the NaN is put into the rows that see such a token, however small its weight.
// A row with nothing visible is zeros.
#include <algorithm>
#include <string>
#include <type_traits>

#include "attn_mfma.h"
#include "pool4.h"

namespace helm {

int report_error(int code, const std::string& msg);

namespace {

constexpr int kP4Waves = 4;
constexpr int kP4Rows = 16;
// blocks of a wave in registers, all but one in flight; D = 256's are twice as large
constexpr int p4_bufs(int D) { return D == 256 ? 2 : 3; }
constexpr float kP4Slack = 8.f;      // base-2 units
constexpr float kP4Log2E = 1.4426950408889634f;

struct P4Attn {
  const void* q;
  void* out;
  const char* pool;
  int64_t slot_bytes, head_bytes;
  int n_slots;
  const int32_t* table;
  int64_t table_stride;
  int max_pages, tpp, tpp_log2;      // tiles per page; its log2 or -1
  const int32_t* seq_lens;
  int B, Hq, Hkv, G, S, row_tiles;
  int q16;                           // 1: q and out are f16, else bf16
  int splits;
  int causal;
  float scale, softcap;
  const char* mask;
  int64_t mask_b, mask_h, mask_q;    // elements
  int mask_dt, mask_len;             // tokens from mask_len on are hidden
  float* part_o;                     // [tile][splits][16 rows][D], tile = (b, KV head, row tile)
  float* part_ml;                    // [tile][splits][16 rows][2]
};

// Sequence b's tokens, tiles, blocks, and the splits that have any of them.
struct P4Seq {
  int len, tiles, blocks, splits;
};
__device__ __forceinline__ P4Seq p4_seq(const P4Attn& a, int b) {
  P4Seq s;
  const int64_t room = (int64_t)a.max_pages * a.tpp * kP4Tok;
  s.len = (int)min((int64_t)max(0, a.seq_lens[b]), room);
  s.tiles = (int)(((int64_t)s.len + kP4Tok - 1) / kP4Tok);
  s.blocks = (s.tiles + 1) / 2;
  s.splits = min(a.splits, (s.blocks + kP4Waves - 1) / kP4Waves);
  return s;
}

// What a lane reads of one tile.
template <int D> struct P4Raw {
  uint32_t k[D / 32], v[D / 32];     // codes
  uint32_t ke, ve;                   // exponent bytes: K of its group(s), V of its four tokens
};

template <int D>
__device__ __forceinline__ P4Raw<D> p4_load(const char* tile, bool there, int n, int h) {
  P4Raw<D> r;
  const auto rs = make_rsrc(tile, there ? P4<D>::kBytes : 0);   // (absent: zeros)
  constexpr int W = D / 32;
  const int ko = n * (D / 2) + h * (D / 8);
  const int vo = P4<D>::kVc + n * (D / 2) + h * (D / 8);
  if constexpr (W == 2) {
    const auto k = __builtin_amdgcn_raw_buffer_load_b64(rs, ko, 0, 2);
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(rs, vo, 0, 2);
    r.k[0] = k[0]; r.k[1] = k[1];
    r.v[0] = v[0]; r.v[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const mf_u32x4 k = buf_load16_nt(rs, ko + 4 * i), v = buf_load16_nt(rs, vo + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r.k[i + j] = k[j];
        r.v[i + j] = v[j];
      }
    }
  }
  const int ke = P4<D>::kKe + n * P4<D>::kGroups;
  if constexpr (D == 256) r.ke = __builtin_amdgcn_raw_buffer_load_b16(rs, ke + 2 * h, 0, 0);
  else r.ke = __builtin_amdgcn_raw_buffer_load_b8(rs, ke + (D == 64 ? h / 2 : h), 0, 0);
  const int group = n * (D / 16) / kP4Group;
  r.ve = __builtin_amdgcn_raw_buffer_load_b32(rs, P4<D>::kVe + group * kP4Tok + 4 * h, 0, 0);
  return r;
}

// The two codes of byte B of w, or all eight, times s, as bf16 (exact).
template <int B> __device__ __forceinline__ uint32_t p4_decode2(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
}
__device__ __forceinline__ mf_u32x4 p4_decode8(uint32_t w, float s) {
  return mf_u32x4{p4_decode2<0>(w, s), p4_decode2<1>(w, s), p4_decode2<2>(w, s),
                  p4_decode2<3>(w, s)};
}
// Pair c (dims 2c, 2c + 1 of the lane's chunk) of token j of a tile's four.
template <int D>
__device__ __forceinline__ uint32_t p4_v_pair(const P4Raw<D>& r, int j, int c, float s) {
  constexpr int PB = D / 32;                 // bytes a token's chunk: pairs
  const int byte = j * PB + c;
  const uint32_t w = r.v[byte >> 2];
  switch (byte & 3) {
    case 0: return p4_decode2<0>(w, s);
    case 1: return p4_decode2<1>(w, s);
    case 2: return p4_decode2<2>(w, s);
    default: return p4_decode2<3>(w, s);
  }
}

__device__ __forceinline__ mf_u32x2 load8_any(const char* p) {
  struct __attribute__((packed)) Any { mf_u32x2 v; };
  return reinterpret_cast<const Any*>(p)->v;
}

// Any byte of x or y from 192 on: a group past 2^65, a NaN (255), or a byte that no write leaves
// (253 and 254, whose codes pass bf16's range).
__device__ __forceinline__ bool any_high(uint32_t x, uint32_t y) {
  return (((x & (x << 1)) | (y & (y << 1))) & 0x80808080u) != 0u;
}

__device__ __forceinline__ void add_scaled(float4& acc, float f, const float4 v) {
  acc.x += f * v.x;
  acc.y += f * v.y;
  acc.z += f * v.z;
  acc.w += f * v.w;
}

// Dims 4 col .. of query row `row` (of the head's G * S) of the output: acc / sum.
template <int D>
__device__ __forceinline__ void store_row(const P4Attn& a, int b, int hk, int row, int col,
                                          const float4 acc, float sum) {
  const RowCoord c = row_coord(row, a.G);
  const int64_t r = (int64_t)(b * a.Hq + hk * a.G + c.g) * a.S + c.s;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint2 w;
  if (a.q16)
    w = make_uint2(MfmaOps<f16_t>::pk(acc.x * inv, acc.y * inv),
                   MfmaOps<f16_t>::pk(acc.z * inv, acc.w * inv));
  else
    w = make_uint2(MfmaOps<bf16_t>::pk(acc.x * inv, acc.y * inv),
                   MfmaOps<bf16_t>::pk(acc.z * inv, acc.w * inv));
  // (out is 8-byte aligned or better: checked on the host)
  *reinterpret_cast<uint2*>(reinterpret_cast<char*>(a.out) + 2 * (r * D + 4 * col)) = w;
}

// MB: bytes of a mask element (0: no mask).
template <int D, int QP, int MB, bool kCap>
__global__ __launch_bounds__(64 * kP4Waves) void pool4_attn_kernel(P4Attn a) {
  constexpr bool kMask = MB != 0;
  constexpr int NB = p4_bufs(D);
  constexpr int NS = D / 32;                 // 32-dim steps of q . k
  constexpr int NE = D / 16;                 // dims of a V chunk: products of P . V
  using Ops = MfmaOps<bf16_t>;
  __shared__ float sh_o[kP4Waves][kP4Rows][D + 4];
  __shared__ float2 sh_ml[kP4Waves][kP4Rows];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, n = lane & 15, h = lane >> 4;
  const int split = blockIdx.x;
  const int hk = blockIdx.y % a.Hkv, rt = blockIdx.y / a.Hkv;
  const int b = blockIdx.z;
  const int rows_all = a.G * a.S;
  const int row0 = rt * kP4Rows, nrows = min(kP4Rows, rows_all - row0);

  // Lane i holds the slot of tile i % 2 of the wave's block win0 + i / 2, a window of
  // blocks read before the first and then ahead of the next (scalar loads a block
  // ahead came too late: 64 k tokens x 4 at 256 workgroups 56 -> 64 us); a tile's place
  // in its page is stepped without a division.
  const char* head_base = a.pool + hk * a.head_bytes;
  const int blk0 = split * kP4Waves + wave, hop = a.splits * kP4Waves;
  auto slots_from = [&](int j0) -> int {
    const int64_t t = 2 * (blk0 + (int64_t)hop * (j0 + (lane >> 1))) + (lane & 1);
    const int64_t page = a.tpp_log2 >= 0 ? t >> a.tpp_log2 : t / a.tpp;
    return page < a.max_pages ? a.table[(int64_t)b * a.table_stride + page] : -1;
  };
  constexpr int kWin = 30;                 // blocks of a later window: whole rounds
  int slots = slots_from(0), win0 = 0;
  int refill = NB - 1 + (32 - (NB - 1)) / NB * NB;
  int slots_next = slots_from(refill);
  const int hop_in = a.tpp_log2 >= 0 ? (2 * hop) & (a.tpp - 1) : 2 * hop % a.tpp;
  int in_page = a.tpp_log2 >= 0 ? (2 * blk0) & (a.tpp - 1) : 2 * blk0 % a.tpp;
  const P4Seq sq = p4_seq(a, b);
  if (split >= max(1, sq.splits)) return;
  const int mine = blk0 < sq.blocks ? (sq.blocks - 1 - blk0) / hop + 1 : 0;

  // query row n of the tile: position and head of its group
  const bool row_ok = n < nrows;
  const RowCoord rc = row_coord(row0 + (row_ok ? n : 0), a.G);
  const int head = hk * a.G + rc.g;
  mf_u32x4 qop[QP][NS];
  {
    const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) +
                         ((int64_t)(b * a.Hq + head) * a.S + rc.s) * D + (D / 4) * h;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      mf_u32x4 w = *reinterpret_cast<const mf_u32x4*>(qp + 8 * i);
      if (!row_ok) w = mf_u32x4{0u, 0u, 0u, 0u};
      if constexpr (QP == 1) {
        qop[0][i] = w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          const uint32_t wj = w[j];
          const h2 x = __builtin_bit_cast(h2, wj);
          uint32_t hi, lo;
          Ops::split2((float)x[0], (float)x[1], hi, lo);
          qop[0][i][j] = hi;
          qop[1][i][j] = lo;
        }
      }
    }
  }
  // row n of the mask; a block's elements are loaded with its K and V (a load behind
  // the next blocks' would have to wait for those too), four at a time at the mask's
  // own alignment, pulled back into the row where they would pass its end
  const char* mrow = nullptr;
  const bool mwide = a.mask_len >= 4;
  if constexpr (kMask)
    mrow = a.mask + MB * (b * a.mask_b + head * a.mask_h + rc.s * a.mask_q);
  // with a mask the logits stay in natural units (finfo.min would leave fp32's
  // range in base 2), the weight's exponent is scaled instead
  const float unit = kMask ? 1.f : kP4Log2E, to2 = kMask ? kP4Log2E : 1.f;
  const float slack = kMask ? kP4Slack / kP4Log2E : kP4Slack;
  const float qscale = a.scale * unit;
  const float inv_cap = kCap ? 1.f / a.softcap : 0.f, cap = a.softcap * unit;
  // row n's last visible token
  const int last_vis = a.causal ? min(sq.len - 1, sq.len - a.S + rc.s) : sq.len - 1;
  // the block's tokens all lie at or before every row's last visible one
  const int all_vis = a.causal ? sq.len - a.S + row0 / a.G : sq.len - 1;

  float m = -INFINITY, l = 0.f;
  mf_f32x4 o[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) o[e] = mf_f32x4{0.f, 0.f, 0.f, 0.f};

  struct Block {
    P4Raw<D> r[2];
    uint32_t mk[kMask ? 2 * MB : 1];       // eight mask elements
    int gone;                              // bit s: tile s is not there
  };
  // the wave's block j (past its last: zeros, nothing read)
  auto load = [&](int j, Block& k) {
    if constexpr (kMask) {
      const int64_t tok = 32 * (blk0 + (int64_t)hop * j) + 4 * h;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const char* src = mwide ? mrow + MB * min(tok + 16 * s, (int64_t)a.mask_len - 4)
                                : reinterpret_cast<const char*>(a.q);
        if constexpr (MB == 2) {
          const mf_u32x2 w = load8_any(src);
          k.mk[2 * s] = w[0];
          k.mk[2 * s + 1] = w[1];
        } else {
          const mf_u32x4 w = load16_any(src);
#pragma unroll
          for (int i = 0; i < 4; ++i) k.mk[4 * s + i] = w[i];
        }
      }
    }
    k.gone = 0;
    const int in[2] = {in_page, in_page + 1 == a.tpp ? 0 : in_page + 1};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int slot = __builtin_amdgcn_readlane(slots, 2 * (j - win0) + s);
      // (a slot that the pool does not have hides its tile)
      const bool there = (j < mine) & (2 * (blk0 + hop * j) + s < sq.tiles) &
                         ((uint32_t)slot < (uint32_t)a.n_slots);
      // (64 bits: a page of eight million tokens of 256 dims passes 2^31 bytes)
      const char* tile = head_base + (there ? slot : 0) * a.slot_bytes +
                         (int64_t)in[s] * P4<D>::kBytes;
      k.r[s] = p4_load<D>(tile, there, n, h);
      if (!there) k.gone |= 1 << s;
    }
    in_page += hop_in;
    if (in_page >= a.tpp) in_page -= a.tpp;
  };
  auto step = [&](int j, Block& k) {
    P4Raw<D> (&r)[2] = k.r;
    const int tok0 = 32 * (blk0 + hop * j);
    float x[8];
    {
      mf_f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) {      // (the two tiles' sums side by side)
          const uint32_t e = D == 256 && i >= NS / 2 ? r[s].ke >> 8 : r[s].ke & 255u;
          const mf_u32x4 kop = p4_decode8(r[s].k[i], p4_scale(e));
#pragma unroll
          for (int p = 0; p < QP; ++p) sc[s] = Ops::mma(kop, qop[p][i], sc[s]);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = sc[j >> 2][j & 3];
    }
    if constexpr (kCap) {
      softcap_scores<8>(x, a.scale * inv_cap, cap);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= qscale;
    }
    auto tok = [&](int j) { return tok0 + 16 * (j >> 2) + 4 * h + (j & 3); };
    if constexpr (kMask) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float mk;
        if constexpr (MB == 2) {
          const uint32_t w = k.mk[j >> 1] >> (16 * (j & 1)) & 0xffffu;
          mk = a.mask_dt == HELM_BF16
                   ? __uint_as_float(w << 16)
                   : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
        } else {
          mk = __uint_as_float(k.mk[j]);
        }
        if (tok0 + 31 >= a.mask_len) {       // (uniform: the mask's last block)
          mk = -INFINITY;
          if (tok(j) < a.mask_len) mk = (MaskRow{mrow, a.mask_dt})[tok(j)];
        }
        x[j] = mk == -INFINITY ? -INFINITY : x[j] + mk;
      }
    }
    const bool limits = k.gone || tok0 + 31 > all_vis;      // uniform
    if (limits) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (tok(j) > last_vis || (k.gone >> (j >> 2) & 1)) x[j] = -INFINITY;
      // exponents of tokens past the sequence are whatever the page held
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (tok(j) >= sq.len) r[j >> 2].ve &= ~(255u << (8 * (j & 3)));
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
    if (__builtin_amdgcn_ballot_w64(top > m + slack)) {
      float mn = fmaxf(m, top);
      mn = fmaxf(mn, __shfl_xor(mn, 16, 64));
      mn = fmaxf(mn, __shfl_xor(mn, 32, 64));
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * to2);
      m = mn;
      l *= f;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[e] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f((x[j] - base) * to2);
    l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    mf_u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a0, b0;
      Ops::split2(w[2 * j], w[2 * j + 1], a0, b0);
      hi[j] = a0;
      lo[j] = b0;
    }
    const bool high = __builtin_amdgcn_ballot_w64(any_high(r[0].ve, r[1].ve)) != 0;
    uint32_t ff = 0;                         // bit j: token j's group stands for NaN
    if (__builtin_expect(high, 0)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t& ve = r[j >> 2].ve;
        if (((ve >> (8 * (j & 3))) & 255u) > 252u) {
          ff |= 1u << j;
          ve &= ~(255u << (8 * (j & 3)));
        }
      }
    }
    float vs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vs[j] = p4_scale((r[j >> 2].ve >> (8 * (j & 3))) & 255u);
#pragma unroll
    for (int c = 0; c < NE / 2; ++c) {
      uint32_t d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = p4_v_pair<D>(r[j >> 2], j & 3, c, vs[j]);
      const mf_u32x4 even{pack_lo(d[0], d[1]), pack_lo(d[2], d[3]), pack_lo(d[4], d[5]),
                          pack_lo(d[6], d[7])};
      const mf_u32x4 odd{pack_hi(d[0], d[1]), pack_hi(d[2], d[3]), pack_hi(d[4], d[5]),
                         pack_hi(d[6], d[7])};
      o[2 * c] = Ops::mma(even, hi, o[2 * c]);
      o[2 * c + 1] = Ops::mma(odd, hi, o[2 * c + 1]);
      o[2 * c] = Ops::mma(even, lo, o[2 * c]);
      o[2 * c + 1] = Ops::mma(odd, lo, o[2 * c + 1]);
    }
    if (__builtin_expect(high, 0)) {
      // ones at the NaN tokens (a whole chunk lies in one group) times ones at those that
      // the row sees (not its weights, which may be zero by rounding): a row that sees any
      // gets NaN in every dim of the chunk, and no later factor takes that away
      mf_u32x4 one, sees;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        one[j] = (((ff >> (2 * j)) & 1u) ? 0x3F80u : 0u) |
                 (((ff >> (2 * j + 1)) & 1u) ? 0x3F800000u : 0u);
        sees[j] = (x[2 * j] != -INFINITY ? 0x3F80u : 0u) |
                  (x[2 * j + 1] != -INFINITY ? 0x3F800000u : 0u);
      }
      const mf_f32x4 hit = Ops::mma(one, sees, mf_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        if (!(hit[r4] == 0.f))
#pragma unroll
          for (int e = 0; e < NE; ++e) o[e][r4] = __builtin_nanf("");
    }
  };
  // block j is computed while the next NB - 1 are on their way; loads past the
  // last block read nothing, so that every round issues the same
  Block buf[NB];
#pragma unroll
  for (int i = 0; i < NB - 1; ++i) load(i, buf[i]);
  for (int j = 0; j < mine; j += NB) {
    if (j + NB - 1 == refill) {
      slots = slots_next;
      win0 = refill;
      refill += kWin;
      slots_next = slots_from(refill);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      load(j + i + NB - 1, buf[(i + NB - 1) % NB]);
      __builtin_amdgcn_sched_barrier(0);
      if (j + i < mine) step(j + i, buf[i]);
    }
  }

  // the split's rows: the waves' states joined in LDS, four dims a thread
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (h == 0) sh_ml[wave][n] = make_float2(m, l);
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4)
#pragma unroll
    for (int e = 0; e < NE; ++e) sh_o[wave][n][(4 * h + r4) * NE + e] = o[e][r4];
  __syncthreads();
  constexpr int C = D / 4, R = 64 * kP4Waves / C;     // columns of a row; rows at a time
  const int col = tid % C;
  const int tile = (b * a.Hkv + hk) * a.row_tiles + rt;
  const bool alone = sq.splits <= 1;
  for (int row = tid / C; row < nrows; row += R) {
    float mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kP4Waves; ++w) mx = fmaxf(mx, sh_ml[w][row].x);
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < kP4Waves; ++w) {
      const float2 ml = sh_ml[w][row];
      const float f = __builtin_amdgcn_exp2f((ml.x - base) * to2);
      sum += f * ml.y;
      add_scaled(acc, f, *reinterpret_cast<const float4*>(&sh_o[w][row][4 * col]));
    }
    if (alone) {
      store_row<D>(a, b, hk, row0 + row, col, acc, sum);
    } else {
      const int64_t p = ((int64_t)tile * a.splits + split) * kP4Rows + row;
      reinterpret_cast<float4*>(a.part_o)[p * C + col] = acc;
      if (col == 0) reinterpret_cast<float2*>(a.part_ml)[p] = make_float2(mx, sum);
    }
  }
}

// Row blockIdx.y of tile blockIdx.x from its splits' partials: a thread holds four dims
// and every (256 / (D / 4))th split, eight of them in flight; the threads of one column
// meet in LDS.  (3.4 us at 32 splits.  Joined by the last split of a tile to arrive, one
// launch less but coherent accesses and a ticket: 32 k tokens 16.2 us against 15.9 for
// both kernels, 64 k x 4 54.7 against 55.)
template <int D>
__global__ __launch_bounds__(256) void pool4_join_kernel(P4Attn a) {
  constexpr int C = D / 4, R = 256 / C, U = 8;
  __shared__ float4 sh_o[R][C];
  __shared__ float2 sh_ml[R];
  const int tile = blockIdx.x, row = blockIdx.y;
  const int rt = tile % a.row_tiles, hk = tile / a.row_tiles % a.Hkv;
  const int b = tile / a.row_tiles / a.Hkv;
  if (rt * kP4Rows + row >= a.G * a.S) return;
  const int n = p4_seq(a, b).splits;
  if (n <= 1) return;                              // written by its only split
  const float to2 = a.mask ? kP4Log2E : 1.f;       // (the units of the partials' maxima)
  const int c = threadIdx.x % C, g = threadIdx.x / C;
  const int64_t p0 = (int64_t)tile * a.splits * kP4Rows + row;
  const float2* part_ml = reinterpret_cast<const float2*>(a.part_ml) + p0;
  const float4* part_o = reinterpret_cast<const float4*>(a.part_o) + p0 * C + c;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = g; s0 < n; s0 += U * R) {
    float2 ml[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = (int64_t)min(s0 + u * R, n - 1) * kP4Rows;
      ml[u] = part_ml[i];
      v[u] = part_o[i * C];
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * R < n) mn = fmaxf(mn, ml[u].x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f((m - base) * to2);
    l *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * R < n) {
        const float w = __builtin_amdgcn_exp2f((ml[u].x - base) * to2);
        l += w * ml[u].y;
        add_scaled(acc, w, v[u]);
      }
  }
  sh_o[g][c] = acc;
  if (c == 0) sh_ml[g] = make_float2(m, l);
  __syncthreads();
  if (g > 0) return;
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) mx = fmaxf(mx, sh_ml[i].x);
  const float base = mx == -INFINITY ? 0.f : mx;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float2 p = sh_ml[i];
    const float f = __builtin_amdgcn_exp2f((p.x - base) * to2);
    sum += f * p.y;
    add_scaled(acc, f, sh_o[i][c]);
  }
  store_row<D>(a, b, hk, rt * kP4Rows + row, c, acc, sum);
}

template <int D, int QP, int MB>
void launch_mask(const P4Attn& a, dim3 grid, dim3 block, bool cap, hipStream_t st) {
  if (cap) hipLaunchKernelGGL((pool4_attn_kernel<D, QP, MB, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((pool4_attn_kernel<D, QP, MB, false>), grid, block, 0, st, a);
}

template <int D, int QP>
void launch_attn(const P4Attn& a, hipStream_t st) {
  const dim3 grid(a.splits, a.Hkv * a.row_tiles, a.B), block(64 * kP4Waves);
  const bool cap = a.softcap > 0.f;
  const int mb = !a.mask ? 0 : a.mask_dt == HELM_F32 ? 4 : 2;
  if (mb == 0) launch_mask<D, QP, 0>(a, grid, block, cap, st);
  else if (mb == 2) launch_mask<D, QP, 2>(a, grid, block, cap, st);
  else launch_mask<D, QP, 4>(a, grid, block, cap, st);
  if (a.splits > 1)
    hipLaunchKernelGGL((pool4_join_kernel<D>),
                       dim3((uint32_t)(a.B * a.Hkv * a.row_tiles), std::min(kP4Rows, a.G * a.S)),
                       dim3(256), 0, st, a);
}

struct P4Plan {
  int splits, row_tiles;
  size_t parts, bytes;
};
// Splits (grid.x) from the widest table: a workgroup a CU over the whole launch, two
// where a wave would still have eight blocks or more (64 k x 4 sequences: 53.2 us against
// 55.8 with one; 32 k, one sequence, 14.6 against 14.1, whose joining kernel has half the
// partials); at least one per 128 blocks, so that a long sequence of a ragged batch does
// not trail behind, and no more workgroups than that gains from (their partials are 16
// rows each).  A split has a block a wave, and up to 16 blocks are one split, written
// without a joining kernel: 256 / 512 tokens, 8 KV heads of 128, 5.6 / 7.0 us against
// 8.5 / 8.5 (768: 8.1, 8.3; 1,024: 9.6, 8.4).
P4Plan p4_plan(int B, int Hq, int Hkv, int S, int D, int max_pages, int page_size) {
  P4Plan p{};
  const int64_t blocks = ((int64_t)max_pages * (page_size / kP4Tok) + 1) / 2;
  p.row_tiles = ((int64_t)(Hq / Hkv) * S + kP4Rows - 1) / kP4Rows;
  const int64_t wgs = (int64_t)B * Hkv * p.row_tiles;
  const int64_t target = wgs * blocks >= 512 * kP4Waves * 8 ? 512 : 256;
  int64_t n = std::max<int64_t>(target / wgs, (blocks + 127) / 128);
  n = std::min<int64_t>(n, 16384 / wgs);
  n = blocks <= 16 ? 1 : std::min<int64_t>(n, (blocks + kP4Waves - 1) / kP4Waves);
  p.splits = (int)std::max<int64_t>(1, n);
  p.parts = p.splits > 1 ? (size_t)wgs * p.splits * kP4Rows : 0;
  p.bytes = p.parts * (D + 2) * sizeof(float);
  return p;
}

bool p4_shape_ok(int B, int Hq, int Hkv, int S, int max_pages, int page_size) {
  return B >= 0 && B <= 65535 && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && S >= 1 &&
         max_pages >= 0 && page_size >= kP4Tok && page_size % kP4Tok == 0 &&
         (int64_t)max_pages * page_size <= 0x7fffffff && (int64_t)B * Hq * S <= 0x7fffffff &&
         (int64_t)Hkv * (((int64_t)(Hq / Hkv) * S + kP4Rows - 1) / kP4Rows) <= 65535;
}

}  // namespace
}  // namespace helm

extern "C" size_t helm_pool4_workspace_bytes(int B, int Hq, int Hkv, int q_len, int D,
                                             int max_pages, int page_size) {
  if (!helm::p4_shape_ok(B, Hq, Hkv, q_len, max_pages, page_size) || D < 1) return 0;
  return helm::p4_plan(std::max(B, 1), Hq, Hkv, q_len, D, max_pages, page_size).bytes;
}

extern "C" int helm_pool4_decode_attn(const void* q, void* out, const void* pool, int64_t n_slots,
                                      int page_size, const int32_t* page_table,
                                      int64_t table_stride, int max_pages,
                                      const int32_t* seq_lens, int B, int Hq, int Hkv, int q_len,
                                      int D, float scale, float softcap, const void* mask,
                                      int64_t mask_bstride, int64_t mask_hstride,
                                      int64_t mask_qstride, int mask_len, int mask_dtype,
                                      int causal, int q_dtype,
                                      void* workspace, size_t ws_bytes, void* stream) {
  using namespace helm;
  if (q_dtype != HELM_F16 && q_dtype != HELM_BF16)
    return report_error(HELM_E_UNSUPPORTED, "queries over a 4-bit pool are float16 or bfloat16");
  if (D != 64 && D != 128 && D != 256)
    return report_error(HELM_E_UNSUPPORTED, "a 4-bit pool has head_dim 64, 128 or 256");
  if (!p4_shape_ok(B, Hq, Hkv, q_len, max_pages, page_size) || n_slots < 0 ||
      n_slots > 0x7fffffff || table_stride < 0)
    return report_error(HELM_E_INVALID, "bad 4-bit decode shape");
  if (mask && mask_dtype != HELM_F32 && mask_dtype != HELM_BF16 && mask_dtype != HELM_F16)
    return report_error(HELM_E_INVALID, "unknown mask dtype");
  if (mask && mask_len < 1) return report_error(HELM_E_INVALID, "mask without a column");
  if (!scores_ok(scale, softcap))
    return report_error(HELM_E_INVALID, "scale, softcap or their quotient out of fp32's range");
  if (B == 0) return HELM_OK;
  if (!q || !out || (!pool && n_slots) || (!page_table && max_pages) || !seq_lens)
    return report_error(HELM_E_INVALID, "null pointer argument");
  if ((reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(pool) |
       reinterpret_cast<uint64_t>(out) | reinterpret_cast<uint64_t>(workspace)) & 15)
    return report_error(HELM_E_INVALID,
                        "q, out, the pool and the workspace must be 16-byte aligned");
  const P4Plan pl = p4_plan(B, Hq, Hkv, q_len, D, max_pages, page_size);
  if (pl.bytes && (!workspace || ws_bytes < pl.bytes))
    return report_error(HELM_E_WORKSPACE, "workspace too small: need " + std::to_string(pl.bytes));
  P4Attn a{};
  a.q = q;
  a.out = out;
  a.pool = static_cast<const char*>(pool);
  a.tpp = page_size / kP4Tok;
  a.tpp_log2 = (a.tpp & (a.tpp - 1)) ? -1 : __builtin_ctz(a.tpp);
  a.head_bytes = (int64_t)a.tpp * 17 * D;
  a.slot_bytes = a.head_bytes * Hkv;
  a.n_slots = (int)n_slots;
  a.table = page_table;
  a.table_stride = table_stride;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.S = q_len;
  a.row_tiles = pl.row_tiles;
  a.q16 = q_dtype == HELM_F16;
  a.splits = pl.splits;
  a.causal = causal;
  a.scale = scale;
  a.softcap = softcap;
  a.mask = static_cast<const char*>(mask);
  a.mask_b = mask_bstride;
  a.mask_h = mask_hstride;
  a.mask_q = mask_qstride;
  a.mask_dt = mask_dtype;
  a.mask_len = mask_len;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + pl.parts * D;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (q_dtype == HELM_BF16) {
    if (D == 64) launch_attn<64, 1>(a, st);
    else if (D == 128) launch_attn<128, 1>(a, st);
    else launch_attn<256, 1>(a, st);
  } else {
    if (D == 64) launch_attn<64, 2>(a, st);
    else if (D == 128) launch_attn<128, 2>(a, st);
    else launch_attn<256, 2>(a, st);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return report_error((int)e, std::string("4-bit decode launch: ") + hipGetErrorString(e));
  return HELM_OK;
}
