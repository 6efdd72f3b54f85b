// Decode attention over a pool of 4-bit pages (helm_pool4_decode_attn): for
// every sequence, KV head and query row softmax(cap(q . K^T scale) + mask) . V
// over the cached tokens, K and V as pool4.h stores them.
//
// Bound by memory: 17 D / 16 bytes a token and KV head (K and V), each read
// once.  The codes become bf16 matrix-core operands in registers (two values an
// instruction, exact), so nothing but the 4-bit page crosses memory.
//
// Work: grid.x = split of the sequence's tiles, grid.y = KV head * row tiles of
// 16 query rows, grid.z = sequence; four waves, wave w takes blocks w, w + 4, ..
// of 32 tokens (two tiles) of the split.  A split's length comes from the
// sequence's own length, read on the device: ceil(tiles / splits), so that one
// launch shape serves any lengths.  Lane (n, h) = (lane % 16, lane / 16):
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
// and the NaN is put into the rows that weigh such a token (block_nan).
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
constexpr int kP4MaxTiles = 2048;    // of a split (their slots sit in LDS)
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
  int min_tiles;                     // a split's least tiles (whole waves' blocks)
  int causal;
  float scale, softcap;
  const char* mask;
  int64_t mask_b, mask_h, mask_q;    // elements
  int mask_dt, mask_len;             // tokens from mask_len on are hidden
  float* part_o;                     // [B][Hq * S][splits][D]
  float* part_ml;                    // [B][Hq * S][splits][2]
};

// Tiles of sequence b, and how its splits share them.
struct P4Split {
  int len, tiles, per, n;            // tokens; tiles; tiles a split; splits in use
};
__device__ __forceinline__ P4Split p4_split(const P4Attn& a, int b) {
  P4Split s;
  const int64_t room = (int64_t)a.max_pages * a.tpp * kP4Tok;
  s.len = (int)min((int64_t)max(0, a.seq_lens[b]), room);
  s.tiles = (s.len + kP4Tok - 1) / kP4Tok;
  s.per = max(a.min_tiles, (s.tiles + a.splits - 1) / a.splits);
  s.per = (s.per + 1) & ~1;          // whole blocks
  s.n = (s.tiles + s.per - 1) / s.per;
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

__device__ __forceinline__ mf_u32x4 p4_decode8(uint32_t w, float s) {
  return mf_u32x4{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
}
// Pair c (dims 2c, 2c + 1 of the lane's chunk) of token j of a tile's four.
template <int D>
__device__ __forceinline__ uint32_t p4_v_pair(const P4Raw<D>& r, int j, int c, float s) {
  constexpr int PB = D / 32;                 // bytes a token's chunk: pairs
  const int byte = j * PB + c;
  const uint32_t w = r.v[byte >> 2];
  switch (byte & 3) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
  }
}

// Any byte of x equal to 255.
__device__ __forceinline__ bool any_ff(uint32_t x) {
  return ((~x - 0x01010101u) & x & 0x80808080u) != 0u;
}

template <int D, int QP, bool kMask, bool kCap>
__global__ __launch_bounds__(64 * kP4Waves) void pool4_attn_kernel(P4Attn a) {
  constexpr int NS = D / 32;                 // 32-dim steps of q . k
  constexpr int NE = D / 16;                 // dims of a V chunk: products of P . V
  using Ops = MfmaOps<bf16_t>;
  __shared__ int slots[kP4MaxTiles];
  __shared__ float sh_o[kP4Waves][kP4Rows][D + 4];
  __shared__ float sh_m[kP4Waves][kP4Rows], sh_l[kP4Waves][kP4Rows];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, n = lane & 15, h = lane >> 4;
  const int split = blockIdx.x;
  const int hk = blockIdx.y % a.Hkv, rt = blockIdx.y / a.Hkv;
  const int b = blockIdx.z;
  const P4Split sp = p4_split(a, b);
  const int rows_all = a.G * a.S;
  const int row0 = rt * kP4Rows, nrows = min(kP4Rows, rows_all - row0);
  if (split >= max(1, sp.n)) return;
  const int t_lo = split * sp.per, t_n = min(sp.per, sp.tiles - t_lo);   // (0 tiles: n = 0)

  for (int i = tid; i < t_n; i += 64 * kP4Waves) {
    const int t = t_lo + i;
    const int page = a.tpp_log2 >= 0 ? t >> a.tpp_log2 : t / a.tpp;
    const int s = a.table[(int64_t)b * a.table_stride + page];
    slots[i] = s >= 0 && s < a.n_slots ? s : -1;
  }

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
  MaskRow mrow{nullptr, HELM_F32};
  if constexpr (kMask) {
    const int64_t e = b * a.mask_b + head * a.mask_h + rc.s * a.mask_q;
    mrow = MaskRow{a.mask, a.mask_dt} + e;
  }
  // with a mask the logits stay in natural units (finfo.min would leave fp32's
  // range in base 2), the weight's exponent is scaled instead
  const float unit = kMask ? 1.f : kP4Log2E, to2 = kMask ? kP4Log2E : 1.f;
  const float slack = kMask ? kP4Slack / kP4Log2E : kP4Slack;
  const float qscale = a.scale * unit;
  const float inv_cap = kCap ? 1.f / a.softcap : 0.f, cap = a.softcap * unit;
  // row n's last visible token
  const int last_vis = a.causal ? min(sp.len - 1, sp.len - a.S + rc.s) : sp.len - 1;
  // the block's tokens all lie at or before every row's last visible one
  const int all_vis = a.causal ? sp.len - a.S + row0 / a.G : sp.len - 1;

  float m = -INFINITY, l = 0.f;
  mf_f32x4 o[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) o[e] = mf_f32x4{0.f, 0.f, 0.f, 0.f};

  __syncthreads();
  const char* head_base = a.pool + hk * a.head_bytes;
  auto load = [&](int blk, P4Raw<D> (&r)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = 2 * blk + s;
      const int slot = __builtin_amdgcn_readfirstlane(i < t_n ? slots[i] : -1);
      const int t = t_lo + i;
      const int in_page = a.tpp_log2 >= 0 ? t & (a.tpp - 1) : t % a.tpp;
      r[s] = p4_load<D>(head_base + max(slot, 0) * a.slot_bytes +
                            (int64_t)in_page * P4<D>::kBytes,
                        slot >= 0, n, h);
    }
  };
  auto step = [&](int blk, P4Raw<D> (&r)[2]) {
    const int tok0 = (t_lo + 2 * blk) * kP4Tok;
    // a slot that the pool does not have hides its tile
    const bool gone0 = __builtin_amdgcn_readfirstlane(slots[2 * blk]) < 0;
    const bool gone1 =
        2 * blk + 1 >= t_n || __builtin_amdgcn_readfirstlane(slots[2 * blk + 1]) < 0;
    float x[8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      mf_f32x4 sc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const uint32_t e = D == 256 && i >= NS / 2 ? r[s].ke >> 8 : r[s].ke & 255u;
        const mf_u32x4 kop = p4_decode8(r[s].k[i], p4_scale(e));
#pragma unroll
        for (int p = 0; p < QP; ++p) sc = Ops::mma(kop, qop[p][i], sc);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * s + j] = sc[j];
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
        const float mk = mrow[min(tok(j), a.mask_len - 1)];
        x[j] = mk == -INFINITY || tok(j) >= a.mask_len ? -INFINITY : x[j] + mk;
      }
    }
    const bool limits = gone0 || gone1 || tok0 + 31 > all_vis;      // uniform
    if (limits) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (tok(j) > last_vis || (j < 4 ? gone0 : gone1)) x[j] = -INFINITY;
      // exponents of tokens past the sequence are whatever the page held
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (tok(j) >= sp.len) r[j >> 2].ve &= ~(255u << (8 * (j & 3)));
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
    const bool nan = __builtin_amdgcn_ballot_w64(any_ff(r[0].ve) || any_ff(r[1].ve)) != 0;
    uint32_t ff = 0;                         // bit j: token j's group stands for NaN
    if (__builtin_expect(nan, 0)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t& ve = r[j >> 2].ve;
        if (((ve >> (8 * (j & 3))) & 255u) == 255u) {
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
      o[2 * c] = Ops::mma(even, lo, o[2 * c]);
      o[2 * c + 1] = Ops::mma(odd, hi, o[2 * c + 1]);
      o[2 * c + 1] = Ops::mma(odd, lo, o[2 * c + 1]);
    }
    if (__builtin_expect(nan, 0)) {
      // ones at the NaN tokens (a whole chunk lies in one group): a row that
      // weighs any gets NaN in every dim of the chunk
      mf_u32x4 one;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        one[j] = (((ff >> (2 * j)) & 1u) ? 0x3F80u : 0u) |
                 (((ff >> (2 * j + 1)) & 1u) ? 0x3F800000u : 0u);
      const mf_f32x4 hit = Ops::mma(one, hi, mf_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        if (!(hit[r4] == 0.f))
#pragma unroll
          for (int e = 0; e < NE; ++e) o[e][r4] = __builtin_nanf("");
    }
  };
  const int nblk = (t_n + 1) / 2;
  for (int blk = wave; blk < nblk; blk += kP4Waves) {
    P4Raw<D> r[2];
    load(blk, r);
    step(blk, r);
  }

  // the split's rows: the waves' states joined in LDS
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (h == 0) {
    sh_m[wave][n] = m;
    sh_l[wave][n] = l;
  }
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4)
#pragma unroll
    for (int e = 0; e < NE; ++e) sh_o[wave][n][(4 * h + r4) * NE + e] = o[e][r4];
  __syncthreads();
  for (int i = tid; i < nrows * D; i += 64 * kP4Waves) {
    const int row = i / D, d = i % D;
    float mx = sh_m[0][row];
#pragma unroll
    for (int w = 1; w < kP4Waves; ++w) mx = fmaxf(mx, sh_m[w][row]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kP4Waves; ++w) {
      const float f = __builtin_amdgcn_exp2f((sh_m[w][row] - base) * to2);
      sum += f * sh_l[w][row];
      acc += f * sh_o[w][row][d];
    }
    const RowCoord c = row_coord(row0 + row, a.G);
    const int64_t r = (int64_t)(b * a.Hq + hk * a.G + c.g) * a.S + c.s;
    if (sp.n <= 1) {
      char* dst = reinterpret_cast<char*>(a.out) + 2 * (r * D + d);
      const float v = sum == 0.f ? 0.f : acc / sum;
      if (a.q16) store_elem<f16_t>(dst, v);
      else store_elem<bf16_t>(dst, v);
    } else {
      const int64_t p = r * a.splits + split;
      a.part_o[p * D + d] = acc;
      if (d == 0) {
        a.part_ml[2 * p] = mx;
        a.part_ml[2 * p + 1] = sum;
      }
    }
  }
}

// Row blockIdx.x of the output from its splits' partials; a thread a dim.
template <int D>
__global__ __launch_bounds__(D) void pool4_join_kernel(P4Attn a) {
  const int64_t r = blockIdx.x;
  const int b = (int)(r / ((int64_t)a.Hq * a.S));
  const P4Split sp = p4_split(a, b);
  if (sp.n <= 1) return;                     // written by its only split
  const float* ml = a.part_ml + 2 * r * a.splits;
  const float* po = a.part_o + r * a.splits * D + threadIdx.x;
  const float to2 = a.mask ? kP4Log2E : 1.f;   // (the units of the partials' maxima)
  float mx = -INFINITY;
  for (int s = 0; s < sp.n; ++s) mx = fmaxf(mx, ml[2 * s]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f, acc = 0.f;
  for (int s = 0; s < sp.n; ++s) {
    const float f = __builtin_amdgcn_exp2f((ml[2 * s] - base) * to2);
    sum += f * ml[2 * s + 1];
    acc += f * po[(int64_t)s * D];
  }
  char* dst = reinterpret_cast<char*>(a.out) + 2 * (r * D + threadIdx.x);
  const float v = sum == 0.f ? 0.f : acc / sum;
  if (a.q16) store_elem<f16_t>(dst, v);
  else store_elem<bf16_t>(dst, v);
}

template <int D, int QP>
void launch_attn(const P4Attn& a, hipStream_t st) {
  const dim3 grid(a.splits, a.Hkv * a.row_tiles, a.B), block(64 * kP4Waves);
  const bool cap = a.softcap > 0.f;
  if (a.mask && cap) hipLaunchKernelGGL((pool4_attn_kernel<D, QP, true, true>), grid, block, 0, st, a);
  else if (a.mask) hipLaunchKernelGGL((pool4_attn_kernel<D, QP, true, false>), grid, block, 0, st, a);
  else if (cap) hipLaunchKernelGGL((pool4_attn_kernel<D, QP, false, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((pool4_attn_kernel<D, QP, false, false>), grid, block, 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((pool4_join_kernel<D>), dim3((uint32_t)(a.B * a.Hq * a.S)), dim3(D), 0, st, a);
}

struct P4Plan {
  int splits, min_tiles, row_tiles;
  size_t bytes;
};
// Splits: enough workgroups for every CU several times over, none with less than
// one block a wave; at most kP4MaxTiles tiles each.
P4Plan p4_plan(int B, int Hq, int Hkv, int S, int D, int max_pages, int page_size) {
  P4Plan p{};
  const int64_t tiles = (int64_t)max_pages * (page_size / kP4Tok);
  p.row_tiles = ((int64_t)(Hq / Hkv) * S + kP4Rows - 1) / kP4Rows;
  p.min_tiles = 2 * kP4Waves;
  const int64_t wgs = (int64_t)B * Hkv * p.row_tiles;
  int64_t n = std::max<int64_t>(1, (1024 + wgs - 1) / wgs);
  n = std::min<int64_t>(n, (tiles + p.min_tiles - 1) / p.min_tiles);
  n = std::max<int64_t>(n, (tiles + kP4MaxTiles - 1) / kP4MaxTiles);
  p.splits = (int)std::max<int64_t>(1, n);
  p.bytes = p.splits > 1 ? (size_t)B * Hq * S * p.splits * (D + 2) * sizeof(float) : 0;
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
      n_slots > 0x7fffffff || table_stride < max_pages)
    return report_error(HELM_E_INVALID, "bad 4-bit decode shape");
  if (mask && mask_dtype != HELM_F32 && mask_dtype != HELM_BF16 && mask_dtype != HELM_F16)
    return report_error(HELM_E_INVALID, "unknown mask dtype");
  if (mask && mask_len < 1) return report_error(HELM_E_INVALID, "mask without a column");
  if (B == 0) return HELM_OK;
  if (!q || !out || (!pool && n_slots) || (!page_table && max_pages) || !seq_lens)
    return report_error(HELM_E_INVALID, "null pointer argument");
  if ((reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(pool)) & 15)
    return report_error(HELM_E_INVALID, "q and the pool must be 16-byte aligned");
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
  a.min_tiles = pl.min_tiles;
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
  a.part_ml = a.part_o + (pl.splits > 1 ? (int64_t)B * Hq * q_len * pl.splits * D : 0);
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
