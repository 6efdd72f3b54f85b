// Rows of K and V into the pages of a 4-bit pool, and the values they stand for
// back out (helm_pool4_write, helm_pool4_read).  Layout and rounding: pool4.h.
//
// Both are bound by memory: a bf16 row of D dims is 2 D bytes on one side and
// 17 D / 32 on the other.  A thread owns eight dims of K or V of one head (16 bytes of a
// 16-bit row; four lanes are a group, whose largest magnitude they share by two quad
// moves) and takes them of two consecutive rows: where its place in a row is worked out
// once for both.  The workgroups of neighbouring rows run on one XCD, so that the 16
// rows of a tile, which share cache lines, meet in one L2 instead of leaving it in
// parts.  16,384 rows of 8 heads of 128, bf16, write / read: a thread a row and place
// 31 / 28.5 us (half of it divisions), four rows 26 / 22, on one XCD 18.8 / 18.9, two
// rows 18.1 / 17.5 (8: 21 / 24); 85 MB each, 14.7 us at 5.78 TB/s.
// The conversions of gfx950 encode and decode two values an instruction, exactly and
// with ties to the even code (checked over every code and exponent).
#include "pool4.h"

#include <algorithm>
#include <string>

#include "attn_kernel.h"
#include "helm_amd.h"

namespace helm {

int report_error(int code, const std::string& msg);

namespace {

constexpr int kThreads4 = 256;
constexpr int kRowsLaunch = 1 << 24;   // rows of a launch (its threads stay below 2^32)

constexpr int kRowsPer = 2;         // consecutive rows of a thread

struct P4Rows {
  char* pool;
  int64_t slot_bytes;        // of one slot (page), all heads
  int64_t head_bytes;        // of one head of a page
  int64_t n_rows;            // slots * page tokens
  int page, page_log2;       // its log2 or -1
  const int64_t* slots;
  int n_tok;
  int items;                 // places of a row: K's, then V's, D / 8 a head each
  int abreast;               // rows that a workgroup's threads hold side by side
  char* k;
  char* v;
  int64_t k_tok, k_head, v_tok, v_head;   // elements
};

// Row `slot` of the pool (inside it): its tile of head 0, and its token in the tile.
struct P4Place {
  char* tile;
  int t;
};
template <int D>
__device__ __forceinline__ P4Place p4_place(const P4Rows& a, int64_t slot) {
  int64_t s;
  int r;
  if (a.page_log2 >= 0) {
    s = slot >> a.page_log2;
    r = (int)slot & (a.page - 1);
  } else {
    s = slot / a.page;
    r = (int)(slot - s * a.page);
  }
  return {a.pool + s * a.slot_bytes + (int64_t)(r / kP4Tok) * P4<D>::kBytes, r % kP4Tok};
}

// Byte of the codes of dims 8c .. 8c + 7 of token t (V at D = 64: the first of its two
// chunks; see p4_v_store)
template <int D> __device__ __forceinline__ int p4_k_byte(int t, int c) {
  return t * (D / 2) + 4 * c;
}
template <int D> __device__ __forceinline__ int p4_v_byte(int t, int c) {
  constexpr int VB = P4<D>::kChunk;
  const int byte = 4 * c;                         // of the row's D / 2
  return P4<D>::kVc + ((byte / VB) * kP4Tok + t) * VB + byte % VB;
}

template <typename T> __device__ __forceinline__ void load8(const char* p, int64_t elem, float* x) {
  if constexpr (std::is_same<T, float>::value) {
    const float4 a = reinterpret_cast<const float4*>(p + 4 * elem)[0];
    const float4 b = reinterpret_cast<const float4*>(p + 4 * elem)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(p + 2 * elem);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t h = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
      if constexpr (std::is_same<T, bf16_t>::value) x[i] = __uint_as_float((uint32_t)h << 16);
      else x[i] = (float)__builtin_bit_cast(_Float16, h);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(char* p, int64_t elem, const float* x) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(p + 4 * elem)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p + 4 * elem)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) store_elem<T>(reinterpret_cast<char*>(&h[i]), x[i]);
    uint4 w;
    w.x = h[0] | (uint32_t)h[1] << 16;
    w.y = h[2] | (uint32_t)h[3] << 16;
    w.z = h[4] | (uint32_t)h[5] << 16;
    w.w = h[6] | (uint32_t)h[7] << 16;
    *reinterpret_cast<uint4*>(p + 2 * elem) = w;
  }
}

// A thread's place in a row (eight dims, chunk c of head h of K or V) and its rows
// n .. n + kRowsPer - 1; place < 0: none.  All four lanes of a group share all but c.
template <int D> struct P4Item {
  int64_t n;
  int h, c;
  bool some, is_v;
  __device__ __forceinline__ explicit P4Item(const P4Rows& a) {
    const int tid = threadIdx.x;
    const int sub = a.abreast > 1 ? tid / a.items : 0;
    int i = a.abreast > 1 ? tid - sub * a.items : (int)blockIdx.y * kThreads4 + tid;
    some = sub < a.abreast && i < a.items;
    // neighbouring rows stay on one XCD (workgroups go round the eight of them)
    const int64_t wg = (int64_t)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    n = (wg * a.abreast + sub) * kRowsPer;
    is_v = i >= a.items / 2;
    if (is_v) i -= a.items / 2;
    h = i / (D / 8);
    c = i % (D / 8);
  }
};

// Eight dims of V codes go to one word, or two chunks' half words (D = 64).
template <int D> __device__ __forceinline__ void p4_v_store(char* tile, int t, int c, uint32_t w) {
  char* dst = tile + p4_v_byte<D>(t, c);
  if constexpr (D == 64) {
    *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
    *reinterpret_cast<uint16_t*>(dst + 2 * kP4Tok) = (uint16_t)(w >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = w;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads4) void pool4_write_kernel(P4Rows a) {
  const P4Item<D> it(a);
  if (!it.some || it.n >= a.n_tok) return;                // (whole groups of four lanes)
  const int m = min(kRowsPer, (int)(a.n_tok - it.n));
  const char* src = it.is_v ? a.v : a.k;
  const int64_t tok = it.is_v ? a.v_tok : a.k_tok;
  const int64_t at = (it.is_v ? a.v_head : a.k_head) * it.h + 8 * it.c;
  int64_t slot[kRowsPer];
  float x[kRowsPer][8];
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    const int64_t n = it.n + min(i, m - 1);
    slot[i] = i < m ? a.slots[n] : -1;
    load8<T>(src, n * tok + at, x[i]);
  }
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    uint32_t top = 0;                      // largest magnitude's bits (NaN above infinity)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
    const uint32_t e = p4_exponent(top);
    uint32_t w = 0;
    if (e != 255u) {
      const float s = p4_scale(e);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[i][0], x[i][1], s, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[i][2], x[i][3], s, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[i][4], x[i][5], s, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[i][6], x[i][7], s, 3);
    }
    if (slot[i] < 0 || slot[i] >= a.n_rows) continue;
    const P4Place p = p4_place<D>(a, slot[i]);
    char* tile = p.tile + it.h * a.head_bytes;
    if (it.is_v) {
      p4_v_store<D>(tile, p.t, it.c, w);
      if ((it.c & 3) == 0) tile[P4<D>::kVe + (it.c >> 2) * kP4Tok + p.t] = (char)e;
    } else {
      *reinterpret_cast<uint32_t*>(tile + p4_k_byte<D>(p.t, it.c)) = w;
      if ((it.c & 3) == 0) tile[P4<D>::kKe + p.t * P4<D>::kGroups + (it.c >> 2)] = (char)e;
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads4) void pool4_read_kernel(P4Rows a) {
  const P4Item<D> it(a);
  if (!it.some || it.n >= a.n_tok) return;
  const int m = min(kRowsPer, (int)(a.n_tok - it.n));
  uint32_t w[kRowsPer], e[kRowsPer];
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    const int64_t slot = a.slots[it.n + min(i, m - 1)];
    w[i] = e[i] = 0u;                      // (a row outside the pool: zeros)
    if (slot < 0 || slot >= a.n_rows) continue;
    const P4Place p = p4_place<D>(a, slot);
    const char* tile = p.tile + it.h * a.head_bytes;
    if (it.is_v) {
      const char* src = tile + p4_v_byte<D>(p.t, it.c);
      if constexpr (D == 64)
        w[i] = *reinterpret_cast<const uint16_t*>(src) |
               (uint32_t)*reinterpret_cast<const uint16_t*>(src + 2 * kP4Tok) << 16;
      else
        w[i] = *reinterpret_cast<const uint32_t*>(src);
      e[i] = (uint8_t)tile[P4<D>::kVe + (it.c >> 2) * kP4Tok + p.t];
    } else {
      w[i] = *reinterpret_cast<const uint32_t*>(tile + p4_k_byte<D>(p.t, it.c));
      e[i] = (uint8_t)tile[P4<D>::kKe + p.t * P4<D>::kGroups + (it.c >> 2)];
    }
  }
  char* dst = it.is_v ? a.v : a.k;
  const int64_t tok = it.is_v ? a.v_tok : a.k_tok;
  const int64_t at = (it.is_v ? a.v_head : a.k_head) * it.h + 8 * it.c;
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    if (i >= m) break;
    const float s = p4_scale(e[i]);        // (e = 255: NaN, and so is every product)
    const auto a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 0);
    const auto a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 1);
    const auto a2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 2);
    const auto a3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 3);
    const float x[8] = {a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
    store8<T>(dst, (it.n + i) * tok + at, x);
  }
}

template <typename T, int D>
void launch_rows(bool write, const P4Rows& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.abreast * kRowsPer;
  const dim3 grid((uint32_t)((a.n_tok + 8 * rows - 1) / (8 * rows) * 8),
                  (uint32_t)((a.items + kThreads4 - 1) / kThreads4));
  if (write) hipLaunchKernelGGL((pool4_write_kernel<T, D>), grid, dim3(kThreads4), 0, st, a);
  else hipLaunchKernelGGL((pool4_read_kernel<T, D>), grid, dim3(kThreads4), 0, st, a);
}
template <typename T>
void launch_rows_d(bool write, int D, const P4Rows& a, hipStream_t st) {
  if (D == 64) launch_rows<T, 64>(write, a, st);
  else if (D == 128) launch_rows<T, 128>(write, a, st);
  else launch_rows<T, 256>(write, a, st);
}

int rows_call(bool write, const char* name, void* pool, int64_t n_slots, int page_size, int Hkv,
              int D, const int64_t* slots, int n_tok, void* k, int64_t k_tok, int64_t k_head,
              void* v, int64_t v_tok, int64_t v_head, int dtype, void* stream) {
  if (dtype != HELM_F16 && dtype != HELM_BF16 && dtype != HELM_F32)
    return report_error(HELM_E_INVALID, "unknown dtype");
  if (D != 64 && D != 128 && D != 256)
    return report_error(HELM_E_UNSUPPORTED, "a 4-bit pool has head_dim 64, 128 or 256");
  if (n_slots < 0 || page_size < kP4Tok || page_size % kP4Tok || Hkv < 1 || Hkv > 65535 ||
      n_tok < 0)
    return report_error(HELM_E_INVALID,
                        "bad 4-bit pool shape (page_size a multiple of 16, 1 to 65535 heads)");
  if (n_tok == 0) return HELM_OK;
  const int eb = dtype == HELM_F32 ? 4 : 2;
  if (!slots || !k || !v || (!pool && n_slots))
    return report_error(HELM_E_INVALID, "null pointer argument");
  const uint64_t bits = reinterpret_cast<uint64_t>(pool) | reinterpret_cast<uint64_t>(k) |
                        reinterpret_cast<uint64_t>(v) | (uint64_t)(k_tok * eb) |
                        (uint64_t)(k_head * eb) | (uint64_t)(v_tok * eb) | (uint64_t)(v_head * eb);
  if (bits & 15) return report_error(HELM_E_INVALID, "pool, k and v rows must be 16-byte aligned");
  P4Rows a{};
  a.pool = static_cast<char*>(pool);
  a.head_bytes = (int64_t)(page_size / kP4Tok) * 17 * D;
  a.slot_bytes = a.head_bytes * Hkv;
  a.n_rows = n_slots * page_size;
  a.page = page_size;
  a.page_log2 = (page_size & (page_size - 1)) ? -1 : __builtin_ctz(page_size);
  a.slots = slots;
  a.n_tok = n_tok;
  a.items = Hkv * (D / 4);
  a.abreast = std::max(1, kThreads4 / a.items);
  a.k = static_cast<char*>(k);
  a.v = static_cast<char*>(v);
  a.k_tok = k_tok;
  a.k_head = k_head;
  a.v_tok = v_tok;
  a.v_head = v_head;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int n0 = 0; n0 < n_tok; n0 += kRowsLaunch) {
    P4Rows part = a;
    part.n_tok = std::min(kRowsLaunch, n_tok - n0);
    part.slots += n0;
    part.k += n0 * k_tok * eb;
    part.v += n0 * v_tok * eb;
    if (dtype == HELM_F16) launch_rows_d<f16_t>(write, D, part, st);
    else if (dtype == HELM_BF16) launch_rows_d<bf16_t>(write, D, part, st);
    else launch_rows_d<float>(write, D, part, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return report_error((int)e, std::string(name) + " launch: " + hipGetErrorString(e));
    if (n_tok - n0 <= kRowsLaunch) break;
  }
  return HELM_OK;
}

}  // namespace
}  // namespace helm

extern "C" int helm_pool4_write(void* pool, int64_t n_slots, int page_size, int Hkv, int D,
                                const int64_t* slot_map, int n_tok, const void* k,
                                int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                                int64_t v_tok_stride, int64_t v_head_stride, int dtype,
                                void* stream) {
  return helm::rows_call(true, "4-bit pool write", pool, n_slots, page_size, Hkv, D, slot_map,
                         n_tok, const_cast<void*>(k), k_tok_stride, k_head_stride,
                         const_cast<void*>(v), v_tok_stride, v_head_stride, dtype, stream);
}

extern "C" int helm_pool4_read(const void* pool, int64_t n_slots, int page_size, int Hkv, int D,
                               const int64_t* slot_map, int n_tok, void* k, int64_t k_tok_stride,
                               int64_t k_head_stride, void* v, int64_t v_tok_stride,
                               int64_t v_head_stride, int dtype, void* stream) {
  return helm::rows_call(false, "4-bit pool read", const_cast<void*>(pool), n_slots, page_size,
                         Hkv, D, slot_map, n_tok, k, k_tok_stride, k_head_stride, v, v_tok_stride,
                         v_head_stride, dtype, stream);
}
