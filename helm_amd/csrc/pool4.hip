// Rows of K and V into the pages of a 4-bit pool, and the values they stand for
// back out (helm_pool4_write, helm_pool4_read).  Layout and rounding: pool4.h.
//
// Both are bound by memory: a bf16 row of D dims is 2 D bytes on one side and
// 17 D / 32 on the other.  A lane owns eight dims of one row (one 16-byte load of
// 16-bit values), four lanes a group, whose largest magnitude they share by two
// quad moves; the matrix-core conversions of gfx950 encode and decode two
// values an instruction (exact, ties to even, as checked over every code and
// exponent).
#include "pool4.h"

#include <algorithm>
#include <string>

#include "attn_kernel.h"
#include "helm_amd.h"

namespace helm {

int report_error(int code, const std::string& msg);

namespace {

constexpr int kThreads4 = 256;

struct P4Rows {
  char* pool;
  int64_t slot_bytes;        // of one slot (page), all heads
  int64_t head_bytes;        // of one head of a page
  int64_t n_rows;            // slots * page tokens
  int page;
  const int64_t* slots;
  int n_tok;
  int Hkv;
  char* k;
  char* v;
  int64_t k_tok, k_head, v_tok, v_head;   // elements
};

// Row `slot` of the pool, head h: its tile and its token in it.
struct P4Place {
  char* tile;
  int t;
};
template <int D>
__device__ __forceinline__ P4Place p4_place(const P4Rows& a, int64_t slot, int h) {
  int64_t s;
  int r;
  if (a.n_rows <= 0x7fffffff) {     // (uniform; a 64-bit division is ~100 instructions)
    s = (uint32_t)slot / (uint32_t)a.page;
    r = (int)((uint32_t)slot % (uint32_t)a.page);
  } else {
    s = slot / a.page;
    r = (int)(slot % a.page);
  }
  return {a.pool + s * a.slot_bytes + h * a.head_bytes + (r / kP4Tok) * P4<D>::kBytes,
          r % kP4Tok};
}

// Byte of the codes of dims 8c .. 8c + 7 of token t (V: D = 64 two chunks of two
// bytes, 32 apart; see p4_v_store)
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

template <typename T> __device__ __forceinline__ void store8(char* p, int64_t elem, const float* x) {
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

// Item i of the launch: eight dims (chunk c) of K or V of head h of row n.
template <int D> struct P4Item {
  int n, h, c;
  bool is_v;
  __device__ __forceinline__ P4Item(int64_t i, int Hkv) {
    c = (int)(i % (D / 8));
    const int64_t j = i / (D / 8);
    is_v = j & 1;
    const uint32_t r = (uint32_t)(j >> 1);       // n * Hkv + h < 2^31 (checked on the host)
    h = (int)(r % (uint32_t)Hkv);
    n = (int)(r / (uint32_t)Hkv);
  }
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads4) void pool4_write_kernel(P4Rows a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads4 + threadIdx.x;
  if (i >= (int64_t)a.n_tok * a.Hkv * (D / 4)) return;      // (whole groups of four lanes)
  const P4Item<D> it(i, a.Hkv);
  const int64_t slot = a.slots[it.n];
  if (slot < 0 || slot >= a.n_rows) return;                 // (one row: whole groups again)
  float x[8];
  if (it.is_v) load8<T>(a.v, it.n * a.v_tok + it.h * a.v_head + 8 * it.c, x);
  else load8<T>(a.k, it.n * a.k_tok + it.h * a.k_head + 8 * it.c, x);
  uint32_t top = 0;                        // largest magnitude's bits (NaN above infinity)
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
  const uint32_t e = p4_exponent(top);
  uint32_t w = 0;
  if (e != 255u) {
    const float s = p4_scale(e);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  }
  const P4Place p = p4_place<D>(a, slot, it.h);
  if (it.is_v) {
    if constexpr (D == 64) {               // two chunks of four dims
      char* dst = p.tile + p4_v_byte<D>(p.t, it.c);
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(dst + 2 * kP4Tok) = (uint16_t)(w >> 16);
    } else {
      *reinterpret_cast<uint32_t*>(p.tile + p4_v_byte<D>(p.t, it.c)) = w;
    }
    if ((it.c & 3) == 0) p.tile[P4<D>::kVe + (it.c >> 2) * kP4Tok + p.t] = (char)e;
  } else {
    *reinterpret_cast<uint32_t*>(p.tile + p4_k_byte<D>(p.t, it.c)) = w;
    if ((it.c & 3) == 0) p.tile[P4<D>::kKe + p.t * P4<D>::kGroups + (it.c >> 2)] = (char)e;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads4) void pool4_read_kernel(P4Rows a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads4 + threadIdx.x;
  if (i >= (int64_t)a.n_tok * a.Hkv * (D / 4)) return;
  const P4Item<D> it(i, a.Hkv);
  const int64_t slot = a.slots[it.n];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.n_rows) {
    const P4Place p = p4_place<D>(a, slot, it.h);
    uint32_t w, e;
    if (it.is_v) {
      const char* src = p.tile + p4_v_byte<D>(p.t, it.c);
      if constexpr (D == 64)
        w = *reinterpret_cast<const uint16_t*>(src) |
            (uint32_t)*reinterpret_cast<const uint16_t*>(src + 2 * kP4Tok) << 16;
      else
        w = *reinterpret_cast<const uint32_t*>(src);
      e = (uint8_t)p.tile[P4<D>::kVe + (it.c >> 2) * kP4Tok + p.t];
    } else {
      w = *reinterpret_cast<const uint32_t*>(p.tile + p4_k_byte<D>(p.t, it.c));
      e = (uint8_t)p.tile[P4<D>::kKe + p.t * P4<D>::kGroups + (it.c >> 2)];
    }
    const float s = p4_scale(e);           // (e = 255: NaN, and so is every product)
    const auto a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
    const auto a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const auto a2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
    const auto a3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    x[0] = a0[0]; x[1] = a0[1]; x[2] = a1[0]; x[3] = a1[1];
    x[4] = a2[0]; x[5] = a2[1]; x[6] = a3[0]; x[7] = a3[1];
  }
  if (it.is_v) store8<T>(a.v, it.n * a.v_tok + it.h * a.v_head + 8 * it.c, x);
  else store8<T>(a.k, it.n * a.k_tok + it.h * a.k_head + 8 * it.c, x);
}

template <typename T, int D>
void launch_rows(bool write, const P4Rows& a, hipStream_t st) {
  const int64_t items = (int64_t)a.n_tok * a.Hkv * (D / 4);
  const dim3 grid((uint32_t)((items + kThreads4 - 1) / kThreads4));
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
  if (n_slots < 0 || page_size < kP4Tok || page_size % kP4Tok || Hkv < 1 || n_tok < 0 ||
      (int64_t)n_tok * Hkv > 0x7fffffff)
    return report_error(HELM_E_INVALID,
                        "bad 4-bit pool shape (page_size a multiple of 16, rows * heads < 2^31)");
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
  a.slots = slots;
  a.n_tok = n_tok;
  a.Hkv = Hkv;
  a.k = static_cast<char*>(k);
  a.v = static_cast<char*>(v);
  a.k_tok = k_tok;
  a.k_head = k_head;
  a.v_tok = v_tok;
  a.v_head = v_head;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HELM_F16) launch_rows_d<f16_t>(write, D, a, st);
  else if (dtype == HELM_BF16) launch_rows_d<bf16_t>(write, D, a, st);
  else launch_rows_d<float>(write, D, a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return report_error((int)e, std::string(name) + " launch: " + hipGetErrorString(e));
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
