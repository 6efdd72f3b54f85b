// bfloat16 instantiations of the prompt kernel (prompt.h), and its C-ABI entry.
#include "prompt.h"

#include <algorithm>
#include <cfloat>
#include <string>

namespace helm {
int report_error(int code, const std::string& msg);
hipError_t launch_prompt_bf16(const PromptParams& p, int D, hipStream_t st) {
  return launch_prompt_type<bf16_t>(p, D, st);
}
}  // namespace helm

extern "C" int helm_prompt_attn(const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                const void* k, int64_t k_tok_stride, int64_t k_head_stride,
                                const void* v, int64_t v_tok_stride, int64_t v_head_stride,
                                void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                const int32_t* cu_seqlens, int B, int N, int Hq, int Hkv, int D,
                                float scale, float softcap, int window, int zero_rest, int dtype,
                                void* stream) {
  using namespace helm;
  if (dtype != HELM_F16 && dtype != HELM_BF16)
    return report_error(HELM_E_UNSUPPORTED, "prompt attention takes float16 or bfloat16");
  if (D != 64 && D != 128 && D != 256)
    return report_error(HELM_E_UNSUPPORTED, "prompt attention takes head_dim 64, 128 or 256");
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv)
    return report_error(HELM_E_INVALID, "bad prompt attention shape");
  if (!scores_ok(scale, softcap))
    return report_error(HELM_E_INVALID, "scale, softcap or their quotient out of fp32's range");
  if (N == 0) return HELM_OK;
  if (!q || !k || !v || !out || !cu_seqlens)
    return report_error(HELM_E_INVALID, "null pointer argument");
  const int64_t strides[8] = {q_tok_stride, q_head_stride, k_tok_stride,   k_head_stride,
                              v_tok_stride, v_head_stride, out_tok_stride, out_head_stride};
  for (int64_t s : strides)
    if (s % 8) return report_error(HELM_E_INVALID, "rows must be 16-byte aligned");
  if ((reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(k) |
       reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(out)) & 15)
    return report_error(HELM_E_INVALID, "rows must be 16-byte aligned");
  // a block's 16 rows are addressed by 32-bit offsets
  if (k_tok_stride < 0 || v_tok_stride < 0 || k_tok_stride > (1 << 25) || v_tok_stride > (1 << 25))
    return report_error(HELM_E_INVALID, "token strides of k and v must be 0 to 2^25 elements");
  PromptParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.out = static_cast<char*>(out);
  p.q_tok = 2 * q_tok_stride;
  p.q_head = 2 * q_head_stride;
  p.k_tok = 2 * k_tok_stride;
  p.k_head = 2 * k_head_stride;
  p.v_tok = 2 * v_tok_stride;
  p.v_head = 2 * v_head_stride;
  p.o_tok = 2 * out_tok_stride;
  p.o_head = 2 * out_head_stride;
  p.cu = cu_seqlens;
  p.B = B;
  p.N = N;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  if (((int64_t)N / 128 + 1 + B) * Hq > 0x7fffffff / 512)     // (tiles * heads * threads)
    return report_error(HELM_E_INVALID, "too many rows and heads for one launch");
  // the kernel takes the row's maximum before it scales
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  p.scale = std::max(scale < 0.f ? -scale : scale, FLT_MIN);
  p.softcap = softcap;
  p.window = window;
  p.zero_rest = zero_rest;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      dtype == HELM_BF16 ? launch_prompt_bf16(p, D, st) : launch_prompt_f16(p, D, st);
  if (e != hipSuccess)
    return report_error((int)e, std::string("prompt attention launch: ") + hipGetErrorString(e));
  return HELM_OK;
}
