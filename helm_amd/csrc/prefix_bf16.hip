// bfloat16 instantiations of the shared-prefix decode kernels (prefix.h), and their C-ABI entry.
#include "prefix.h"

#include <algorithm>
#include <cfloat>
#include <string>

namespace helm {
int report_error(int code, const std::string& msg);
hipError_t launch_prefix_bf16(const PfParams& p, int D, hipStream_t st) {
  return launch_prefix_type<bf16_t>(p, D, st);
}

namespace {

struct PfPlan {
  int wgs, own_tiles, own_rows;
  int64_t group_slots, own_slots, bytes;
};
// Workgroups of a KV head: as many as the device holds at once.
PfPlan pf_plan(int R, int Hq, int Hkv, int S, int D, int n_groups) {
  PfPlan p{};
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  p.wgs = std::max(1, 256 * (D == 256 ? PfShape<256>::kPerCu : PfShape<128>::kPerCu) / Hkv);
  p.own_tiles = (int)((rows + kPfTile - 1) / kPfTile);
  p.own_rows = (int)std::min<int64_t>(rows, kPfTile);
  p.group_slots = n_groups ? n_groups + R * rows / kPfRows + kPfWaves * p.wgs : 0;
  p.own_slots = (int64_t)R * p.own_tiles + p.wgs;
  auto room = [](int64_t n) { return (n + 15) / 16 * 16; };
  p.bytes = room(R * (int64_t)sizeof(PfSeq)) + room(Hkv * p.group_slots * kPfRows * 2 * 4) +
            room(Hkv * p.own_slots * p.own_rows * 2 * 4) +
            4 * Hkv * (p.group_slots * kPfRows + p.own_slots * p.own_rows) * D;
  return p;
}

bool pf_shape_ok(int R, int Hq, int Hkv, int S, int max_pages, int page, int n_groups) {
  if (R < 0 || R > HELM_PREFIX_MAX_SEQS || n_groups < 0 || n_groups > HELM_PREFIX_MAX_GROUPS ||
      Hkv < 1 || Hq < 1 || Hq % Hkv || S < 1 || max_pages < 0 || page < kBlockTok ||
      page % kBlockTok || (int64_t)max_pages * page > 0x7ffff000 ||
      (int64_t)R * Hq * S > 0x7fffffff / kPfJoinThreads || Hkv > 65536)
    return false;
  // the line of a KV head's walks stays within 2^30 steps
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  const int64_t walks = R * ((rows + kPfTile - 1) / kPfTile) + n_groups + R * rows / kPfTile;
  const int64_t steps = ((int64_t)max_pages * page + kPfStep - 1) / kPfStep + 1 + kPfFixed;
  return walks * steps <= 0x3fffffff;
}

}  // namespace
}  // namespace helm

extern "C" size_t helm_prefix_workspace_bytes(int R, int Hq, int Hkv, int q_len, int D,
                                              int n_groups) {
  if (!helm::pf_shape_ok(R, Hq, Hkv, q_len, 0, 16, n_groups) || D < 1) return 0;
  return (size_t)helm::pf_plan(R, Hq, Hkv, q_len, D, n_groups).bytes;
}

extern "C" int helm_prefix_decode_attn(const void* q, void* out, const void* k_pool,
                                       const void* v_pool, int64_t n_slots, int64_t slot_stride,
                                       int64_t head_stride, int page_size,
                                       const int32_t* page_table, int64_t table_stride,
                                       int max_pages, const int32_t* seq_lens,
                                       const int32_t* group_starts, const int32_t* shared_pages,
                                       int n_groups, int R, int Hq, int Hkv, int q_len, int D,
                                       float scale, float softcap, int window, int dtype,
                                       void* workspace, size_t ws_bytes, void* stream) {
  using namespace helm;
  if (dtype != HELM_F16 && dtype != HELM_BF16)
    return report_error(HELM_E_UNSUPPORTED, "shared-prefix decode takes float16 or bfloat16");
  if (D != 64 && D != 128 && D != 256)
    return report_error(HELM_E_UNSUPPORTED, "shared-prefix decode takes head_dim 64, 128 or 256");
  if (!pf_shape_ok(R, Hq, Hkv, q_len, max_pages, page_size, n_groups) || n_slots < 0 ||
      n_slots > 0x7fffffff || table_stride < 0)
    return report_error(HELM_E_INVALID,
                        "bad shared-prefix decode shape (at most " +
                            std::to_string(HELM_PREFIX_MAX_SEQS) + " sequences, " +
                            std::to_string(HELM_PREFIX_MAX_GROUPS) +
                            " groups, 2^30 steps of 32 tokens a KV head)");
  if (!scores_ok(scale, softcap))
    return report_error(HELM_E_INVALID, "scale, softcap or their quotient out of fp32's range");
  if (R == 0) return HELM_OK;
  if (!q || !out || (n_slots && (!k_pool || !v_pool)) || (!page_table && max_pages) || !seq_lens ||
      (n_groups && (!group_starts || !shared_pages)))
    return report_error(HELM_E_INVALID, "null pointer argument");
  if (slot_stride < 0 || head_stride < 0 || slot_stride % 8 || head_stride % 8 ||
      ((reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(out) |
        reinterpret_cast<uint64_t>(k_pool) | reinterpret_cast<uint64_t>(v_pool) |
        reinterpret_cast<uint64_t>(workspace)) & 15))
    return report_error(HELM_E_INVALID,
                        "q, out, the pools' rows and the workspace must be 16-byte aligned");
  const PfPlan pl = pf_plan(R, Hq, Hkv, q_len, D, n_groups);
  if (!workspace || ws_bytes < (size_t)pl.bytes)
    return report_error(HELM_E_WORKSPACE, "workspace too small: need " + std::to_string(pl.bytes));
  PfParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k_pool);
  p.v = static_cast<const char*>(v_pool);
  p.out = static_cast<char*>(out);
  p.slot = 2 * slot_stride;
  p.head = 2 * head_stride;
  p.n_slots = (int)n_slots;
  p.table = page_table;
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.page = page_size;
  p.bpp = page_size / kBlockTok;
  p.lens = seq_lens;
  p.starts = group_starts;
  p.shared = shared_pages;
  p.n_groups = n_groups;
  p.R = R;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.S = q_len;
  p.wgs = pl.wgs;
  p.own_tiles = pl.own_tiles;
  p.own_rows = pl.own_rows;
  p.group_slots = (int)pl.group_slots;
  p.own_slots = (int)pl.own_slots;
  // the kernel takes a row's maximum before it scales
  p.q_sign = scale < 0.f ? 0x80008000u : 0u;
  p.scale = std::max(scale < 0.f ? -scale : scale, FLT_MIN);
  p.softcap = softcap;
  p.window = window;
  char* ws = static_cast<char*>(workspace);
  auto take = [&](int64_t n) {
    char* at = ws;
    ws += (n + 15) / 16 * 16;
    return at;
  };
  p.seqs = reinterpret_cast<PfSeq*>(take(R * (int64_t)sizeof(PfSeq)));
  p.group_ml = reinterpret_cast<float*>(take(Hkv * pl.group_slots * kPfRows * 2 * 4));
  p.own_ml = reinterpret_cast<float*>(take(Hkv * pl.own_slots * pl.own_rows * 2 * 4));
  p.group_o = reinterpret_cast<float*>(take(4 * Hkv * pl.group_slots * kPfRows * D));
  p.own_o = reinterpret_cast<float*>(ws);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      dtype == HELM_BF16 ? launch_prefix_bf16(p, D, st) : launch_prefix_f16(p, D, st);
  if (e != hipSuccess)
    return report_error((int)e,
                        std::string("shared-prefix decode launch: ") + hipGetErrorString(e));
  return HELM_OK;
}
