// xk_paged_attention: checks, the plan's host part and the choice of instance
// (the kernels are in paged_attention.h).
#include <algorithm>

#include "paged_attention.h"

namespace xk {
namespace paged {
namespace {

constexpr int64_t kMostPositions = int64_t{1} << 28;  // a sequence's, by its table row
constexpr int64_t kMostPitch = int64_t{1} << 27;      // bytes from one position to the next
constexpr int64_t kMostPage = int64_t{1} << 35;       // and from one page to the next
constexpr int64_t kMostBlocks = int64_t{1} << 24;     // a launch holds 2^32 threads in a dimension,
                                                      // of which 128 blocks may be idle

constexpr float kLog2e = 1.44269504088896f;

struct Plan {
  int tiles;  // row tiles of a wave
  int64_t groups, shares, bytes;
  int64_t most;  // shares that there can be
};

// The shares of a head and row group: at most two blocks a compute unit in all
// (most kernels take one), none without a least share.
void cut(Plan& x, int64_t M, int64_t Hkv) {
  x.groups = cdiv(M, 16 * x.tiles);
  x.shares = std::min(std::max<int64_t>(1, 2 * num_cus() / (Hkv * x.groups)), x.most);
}

// False where the sizes are beyond what a launch holds.
bool plan_of(int64_t B, int64_t T, int64_t G, int64_t Hkv, int64_t D, int64_t positions,
             xk_dtype dtype, Plan& x) {
  const int64_t M = T * G;
  if (M >= kMostPositions) return false;
  // (two row tiles of fp32 heads of 256 do not fit the registers)
  x.tiles = M > 16 && (D <= 128 || dtype != XK_F32) ? 2 : 1;
  x.most = cdiv(B * std::max<int64_t>(1, cdiv(positions, 16)), kWaves);
  cut(x, M, Hkv);
  const int64_t lines = Hkv * x.groups;
  const int64_t rows = 2 * x.shares * Hkv * M;
  if (x.shares * lines > kMostBlocks - 128 || B * Hkv >= kMostBlocks || rows >= (int64_t{1} << 40))
    return false;
  auto up = [](int64_t n) { return cdiv(n, 256) * 256; };
  // One share holds every sequence whole.
  x.bytes = x.shares > 1 ? up(B * 8) + up(rows * 8) + up(rows * D * 4) : 0;
  return true;
}

// n / by = n * magic >> shift for n < 2^28: by * magic is above 2^shift by e < by
// <= 2^(shift - 28), so n * magic / 2^shift is above n / by by less than 1 / by.
void magic_of(int64_t by, uint32_t& magic, int& shift) {
  shift = 28;
  while ((int64_t{1} << (shift - 28)) < by) ++shift;
  magic = static_cast<uint32_t>(cdiv(int64_t{1} << shift, by));
}

int check_sizes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_pages,
                int64_t page_size) {
  if (B < 0 || T <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || D > 256 || D % 8 ||
      max_pages < 0 || page_size <= 0 || page_size > kMostPositions)
    return XK_ERR_INVALID;
  if (B > (1 << 24) || T > (1 << 20) || Hq > (1 << 16) ||
      (max_pages > 0 && page_size > kMostPositions / max_pages))
    return XK_ERR_INVALID;
  return XK_OK;
}

}  // namespace
}  // namespace paged
}  // namespace xk

using namespace xk;

extern "C" int64_t xk_paged_attention_workspace_bytes(int64_t B, int64_t T, int64_t Hq,
                                                      int64_t Hkv, int64_t head_dim,
                                                      int64_t max_pages, int64_t page_size,
                                                      xk_dtype dtype) {
  paged::Plan x;
  if (paged::check_sizes(B, T, Hq, Hkv, head_dim, max_pages, page_size) != XK_OK || B == 0 ||
      !paged::plan_of(B, T, Hq / Hkv, Hkv, head_dim, max_pages * page_size, dtype, x))
    return 0;
  return x.bytes;
}

extern "C" int xk_paged_attention(
    const void* q, int64_t stride_q_seq, int64_t stride_q_tok, int64_t stride_q_head,
    const void* k_cache, int64_t stride_kc_page, int64_t stride_kc_slot, int64_t stride_kc_head,
    const void* v_cache, int64_t stride_vc_page, int64_t stride_vc_slot, int64_t stride_vc_head,
    xk_dtype cache_dtype, int64_t num_pages, int64_t page_size, const int32_t* block_table,
    int64_t stride_table_row, int64_t max_pages, const int32_t* seq_lens, float scale,
    int64_t window, const float* k_scale, const float* v_scale, void* out, int64_t stride_o_seq,
    int64_t stride_o_tok, int64_t stride_o_head, float* lse, int64_t B, int64_t T, int64_t Hq,
    int64_t Hkv, int64_t head_dim, xk_dtype dtype, void* workspace, size_t workspace_bytes,
    void* stream) {
  using namespace paged;
  const int st = check_sizes(B, T, Hq, Hkv, head_dim, max_pages, page_size);
  if (st != XK_OK) return st;
  if (num_pages < 0 || num_pages > INT32_MAX || window < 0 ||
      !std::isfinite(scale * kLog2e))
    return XK_ERR_INVALID;
  const bool eight = cache_dtype == XK_F8E4M3;
  if (!is_float_dtype(dtype) || (eight ? dtype == XK_F32 : cache_dtype != dtype))
    return XK_ERR_UNSUPPORTED;
  if (!eight && (k_scale || v_scale)) return XK_ERR_INVALID;
  if (B == 0) return XK_OK;
  if (!q || !out || !seq_lens || (max_pages && !block_table) ||
      (num_pages && (!k_cache || !v_cache)))
    return XK_ERR_INVALID;
  // Vectors of 16 bytes (8 of an 8-bit cache) have to be aligned.
  const int eb = elem_bytes(dtype), cb = eight ? 1 : eb, n = 16 / eb;
  const int cv = n * cb;
  if (!aligned(q, 16) || stride_q_seq % n || stride_q_tok % n || stride_q_head % n ||
      !aligned(k_cache, cv) || !aligned(v_cache, cv) || stride_kc_page % n ||
      stride_kc_slot % n || stride_kc_head % n || stride_vc_page % n || stride_vc_slot % n ||
      stride_vc_head % n || !aligned(out, 4 * eb) || stride_o_seq % 4 || stride_o_tok % 4 ||
      stride_o_head % 4)
    return XK_ERR_UNSUPPORTED;
  if (stride_kc_slot < 0 || stride_vc_slot < 0 || stride_kc_slot >= kMostPitch / cb ||
      stride_vc_slot >= kMostPitch / cb || stride_kc_page < 0 || stride_vc_page < 0 ||
      stride_kc_page >= kMostPage / cb || stride_vc_page >= kMostPage / cb ||
      std::max(stride_kc_slot, stride_vc_slot) * cb * page_size > UINT32_MAX)
    return XK_ERR_INVALID;
  const int64_t positions = num_pages ? max_pages * page_size : 0;
  Plan x;
  if (!plan_of(B, T, Hq / Hkv, Hkv, head_dim, max_pages * page_size, dtype, x))
    return XK_ERR_INVALID;
  // Two blocks with a row tile each read all twice, but are sooner through a few
  // tiles: where a block has at most 384 positions by the table's width.  4 and 16
  // sequences of 1900 on average, 2600 at the most (170 and 680 a block), 4 tokens,
  // 32 / 4 heads, us with one tile and two: 64 bf16 13.8, 16.1; 21.4, 20.3; e4m3
  // 14.3, 15.9; 21.5, 19.7; 128 bf16 18.1, 20.5; 34.2, 29.9; e4m3 16.4, 20.6; 26.8,
  // 29.5; 256 bf16 29.0, 37.8; 61.4, 59.5; e4m3 23.8, 31.5; 43.4, 46.7.  The width
  // is all that the host knows of the lengths: a table much wider than they are
  // gets two.  More than 32 rows get two as well, which is right where there is much
  // to read (32 sequences of 2500, 64 rows, bf16 heads of 256: 105.9, 91.7) and not
  // where there is little (8, 48 rows: 64 15.6, 18.7; 128 21.2, 24.8; 256 36.6, 48.6).
  const int64_t M = T * (Hq / Hkv);
  const int64_t seen = window && window < positions - T ? window + T : positions;
  if (x.tiles == 2 && M <= 32 && B * seen * Hkv <= int64_t{384} * num_cus()) {
    x.tiles = 1;
    cut(x, M, Hkv);  // (fewer shares: the workspace suffices)
  }
  if (x.bytes && (!workspace || workspace_bytes < static_cast<size_t>(x.bytes) ||
                  !aligned(workspace, 256)))
    return XK_ERR_WORKSPACE;
  Params p{};
  p.q = q;
  p.q_seq = stride_q_seq;
  p.q_tok = stride_q_tok;
  p.q_head = stride_q_head;
  p.kc = static_cast<const char*>(k_cache);
  p.k_page = static_cast<uint32_t>(stride_kc_page * cb / 8);
  p.k_slot = static_cast<uint32_t>(stride_kc_slot * cb);
  p.k_head = stride_kc_head * cb;
  p.vc = static_cast<const char*>(v_cache);
  p.v_page = static_cast<uint32_t>(stride_vc_page * cb / 8);
  p.v_slot = static_cast<uint32_t>(stride_vc_slot * cb);
  p.v_head = stride_vc_head * cb;
  p.num_pages = static_cast<int>(num_pages);
  p.page_size = static_cast<int>(page_size);
  magic_of(page_size, p.page_magic, p.page_shift);
  p.table = block_table;
  p.table_row = stride_table_row;
  p.max_pages = static_cast<int>(max_pages);
  p.lens = seq_lens;
  p.most_len = static_cast<int>(positions);
  p.scale2 = scale * kLog2e;
  p.window = static_cast<int>(std::min<int64_t>(window, kMostPositions + (1 << 20)));
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.out = out;
  p.o_seq = stride_o_seq;
  p.o_tok = stride_o_tok;
  p.o_head = stride_o_head;
  p.lse = lse;
  p.B = static_cast<int>(B);
  p.T = static_cast<int>(T);
  p.G = static_cast<int>(Hq / Hkv);
  p.Hkv = static_cast<int>(Hkv);
  p.D = static_cast<int>(head_dim);
  magic_of(Hq / Hkv, p.g_magic, p.g_shift);
  p.M = static_cast<int>(T * (Hq / Hkv));
  p.groups = static_cast<int>(x.groups);
  p.shares = static_cast<int>(x.shares);
  if (x.bytes) {
    char* ws = static_cast<char*>(workspace);
    const int64_t rows = 2 * x.shares * Hkv * p.M;
    p.meta = reinterpret_cast<int2*>(ws);
    ws += cdiv(B * 8, 256) * 256;
    p.ml = reinterpret_cast<float2*>(ws);
    ws += cdiv(rows * 8, 256) * 256;
    p.acc = reinterpret_cast<float*>(ws);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: return run_f32(p, x.tiles, s);
    case XK_BF16: return eight ? run_bf16_f8(p, x.tiles, s) : run_bf16(p, x.tiles, s);
    default: return eight ? run_f16_f8(p, x.tiles, s) : run_f16(p, x.tiles, s);
  }
}
