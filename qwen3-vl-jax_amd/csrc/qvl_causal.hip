// Causal attention of packed prompts over a work list (qvl_causal_worklist): 128 rows a workgroup, or 256 (qvl_causal_wide.hip),
// long tiles split along their keys and joined.
#include "qvl_decoder_core.h"

namespace qvl {

void launch_causal_wide(void* stream, int32_t head_dim, const AttnParams& P, const int32_t* items, int64_t n_items, int64_t n_whole);

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void causal_kernel(AttnParams P, const int32_t* items, int n_whole) {
  using R = RowsUnit<T, D>;
  __shared__ __attribute__((aligned(16))) char smem[std::max(R::kLds, 4 * kWriteLds)];
  const int32_t* it = items + 8 * (int64_t)blockIdx.x;
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4] & kItemHeadMask;
  const int part = (it[4] >> kItemPartShift) & 0xff, parts = (it[4] >> kItemPartsShift) & 0xff, slot = it[5];
  const int64_t start = (int64_t)(((uint64_t)(uint32_t)it[7] << 32) | (uint32_t)it[6]);
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || len < 0 || start < 0 ||
      start > P.kv_rows - len || row0 >= n_new * P.group || (parts && (part >= parts || slot < 0 || slot >= (int)gridDim.x - n_whole))) return;
  const Unit u{P.k.p + start * P.k.row + kvh * P.k.head, P.v.p + start * P.v.row + kvh * P.v.head, len, len - n_new + 1, q0,
               n_new * P.group, row0, kvh};
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int last = min(row0 + kItemRows, u.rows) - 1;
  const int k_hi = max(min(u.lim0 + (int)((uint32_t)last / (uint32_t)P.group), len), 0);
  const int n_t = (k_hi + R::kBN - 1) / R::kBN;
  const int t0 = parts ? (int)((int64_t)n_t * part / parts) : 0, t1 = parts ? (int)((int64_t)n_t * (part + 1) / parts) : n_t;
  Wave<T, D> w;
  w.init(P, u, row0 + wave * 32);
  R::run(P, u, w, smem, t0, t1);
  // A value that is not finite may come from a key that its row does not see: once more, telling them apart.
  if (__builtin_expect(__syncthreads_or(!w.finite()), 0)) {
    w.core.clear();
    w.m = -INFINITY;
    R::run_safe(P, u, w, smem, t0, t1);
  }
  const int r = wave * 32 + (threadIdx.x & 31);
  const int64_t at = (int64_t)slot * kItemRows + r;
  write_rows<T, D>(P, u, w, smem + wave * kWriteLds, row0 + r, parts ? P.part_o + at * D : nullptr, P.part_ml + at, w.lim > t0 * R::kBN);
}

// The rows of split tiles: the workgroup of a part joins its share of the tile's 128 rows.
template <typename T, int D>
__global__ __launch_bounds__(256) void causal_combine_kernel(AttnParams P, const int32_t* items, int n_whole, int tile_rows) {
  const int32_t* it = items + 8 * ((int64_t)n_whole + blockIdx.x);
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4] & kItemHeadMask;
  const int part = (it[4] >> kItemPartShift) & 0xff, parts = (it[4] >> kItemPartsShift) & 0xff, slot = it[5];
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || part >= parts ||
      part > slot || slot - part + parts > (int)gridDim.x) return;
  const Unit u{nullptr, nullptr, len, 0, q0, n_new * P.group, row0, kvh};
  const int64_t first = (int64_t)(slot - part) * tile_rows;
  join_parts<T, D>(P, tile_rows * part / parts, min(tile_rows * (part + 1) / parts, u.rows - row0), parts,
                   [&](int r, int p) { return first + (int64_t)p * tile_rows + r; },
                   [&](int r) { return out_row<T, D>(P, u, row0 + r); });
}

constexpr float kLog2e = 1.4426950408889634f;

// Checks shared by the two entries, and the views.
int attn_params(const char* what, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                       int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows,
                       const void* out, int64_t out_row, int64_t out_head, int64_t n_tokens, int32_t num_heads,
                       int32_t num_kv_heads, int32_t head_dim, float scale, AttnParams& P) {
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", what, head_dim);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(QVL_ERR_INVALID_ARG, "%s: %d heads over %d key/value heads", what, num_heads, num_kv_heads);
  if (num_heads > kItemHeadMask) return set_error(QVL_ERR_UNSUPPORTED, "%s: num_heads=%d", what, num_heads);
  if (n_tokens < 0 || kv_rows < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_tokens > kItemMaxLen || n_tokens * (num_heads / num_kv_heads) > kItemMaxLen || kv_rows > (int64_t)1 << 56)
    return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(QVL_ERR_INVALID_ARG, "%s: scale %g", what, (double)scale);
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  struct { const char* name; const void* p; int64_t row, head; AttnView* to; } views[] = {
      {"q", q, q_row, q_head, &P.q}, {"k", k, k_row, k_head, &P.k}, {"v", v, v_row, v_head, &P.v}, {"out", out, out_row, out_head, &P.out}};
  for (auto& w : views) {
    if (!w.p && n_tokens > 0 && (kv_rows > 0 || w.to == &P.q || w.to == &P.out))
      return set_error(QVL_ERR_INVALID_ARG, "%s: %s is NULL", what, w.name);
    if (w.row < 0 || w.head < 0 || w.row > 0x7fffffffLL || w.head > 0x7fffffffLL)
      return set_error(QVL_ERR_INVALID_ARG, "%s: strides of %s", what, w.name);
    if ((w.to == &P.k || w.to == &P.v) && w.row * size > (int64_t)1 << 26)   // a tile's 64 rows are addressed in 32 bits
      return set_error(QVL_ERR_UNSUPPORTED, "%s: rows of %s are more than 64 MiB apart", what, w.name);
    if ((uintptr_t)w.p % 16 || w.row * size % 16 || w.head * size % 16)
      return set_error(QVL_ERR_MISALIGNED, "%s: %s and its strides must be multiples of 16 bytes", what, w.name);
    *w.to = AttnView{(const char*)w.p, w.row * size, w.head * size};
  }
  P.kv_rows = kv_rows;
  P.n_tokens = n_tokens;
  P.hkv = num_kv_heads;
  P.group = num_heads / num_kv_heads;
  P.scale = scale * kLog2e;
  return QVL_OK;
}

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_causal_workspace_size(int32_t head_dim, int32_t tile_rows, int64_t n_items, int64_t n_whole, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: bytes is NULL");
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "causal_workspace_size: head_dim=%d", head_dim);
  if (n_whole < 0 || n_items < n_whole || (tile_rows != 128 && tile_rows != 256)) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: items");
  *bytes = (size_t)(n_items - n_whole) * tile_rows * ((size_t)head_dim + 2) * sizeof(float);
  return QVL_OK;
}

int qvl_causal_attention(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                         int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows,
                         int32_t tile_rows, const int32_t* items, int64_t n_items, int64_t n_whole, float scale, void* out, int64_t out_row,
                         int64_t out_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* workspace, size_t workspace_bytes) {
  AttnParams P{};
  QVL_TRY_RC(attn_params("causal_attention", dtype, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, kv_rows, out,
                         out_row, out_head, n_tokens, num_heads, num_kv_heads, head_dim, scale, P));
  if (n_whole < 0 || n_items < n_whole || n_items > 0x7fffffffLL) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items");
  if (tile_rows != 128 && tile_rows != 256) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: tile_rows=%d", tile_rows);
  if (tile_rows == 256 && dtype == QVL_DTYPE_F32) return set_error(QVL_ERR_UNSUPPORTED, "causal_attention: tiles of 256 rows are bf16 only");
  if (n_tokens == 0 || n_items == 0) return QVL_OK;
  if (!items) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items is NULL");
  if ((uintptr_t)items % 16) return set_error(QVL_ERR_MISALIGNED, "causal_attention: items");
  size_t need = 0;
  QVL_TRY_RC(qvl_causal_workspace_size(head_dim, tile_rows, n_items, n_whole, &need));
  if (workspace_bytes < need || (need && !workspace))
    return set_error(QVL_ERR_WORKSPACE, "causal_attention: workspace %zu < %zu", workspace_bytes, need);
  if (need && (uintptr_t)workspace % 16) return set_error(QVL_ERR_MISALIGNED, "causal_attention: workspace");
  P.part_o = need ? (float*)workspace : nullptr;
  P.part_ml = need ? (f32x2*)((float*)workspace + (n_items - n_whole) * tile_rows * head_dim) : nullptr;
  if (tile_rows == 256) launch_causal_wide(stream, head_dim, P, items, n_items, n_whole);
  else QVL_ATTN_LAUNCH(causal_kernel, dim3((unsigned)n_items), P, items, (int)n_whole);
  QVL_TRY_RC(check_launch("causal_attention"));
  if (!need) return QVL_OK;
  QVL_ATTN_LAUNCH(causal_combine_kernel, dim3((unsigned)(n_items - n_whole)), P, items, (int)n_whole, tile_rows);
  return check_launch("causal_combine");
}

}  // extern "C"
