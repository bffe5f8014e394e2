// Causal attention of packed prompts over a work list (qvl_causal_worklist): 128 rows a workgroup, or 256 (qvl_causal_wide.hip),
// long tiles cut along their keys and joined.
//
// For a row of scores s_j = scale q . k_j over the keys it sees, out = sum_j w_j v_j / sum_j w_j with w_j = 2^(s_j log2 e - m), m
// a maximum carried along: one pass over keys and values, nothing of the size rows x keys in memory. The rows of a tile are
// the heads of a group token by token, so that a key/value tile in LDS serves them all. Bound by the matrix cores and the
// exponentials beside them: 16411 tokens, 32/8 heads of 128, bf16: 2.06 ms here, 1.87 ms (1180 TFLOP/s) in tiles of 256, at
// the power limit (a large matrix product reaches 1404); fp32, on fp32 matrix instructions: 2000 tokens 307 us, 107 TFLOP/s
// (a large product: 154).
#include "qvl_decoder_core.h"

namespace qvl {

void launch_causal_wide(void* stream, int32_t head_dim, const AttnParams& P, const int32_t* items, int64_t n_items, int64_t n_parts);

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void causal_kernel(AttnParams P, const int32_t* items, int n_parts) {
  using R = RowsUnit<T, D>;
  __shared__ __attribute__((aligned(16))) char smem[std::max(R::kLds, 4 * kWriteLds)];
  Item x;
  if (!item_of(P, items, n_parts, kItemRows, R::kBN, x)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (fp32: one sum a score, 7.5e-7 off over 1181 tokens, as the plain form in fp32; a second sum's registers spill: 82 us, not 66)
  Wave<T, D, 1> w;
  w.init(P, x.u, x.u.row0 + wave * 32);
  R::run(P, x.u, w, smem, x.t0, x.t1);
  // A value that is not finite may come from a key that its row does not see: once more, telling them apart.
  if (__builtin_expect(__syncthreads_or(!w.finite()), 0)) {
    w.core.clear();
    w.m = -INFINITY;
    R::run_safe(P, x.u, w, smem, x.t0, x.t1);
  }
  const int r = wave * 32 + (threadIdx.x & 31);
  const int64_t at = (int64_t)max(x.slot, 0) * kItemRows + r;
  write_rows<T, D>(P, x.u, w, smem + wave * kWriteLds, x.u.row0 + r, x.slot >= 0 ? P.part_o + at * D : nullptr, P.part_ml + at, w.lim > x.t0 * R::kBN);
}

// The rows of tiles in parts: gridDim.y workgroups a tile, so that each does no more than a few rounds of rows (one workgroup
// a part, 85 of 256 rows: 28 us of waiting for 408 parts, 53 MB; so 14).
template <typename T, int D>
__global__ __launch_bounds__(256) void causal_combine_kernel(AttnParams P, const int32_t* joins, int n_parts, int tile_rows) {
  const int32_t* it = joins + kItemWords * (int64_t)blockIdx.x;
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4], slot = it[5], parts = it[9];
  const int64_t start = (int64_t)(((uint64_t)(uint32_t)it[7] << 32) | (uint32_t)it[6]);
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || slot < 0 || parts < 1 ||
      len < 0 || start < 0 || start > P.kv_rows - len || slot > n_parts - parts) return;
  const Unit u{nullptr, nullptr, len, 0, q0, n_new * P.group, row0, kvh};
  const int64_t first = (int64_t)slot * tile_rows;
  const int n = tile_rows / gridDim.y, r0 = blockIdx.y * n;
  join_parts<T, D>(P, r0, min(r0 + n, u.rows - row0), parts, [&](int r, int p) { return first + (int64_t)p * tile_rows + r; },
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
  if (num_heads > kItemMaxHeads) return set_error(QVL_ERR_UNSUPPORTED, "%s: num_heads=%d", what, num_heads);
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

int qvl_causal_workspace_size(int32_t head_dim, int32_t tile_rows, int64_t n_parts, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: bytes is NULL");
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "causal_workspace_size: head_dim=%d", head_dim);
  if (n_parts < 0 || n_parts > 0x7fffffffLL || (tile_rows != 128 && tile_rows != 256)) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: items");
  *bytes = (size_t)n_parts * tile_rows * ((size_t)head_dim + 2) * sizeof(float);
  return QVL_OK;
}

int qvl_causal_attention(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                         int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows,
                         int32_t tile_rows, const int32_t* items, int64_t n_items, int64_t n_parts, int64_t n_joins, float scale,
                         void* out, int64_t out_row, int64_t out_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads,
                         int32_t head_dim, void* workspace, size_t workspace_bytes) {
  AttnParams P{};
  QVL_TRY_RC(attn_params("causal_attention", dtype, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, kv_rows, out,
                         out_row, out_head, n_tokens, num_heads, num_kv_heads, head_dim, scale, P));
  if (n_items < 0 || n_items > 0x7fffffffLL || n_parts < 0 || n_parts > n_items || n_joins < 0 || n_joins > n_parts / 2 ||
      (n_parts > 0 && n_joins == 0)) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items");
  if (tile_rows != 128 && tile_rows != 256) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: tile_rows=%d", tile_rows);
  if (tile_rows == 256 && dtype == QVL_DTYPE_F32) return set_error(QVL_ERR_UNSUPPORTED, "causal_attention: tiles of 256 rows are bf16 only");
  if (n_tokens == 0 || n_items == 0) return QVL_OK;
  if (!items) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items is NULL");
  if ((uintptr_t)items % 16) return set_error(QVL_ERR_MISALIGNED, "causal_attention: items");
  size_t need = 0;
  QVL_TRY_RC(qvl_causal_workspace_size(head_dim, tile_rows, n_parts, &need));
  if (workspace_bytes < need || (need && !workspace))
    return set_error(QVL_ERR_WORKSPACE, "causal_attention: workspace %zu < %zu", workspace_bytes, need);
  if (need && (uintptr_t)workspace % 16) return set_error(QVL_ERR_MISALIGNED, "causal_attention: workspace");
  P.part_o = need ? (float*)workspace : nullptr;
  P.part_ml = need ? (f32x2*)((float*)workspace + n_parts * tile_rows * head_dim) : nullptr;
  if (tile_rows == 256) launch_causal_wide(stream, head_dim, P, items, n_items, n_parts);
  else QVL_ATTN_LAUNCH(causal_kernel, dim3((unsigned)n_items), P, items, (int)n_parts);
  QVL_TRY_RC(check_launch("causal_attention"));
  if (n_joins == 0) return QVL_OK;
  QVL_ATTN_LAUNCH(causal_combine_kernel, dim3((unsigned)n_joins, 16u), P, items + kItemWords * n_items, (int)n_parts, tile_rows);
  return check_launch("causal_combine");
}

}  // extern "C"
