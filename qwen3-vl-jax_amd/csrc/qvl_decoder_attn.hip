// Causal, decode and shared-prefix attention of a text decoder: out = softmax(scale q k^T) v over the keys a token sees,
// grouped heads, bf16 or fp32, head_dim 64 or 128.
//
// A row is one (token, query head); the rows of one key/value head that see the same keys are handled together. One
// pass over the keys holds the running maximum m, the sum l of exp(s - m) and the unnormalised output.
#include <math.h>
#include <type_traits>

#include "qvl_decoder_items.h"
#include "qvl_kernels.h"

namespace qvl {

struct AttnView {
  const char* p;
  int64_t row, head;   // strides in bytes
};

struct AttnParams {
  AttnView q, k, v, out;
  int64_t kv_rows, n_tokens;
  int hkv, group;          // key/value heads, query heads of each
  float scale;             // of the scores, times log2(e): the softmax runs on powers of two
  // causal: items; decode: the sequences' state
  const int32_t* items;
  const int32_t* cu_q;
  const int64_t* k_start;
  const int32_t* k_len;
  const int32_t* cu_groups;
  const int64_t* prefix_start;
  const int32_t* prefix_len;
  int n_seqs, n_groups;
};

template <typename T> __device__ __forceinline__ float load_one(const char* p, int i) {
  return (float)reinterpret_cast<const T*>(p)[i];
}

// One row over up to two runs of cache rows (start, keys), by one wave: 64 keys at a time, a lane's score each; then a
// lane holds D / 64 of the output's dims. `q` is the row in LDS, fp32.
template <typename T, int D>
__device__ __forceinline__ void attend_row(const AttnParams& P, const float* q, int kvh, const int64_t (&start)[2],
                                           const int64_t (&keys)[2], char* out) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f, o[E] = {};
  for (int run = 0; run < 2; ++run) {
    const char* kb = P.k.p + start[run] * P.k.row + kvh * P.k.head;
    const char* vb = P.v.p + start[run] * P.v.row + kvh * P.v.head;
    for (int64_t j0 = 0; j0 < keys[run]; j0 += 64) {
      float s = -INFINITY;
      if (j0 + lane < keys[run]) {
        const char* kr = kb + (j0 + lane) * P.k.row;
        s = 0.f;
        for (int d = 0; d < D; ++d) s = __builtin_fmaf(q[d], load_one<T>(kr, d), s);
        s *= P.scale;
      }
      float mx = s;
      for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
      const float mn = fmaxf(m, mx), shift = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m - shift), p = __builtin_amdgcn_exp2f(s - shift);
      m = mn;
      l *= a;
      for (int e = 0; e < E; ++e) o[e] *= a;
      const int n = (int)min((int64_t)64, keys[run] - j0);
      for (int j = 0; j < n; ++j) {
        const float pj = __shfl(p, j);
        l += pj;
        for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(pj, load_one<T>(vb + (j0 + j) * P.v.row, lane * E + e), o[e]);
      }
    }
  }
  const bool none = keys[0] + keys[1] <= 0;
  for (int e = 0; e < E; ++e) reinterpret_cast<T*>(out)[lane * E + e] = (T)(none ? 0.f : o[e] / l);
}

template <typename T, int D>
__device__ __forceinline__ const float* row_to_lds(const AttnParams& P, float (*lds)[D], int64_t token, int head) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* q = P.q.p + token * P.q.row + head * P.q.head;
  __builtin_amdgcn_wave_barrier();
  for (int d = lane; d < D; d += 64) lds[wave][d] = load_one<T>(q, d);
  __builtin_amdgcn_wave_barrier();
  return lds[wave];
}

template <typename T, int D>
__global__ __launch_bounds__(256) void causal_kernel(AttnParams P) {
  __shared__ float lds[4][D];
  const int32_t* it = P.items + 8 * (int64_t)blockIdx.x;
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4] & kItemHeadMask;
  const int64_t start = (int64_t)(((uint64_t)(uint32_t)it[7] << 32) | (uint32_t)it[6]);
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || len < 0 || start < 0 ||
      start + len > P.kv_rows) return;
  for (int r = row0 + (threadIdx.x >> 6); r < min(row0 + kItemRows, n_new * P.group); r += 4) {
    const int t = r / P.group, head = kvh * P.group + r % P.group;
    const int64_t starts[2] = {start, 0}, keys[2] = {max(len - n_new + t + 1, 0), 0};
    const float* q = row_to_lds<T, D>(P, lds, q0 + t, head);
    attend_row<T, D>(P, q, kvh, starts, keys, const_cast<char*>(P.out.p) + (q0 + t) * P.out.row + head * P.out.head);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void decode_kernel(AttnParams P) {
  __shared__ float lds[4][D];
  const int seq = blockIdx.x, kvh = blockIdx.y;
  const int64_t q0 = P.cu_q ? P.cu_q[seq] : seq, q1 = P.cu_q ? P.cu_q[seq + 1] : seq + 1;
  if (q0 < 0 || q1 > P.n_tokens) return;
  int64_t starts[2] = {0, P.k_start[seq]};
  int64_t len = P.k_len[seq], prefix = 0;
  for (int g = 0; g < P.n_groups; ++g)
    if (P.cu_groups[g] <= seq && seq < P.cu_groups[g + 1]) {
      starts[0] = P.prefix_start[g];
      prefix = P.prefix_len[g];
    }
  const bool bad = len < 0 || starts[1] < 0 || starts[1] > P.kv_rows - len || prefix < 0 || starts[0] < 0 ||
                   starts[0] > P.kv_rows - prefix;
  const int64_t rows = (q1 - q0) * P.group;
  for (int64_t r = threadIdx.x >> 6; r < rows; r += 4) {
    const int64_t t = r / P.group;
    const int head = kvh * P.group + (int)(r % P.group);
    char* out = const_cast<char*>(P.out.p) + (q0 + t) * P.out.row + head * P.out.head;
    if (bad) {
      for (int d = threadIdx.x & 63; d < D; d += 64) reinterpret_cast<T*>(out)[d] = (T)NAN;
      continue;
    }
    const int64_t keys[2] = {prefix, max(len - (q1 - q0) + t + 1, (int64_t)0)};
    const float* q = row_to_lds<T, D>(P, lds, q0 + t, head);
    attend_row<T, D>(P, q, kvh, starts, keys, out);
  }
}

constexpr float kLog2e = 1.4426950408889634f;

// Checks shared by the two entries, and the views.
static int attn_params(const char* what, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
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

#define QVL_ATTN_LAUNCH(KERNEL, GRID)                                                                              \
  do {                                                                                                             \
    const dim3 grid = GRID;                                                                                        \
    if (dtype == QVL_DTYPE_BF16) {                                                                                 \
      if (head_dim == 128) hipLaunchKernelGGL((KERNEL<bf16, 128>), grid, dim3(256), 0, (hipStream_t)stream, P);    \
      else hipLaunchKernelGGL((KERNEL<bf16, 64>), grid, dim3(256), 0, (hipStream_t)stream, P);                     \
    } else {                                                                                                       \
      if (head_dim == 128) hipLaunchKernelGGL((KERNEL<float, 128>), grid, dim3(256), 0, (hipStream_t)stream, P);   \
      else hipLaunchKernelGGL((KERNEL<float, 64>), grid, dim3(256), 0, (hipStream_t)stream, P);                    \
    }                                                                                                              \
  } while (0)

extern "C" {

int qvl_causal_workspace_size(int32_t head_dim, int64_t n_items, int64_t n_whole, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: bytes is NULL");
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "causal_workspace_size: head_dim=%d", head_dim);
  if (n_whole < 0 || n_items < n_whole) return set_error(QVL_ERR_INVALID_ARG, "causal_workspace_size: items");
  *bytes = 0;
  return QVL_OK;
}

int qvl_causal_attention(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                         int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows,
                         const int32_t* items, int64_t n_items, int64_t n_whole, float scale, void* out, int64_t out_row,
                         int64_t out_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* workspace, size_t workspace_bytes) {
  AttnParams P{};
  QVL_TRY_RC(attn_params("causal_attention", dtype, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, kv_rows, out,
                         out_row, out_head, n_tokens, num_heads, num_kv_heads, head_dim, scale, P));
  if (n_whole < 0 || n_items < n_whole || n_items > 0x7fffffffLL) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items");
  if (n_tokens == 0 || n_items == 0) return QVL_OK;
  if (!items) return set_error(QVL_ERR_INVALID_ARG, "causal_attention: items is NULL");
  if ((uintptr_t)items % 16) return set_error(QVL_ERR_MISALIGNED, "causal_attention: items");
  P.items = items;
  QVL_ATTN_LAUNCH(causal_kernel, dim3((unsigned)n_items));
  return check_launch("causal_attention");
}

int qvl_decode_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t max_len, int64_t n_groups, int64_t max_prefix,
                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "decode_workspace_size: bytes is NULL");
  *bytes = 0;
  return QVL_OK;
}

int qvl_decode_attention(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                         int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows,
                         const int32_t* cu_q, int64_t n_seqs, const int64_t* k_start, const int32_t* k_len, int64_t max_len,
                         const int32_t* cu_groups, int64_t n_groups, const int64_t* prefix_start,
                         const int32_t* prefix_len, int64_t max_prefix, float scale, void* out, int64_t out_row,
                         int64_t out_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* workspace, size_t workspace_bytes) {
  AttnParams P{};
  QVL_TRY_RC(attn_params("decode_attention", dtype, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, kv_rows, out,
                         out_row, out_head, n_tokens, num_heads, num_kv_heads, head_dim, scale, P));
  if (n_seqs < 0 || n_groups < 0 || max_len < 0 || max_prefix < 0) return set_error(QVL_ERR_INVALID_ARG, "decode_attention: bad sizes");
  if (n_seqs > 65535 || n_groups > 65535) return set_error(QVL_ERR_UNSUPPORTED, "decode_attention: more than 65535 sequences or groups");
  if (!cu_q && n_tokens != n_seqs) return set_error(QVL_ERR_INVALID_ARG, "decode_attention: %lld tokens of %lld sequences without cu_q", (long long)n_tokens, (long long)n_seqs);
  if (n_tokens == 0 || n_seqs == 0) return QVL_OK;
  if (!k_start || !k_len || (n_groups > 0 && (!cu_groups || !prefix_start || !prefix_len)))
    return set_error(QVL_ERR_INVALID_ARG, "decode_attention: NULL pointer");
  if ((uintptr_t)k_start % 8 || (uintptr_t)k_len % 4 || (uintptr_t)cu_q % 4 || (uintptr_t)cu_groups % 4 ||
      (uintptr_t)prefix_start % 8 || (uintptr_t)prefix_len % 4)
    return set_error(QVL_ERR_MISALIGNED, "decode_attention: the sequences' state");
  P.cu_q = cu_q;
  P.k_start = k_start;
  P.k_len = k_len;
  P.cu_groups = cu_groups;
  P.prefix_start = prefix_start;
  P.prefix_len = prefix_len;
  P.n_seqs = (int)n_seqs;
  P.n_groups = (int)n_groups;
  QVL_ATTN_LAUNCH(decode_kernel, dim3((unsigned)n_seqs, (unsigned)num_kv_heads));
  return check_launch("decode_attention");
}

}  // extern "C"
