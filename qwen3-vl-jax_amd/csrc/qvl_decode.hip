// Attention of a few new tokens of each sequence over a cache, the sequences' state read on the device: bound by reading
// the keys and values once.
//
// Without prefixes one launch streams over all keys of all sequences: their blocks of 32 keys, sequence by sequence, are one
// line cut into equal runs, each taken by one workgroup a key/value head, so that the lengths need not be known on the
// host and unlike ones leave no workgroup slot idle. (A workgroup for each part of each sequence: 96 lengths from 1 to 7900,
// 32/8 heads, bf16: 358 us at best, its slots 58 % occupied; one read of the keys takes 252 us at 6.2 TB/s.) The heads of one
// run go by neighbouring workgroups: they read the same cache rows at the same time, whole rows and not 256 bytes here and
// there. (One line over heads too, its runs at unlike places: 438 us.) A job, a tile of a sequence's rows, that lies in one
// run is finished there; one that crosses runs leaves parts, which a second launch joins.
//
// 96 sequences of up to 7900 keys, 32/8 heads of 128, bf16: 322 us, 4.9 TB/s; one of 9001 keys: 14 us and 5.5 for the join.
//
// With prefixes the tokens of a group are the rows of one more problem, the prefix's keys for all of them at once, 128 (32)
// rows a workgroup and the keys in parts; the sequences' own keys are parts beside them, and one join covers both. (Tiles of
// 256 rows for the prefix, then the own keys and the join in a second launch: 160 us, not 147, for 256 sequences on 24007
// keys: the own keys, bound by memory, no longer run beside the prefix, bound by the matrix cores.)
// 48 sequences after 9216 shared keys 28 us, 256 after 24007 144 us.
#include "qvl_decoder_line.h"

namespace qvl {

template <typename T, int D, typename W>
__device__ __forceinline__ void decode_stream(const AttnParams& P, const DecodeState& S) {
  using K = KeysUnit<T, D>;
  __shared__ __attribute__((aligned(16))) char smem[std::max(K::kLds, kJoinBytes<T, D>)];
  __shared__ Line L;
  const int run = blockIdx.x / P.hkv, kvh = blockIdx.x % P.hkv;
  int64_t total, pos, end, base = 0;
  int n, seq = 0;
  Sequence q;
  find_run(P, S, L, run, gridDim.x / P.hkv, total, n, pos, end, seq, base, q);
  SplitJob joined{};
  while (pos < end) {
    const int blocks = q.blocks;
    const int64_t own = (int64_t)q.jobs * blocks;
    if (pos >= base + own) {           // the next sequence (jobs == 0: it has no rows)
      base += own;
      q = uniform(sequence_of(P, S, ++seq));
      continue;
    }
    Unit u;
    const int64_t start = q.start;
    u.token0 = q.token0;
    u.len = q.len;
    const int64_t into = pos - base;
    int job = 0, b0 = (int)into;
    if (into >= blocks) {
      job = (int)(into / blocks);
      b0 = (int)(into % blocks);
    }
    const int b1 = (int)min((int64_t)blocks, b0 + (end - pos));
    u.kvh = kvh;
    u.row0 = job * W::kRows;
    u.rows = q.tokens * P.group;
    u.lim0 = u.len - q.tokens + 1;
    const int n_rows = min(W::kRows, u.rows - u.row0);
    const bool whole = b0 == 0 && b1 == blocks, bad = bad_keys(P, start, u.len);
    if (bad) {
      for (int i = threadIdx.x; i < n_rows * (D / 4); i += 256)
        store4<T>(out_row<T, D>(P, u, u.row0 + i / (D / 4)), i % (D / 4) * 4, f32x4{NAN, NAN, NAN, NAN});
    } else {
      u.k = P.k.p + start * P.k.row + u.kvh * P.k.head;
      u.v = P.v.p + start * P.v.row + u.kvh * P.v.head;
      W w;
      w.init(P, u, u.row0);
      K::run(P, u, w, smem, b0, min(b1, (u.len + 31) >> 5));
      const int64_t slot = ((int64_t)(2 * run + (b0 == 0)) * P.hkv + kvh) * S.slot_rows;
      join_waves<T, D>(P, u, w, smem, u.row0, b0 * 32, !whole, [&](int r) { return slot + r; });
    }
    if (b0 > 0 && b1 == blocks) {
      // the run that holds the job's first block: the last whose share begins there or before
      const int64_t first = pos - b0;
      int w0 = (int)min((int64_t)((float)first / (float)total * n), (int64_t)run);
      while (w0 > 0 && share(total, w0, n) > first) --w0;
      while (w0 < run && share(total, w0 + 1, n) <= first) ++w0;
      joined = SplitJob{u.token0, u.rows, u.row0, w0, run - w0 + 1};
    }
    pos += b1 - b0;
  }
  if (threadIdx.x == 0 && kvh == 0) S.split[run] = joined;
}
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void decode_stream_kernel(AttnParams P, DecodeState S) { decode_stream<T, D, Wave<T, D>>(P, S); }
template <int D>
__global__ __launch_bounds__(256, 2) void decode_stream_few_kernel(AttnParams P, DecodeState S) { decode_stream<float, D, FewWave<D>>(P, S); }

// Part p of a split job: the second slot of its first run (the job begins inside it), the first slot of each later one.
template <typename T, int D>
__global__ __launch_bounds__(256) void decode_stream_join_kernel(AttnParams P, DecodeState S) {
  const SplitJob j = S.split[blockIdx.x];
  if (j.parts == 0) return;
  const int kvh = blockIdx.y;
  const Unit u{nullptr, nullptr, 0, 0, j.token0, j.rows, j.row0, kvh};
  const int n = min(S.tile, j.rows - j.row0), per = (n + gridDim.z - 1) / gridDim.z, r0 = blockIdx.z * per;
  join_parts<T, D>(P, r0, min(r0 + per, n), j.parts,
                   [&](int r, int p) { return ((int64_t)(2 * (j.first + p) + (p == 0)) * P.hkv + kvh) * S.slot_rows + r; },
                   [&](int r) { return out_row<T, D>(P, u, j.row0 + r); });
}

// ---------------------------------------------------------------------------------------------
// with prefixes
// ---------------------------------------------------------------------------------------------
// Row (token, head) of part `part`, for row r of the unit.
__device__ __forceinline__ int64_t part_row(const AttnParams& P, const Unit& u, int part, int r) {
  const int t = (int)((uint32_t)r / (uint32_t)P.group), g = r - t * P.group;
  return ((int64_t)part * P.n_tokens + u.token0 + t) * (P.hkv * P.group) + u.kvh * P.group + g;
}

// Rows without keys in this part (0), or of keys that may not be read (NaN).
__device__ __forceinline__ void write_fixed(const AttnParams& P, const Unit& u, int part, float value) {
  for (int r = threadIdx.x; r < u.rows; r += 256) P.part_ml[part_row(P, u, part, r)] = f32x2{value == 0.f ? -INFINITY : value, value};
}

// Workgroups [0, prefix units): a part of a group's prefix for a tile of the group's rows (ROWS: tiles of 128, else of W's);
// the others: a part of a sequence's own keys for its rows. The key/value head runs fastest, then the part, so that the
// tiles of one part of the prefix meet in one L2 where heads x parts fill the 8 XCDs evenly.
template <typename T, int D, typename W, bool ROWS>
__device__ __forceinline__ void prefix_unit(const AttnParams& P, const DecodeState& S) {
  using R = RowsUnit<T, D>;
  using K = KeysUnit<T, D>;
  __shared__ __attribute__((aligned(16))) char smem[std::max({K::kLds, kJoinBytes<T, D>, ROWS ? std::max(R::kLds, 4 * kWriteLds) : 0})];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int prefix_units = P.hkv * S.prefix_parts * S.prefix_tiles * S.n_groups;
  const bool own = (int)blockIdx.x >= prefix_units;
  int id = own ? blockIdx.x - prefix_units : blockIdx.x;
  Unit u;
  u.kvh = id % P.hkv;
  id /= P.hkv;
  const int parts = own ? S.own_parts : S.prefix_parts, p = id % parts, chunk = own ? S.own_chunk : S.prefix_chunk;
  const int part = own ? S.prefix_parts + p : p;
  id /= parts;
  const int tile0 = own ? 0 : id % S.prefix_tiles, who = own ? id : id / S.prefix_tiles;   // a sequence, or a group
  int s0 = who, s1 = who + 1;
  if (!own) {
    s0 = min(max(S.cu_groups[who], 0), S.n_seqs);
    s1 = min(max(S.cu_groups[who + 1], 0), S.n_seqs);
  }
  const int tokens = uniform(s1 > s0 ? (int)tokens_of(P, S, s0, s1, u.token0) : 0);
  u.rows = tokens * P.group;
  if (u.rows == 0) return;
  u.token0 = uniform(u.token0);
  // a sequence of no group has no prefix
  if (own && p == 0 && (who < S.cu_groups[0] || who >= S.cu_groups[S.n_groups]))
    for (int i = 0; i < S.prefix_parts; ++i) write_fixed(P, u, i, 0.f);
  const int64_t start = uniform(own ? S.k_start[who] : S.prefix_start[who]);
  u.len = uniform(own ? S.k_len[who] : S.prefix_len[who]);
  if (bad_keys(P, start, u.len)) {
    write_fixed(P, u, part, NAN);
    return;
  }
  u.lim0 = own ? u.len - tokens + 1 : u.len;
  const int ka = (int)min((int64_t)p * chunk, (int64_t)u.len);
  const int kb = p + 1 == parts ? u.len : (int)min((int64_t)ka + chunk, (int64_t)u.len);
  if (ka >= kb) {
    write_fixed(P, u, part, 0.f);
    return;
  }
  u.k = P.k.p + start * P.k.row + u.kvh * P.k.head;
  u.v = P.v.p + start * P.v.row + u.kvh * P.v.head;
  if (ROWS && !own) {
    for (int row0 = tile0 * kItemRows; row0 < u.rows; row0 += S.prefix_tiles * kItemRows) {
      Wave<T, D> w;
      w.init(P, u, row0 + wave * 32);
      R::run(P, u, w, smem, ka / R::kBN, (kb + R::kBN - 1) / R::kBN);
      const int row = row0 + wave * 32 + (threadIdx.x & 31);
      const int64_t at = part_row(P, u, part, min(row, u.rows - 1));
      write_rows<T, D>(P, u, w, smem + wave * kWriteLds, row, P.part_o + at * D, P.part_ml + at, true);
      __syncthreads();                         // the tiles may be written again
    }
  } else {
    const int step = own ? W::kRows : S.prefix_tiles * W::kRows;
    for (int row0 = tile0 * W::kRows; row0 < u.rows; row0 += step) {
      W w;
      w.init(P, u, row0);
      K::run(P, u, w, smem, ka / 32, (kb + 31) / 32);
      join_waves<T, D>(P, u, w, smem, row0, ka, true, [&](int r) { return part_row(P, u, part, row0 + r); });
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void prefix_rows_kernel(AttnParams P, DecodeState S) { prefix_unit<T, D, Wave<T, D>, true>(P, S); }
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void prefix_keys_kernel(AttnParams P, DecodeState S) { prefix_unit<T, D, Wave<T, D>, false>(P, S); }
template <int D>
__global__ __launch_bounds__(256, 2) void prefix_few_kernel(AttnParams P, DecodeState S) { prefix_unit<float, D, FewWave<D>, false>(P, S); }

template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(AttnParams P, DecodeState S) {
  const int64_t heads = P.hkv * P.group, total = P.n_tokens * heads;
  const int64_t first = (S.cu_q ? (int64_t)max(S.cu_q[0], 0) : 0) * heads;
  const int64_t end = (S.cu_q ? min((int64_t)S.cu_q[S.n_seqs], P.n_tokens) : P.n_tokens) * heads;
  const int parts = S.prefix_parts + S.own_parts;
  const int64_t per = 256 / (D / 4) / join_split(parts);   // rows a workgroup
  const int64_t r0 = (int64_t)blockIdx.x * per;
  const int64_t a = max(r0, first), b = min(r0 + per, end);
  if (a >= b) return;
  join_parts<T, D>(P, (int)(a - r0), (int)(b - r0), parts, [&](int r, int p) { return p * total + r0 + r; },
                   [&](int r) {
                     const int64_t token = (r0 + r) / heads;
                     return const_cast<char*>(P.out.p) + token * P.out.row + (r0 + r - token * heads) * P.out.head;
                   });
}

// How a launch is laid out: from the sizes alone, so that the workspace can be told beforehand.
struct DecodePlan {
  int runs, slot_rows;                                                  // streaming
  int own_parts, own_chunk, prefix_parts, prefix_chunk, prefix_tiles;   // with prefixes
  bool prefix_rows, few;   // with prefixes: tiles of 128 rows; fp32: tiles of 16 rows
  int tile;
  int64_t units;
  size_t part_rows, split_bytes;
};

// Parts of at least 128 keys (a block of 32 a wave), as many as fill `slots` workgroups once.
static int split_parts(int64_t keys, int64_t units, int64_t slots, int& chunk) {
  int64_t parts = std::min({slots / std::max<int64_t>(units, 1), (keys + 127) / 128, (int64_t)64});
  parts = std::max<int64_t>(parts, 1);
  const int64_t c = round_up(std::max<int64_t>((keys + parts - 1) / parts, 1), 64);
  chunk = (int)std::min<int64_t>(c, kItemMaxLen);
  return (int)std::max<int64_t>((keys + c - 1) / c, 1);
}

static int decode_plan(const char* what, int64_t n_tokens, int64_t n_seqs, int64_t max_len, int64_t n_groups, int64_t max_prefix,
                       int32_t num_heads, int32_t num_kv_heads, int32_t dtype, int32_t head_dim, DecodePlan& D) {
  if (n_tokens < 0 || n_seqs < 0 || n_groups < 0 || max_len < 0 || max_prefix < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_seqs > 65535 || n_groups > 65535) return set_error(QVL_ERR_UNSUPPORTED, "%s: more than 65535 sequences or groups", what);
  if (max_len > kItemMaxLen || max_prefix > kItemMaxLen) return set_error(QVL_ERR_UNSUPPORTED, "%s: lengths", what);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(QVL_ERR_INVALID_ARG, "%s: %d heads over %d key/value heads", what, num_heads, num_kv_heads);
  const int64_t rows = n_tokens * (num_heads / num_kv_heads);
  if (num_heads > kItemMaxHeads || n_tokens > kItemMaxLen || rows > kItemMaxLen) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  // workgroups a GPU holds: two a CU, one where the tiles take 128 KB (fp32, head_dim 128)
  const int64_t cus = gemm_device_cus(), slots = cus * (dtype == QVL_DTYPE_F32 && head_dim == 128 ? 1 : 2);
  D = DecodePlan{};
  // fp32 is bound by its matrix products (32 rows: 8192 cycles a block of 32 keys), so few rows take tiles of 16: 16/8 heads of
  // 128, 96 sequences of up to 5760 keys 419 us, not 478 (2.3 GB: 5.4 TB/s), one of 9000 26, not 32; nine times two sequences
  // after prefixes of 2000 to 4000 keys, 3 tokens each, 47, not 93
  const int64_t own_rows = (rows + std::max<int64_t>(n_seqs, 1) - 1) / std::max<int64_t>(n_seqs, 1);   // a sequence's, in the mean
  D.few = dtype == QVL_DTYPE_F32 && own_rows <= 16 && (n_groups == 0 || rows <= 16 * n_groups);
  D.tile = D.few ? 16 : 32;
  if (n_groups == 0) {
    // A run for each compute unit where that leaves it at most 40 blocks, else for each slot (8 heads: one sequence of 9001 keys
    // 20 us and not 25, of 31000 33.5 and not 37; 16 of up to 8000 62.5 and not 72); no more than give each wave a block,
    // nor fewer than there are jobs.
    const int64_t tiles = std::max<int64_t>((own_rows + D.tile - 1) / D.tile, 1);
    const int64_t jobs = n_seqs * tiles, blocks = jobs * ((max_len + 31) / 32);
    const int64_t one = cus / num_kv_heads, most = jobs <= one && blocks <= 40 * one ? one : slots / num_kv_heads;
    D.runs = (int)std::max<int64_t>(std::min(most, std::max((blocks + 3) / 4, jobs)), 1);
    D.units = (int64_t)D.runs * num_kv_heads;
    D.slot_rows = (int)std::min<int64_t>(D.tile, std::max<int64_t>(rows, 1));
    D.part_rows = (size_t)D.units * 2 * D.slot_rows;
    D.split_bytes = round_up(D.runs * sizeof(SplitJob), 16);
    return QVL_OK;
  }
  const int64_t mean = (rows + n_groups - 1) / n_groups;
  D.prefix_rows = mean > 32;
  const int64_t tile = D.prefix_rows ? kItemRows : D.tile;
  D.prefix_tiles = (int)std::max<int64_t>(std::min((rows + tile - 1) / tile, (mean + tile - 1) / tile * (n_groups > 1 ? 2 : 1)), 1);
  D.own_parts = split_parts(max_len, n_seqs * num_kv_heads, slots, D.own_chunk);
  // About one unit on the prefixes for each compute unit, beside units on the sequences' own keys (one for each slot: 192
  // rows on 9216 keys 36 us, not 30; 1024 on 24007 141, not 133). Tiles that groups of unlike size may leave empty
  // count half: twice 1024 rows 228 us, not 336.
  const int64_t busy = std::min(n_groups * D.prefix_tiles, (rows + tile - 1) / tile + n_groups / 2) * num_kv_heads;
  D.prefix_parts = split_parts(max_prefix, busy, cus + busy / 8, D.prefix_chunk);
  D.units = (int64_t)num_kv_heads * (n_groups * D.prefix_parts * D.prefix_tiles + n_seqs * D.own_parts);
  if (D.units > 0x7fffffffLL || n_tokens * num_heads > 0x7fffffffLL) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  D.part_rows = (size_t)(D.prefix_parts + D.own_parts) * n_tokens * num_heads;
  return QVL_OK;
}

#define QVL_FEW_LAUNCH(KERNEL, GRID, ...)                                                                        \
  do {                                                                                                           \
    if (head_dim == 128) hipLaunchKernelGGL((KERNEL<128>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__); \
    else hipLaunchKernelGGL((KERNEL<64>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__);                 \
  } while (0)

static size_t workspace_bytes_of(const DecodePlan& D, int32_t head_dim) {
  return D.split_bytes + D.part_rows * ((size_t)head_dim + 2) * sizeof(float);
}

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_decode_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t max_len, int64_t n_groups, int64_t max_prefix,
                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "decode_workspace_size: bytes is NULL");
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "decode_workspace_size: head_dim=%d", head_dim);
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "decode_workspace_size: dtype %d", dtype);
  DecodePlan plan;
  QVL_TRY_RC(decode_plan("decode_workspace_size", n_tokens, n_seqs, max_len, n_groups, max_prefix, num_heads, num_kv_heads, dtype,
                         head_dim, plan));
  *bytes = workspace_bytes_of(plan, head_dim);
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
  DecodePlan plan;
  QVL_TRY_RC(decode_plan("decode_attention", n_tokens, n_seqs, max_len, n_groups, max_prefix, num_heads, num_kv_heads, dtype,
                         head_dim, plan));
  if (!cu_q && n_tokens != n_seqs) return set_error(QVL_ERR_INVALID_ARG, "decode_attention: %lld tokens of %lld sequences without cu_q", (long long)n_tokens, (long long)n_seqs);
  if (n_tokens == 0 || n_seqs == 0) return QVL_OK;
  if (!k_start || !k_len || (n_groups > 0 && (!cu_groups || !prefix_start || !prefix_len)))
    return set_error(QVL_ERR_INVALID_ARG, "decode_attention: NULL pointer");
  if ((uintptr_t)k_start % 8 || (uintptr_t)k_len % 4 || (uintptr_t)cu_q % 4 || (uintptr_t)cu_groups % 4 ||
      (uintptr_t)prefix_start % 8 || (uintptr_t)prefix_len % 4)
    return set_error(QVL_ERR_MISALIGNED, "decode_attention: the sequences' state");
  const size_t need = workspace_bytes_of(plan, head_dim);
  if (workspace_bytes < need || !workspace)
    return set_error(QVL_ERR_WORKSPACE, "decode_attention: workspace %zu < %zu", workspace_bytes, need);
  if ((uintptr_t)workspace % 16) return set_error(QVL_ERR_MISALIGNED, "decode_attention: workspace");
  P.part_o = (float*)((char*)workspace + plan.split_bytes);
  P.part_ml = (f32x2*)(P.part_o + plan.part_rows * head_dim);
  const DecodeState S{cu_q, k_start, k_len, cu_groups, prefix_start, prefix_len, (int)n_seqs, (int)n_groups, plan.own_parts,
                      plan.own_chunk, plan.prefix_parts, plan.prefix_chunk, plan.prefix_tiles, (SplitJob*)workspace, plan.slot_rows, plan.tile};
  const dim3 units((unsigned)plan.units);
  if (n_groups == 0) {
    if (plan.few) QVL_FEW_LAUNCH(decode_stream_few_kernel, units, P, S);
    else QVL_ATTN_LAUNCH(decode_stream_kernel, units, P, S);
    QVL_TRY_RC(check_launch("decode_stream"));
    if (plan.runs == 1) return QVL_OK;
    // a split job's rows over a few workgroups: they are few, and each reads every part
    QVL_ATTN_LAUNCH(decode_stream_join_kernel, dim3((unsigned)plan.runs, (unsigned)num_kv_heads, (unsigned)std::min(plan.slot_rows, 16)), P, S);
    return check_launch("decode_stream_join");
  }
  // (tiles of 128 rows take what lies behind a prefix's last key for zeros; where V's rows lie closer than a row is long it is
  // not, and the tiles of 32 tell it apart)
  if (plan.prefix_rows && v_row >= head_dim) QVL_ATTN_LAUNCH(prefix_rows_kernel, units, P, S);
  else if (plan.few) QVL_FEW_LAUNCH(prefix_few_kernel, units, P, S);
  else QVL_ATTN_LAUNCH(prefix_keys_kernel, units, P, S);
  QVL_TRY_RC(check_launch("prefix_attention"));
  const int64_t per = 256 / (head_dim / 4) / join_split(plan.prefix_parts + plan.own_parts);
  QVL_ATTN_LAUNCH(prefix_join_kernel, dim3((unsigned)((n_tokens * num_heads + per - 1) / per)), P, S);
  return check_launch("prefix_join");
}

}  // extern "C"
