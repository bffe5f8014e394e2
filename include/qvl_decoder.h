/*
 * qvl_decoder.h — the text-decoder side of libqvl.so (gfx950): what a decoder layer computes between its qkv Dense and
 * its output Dense, for prompts that hold injected vision rows and for the tokens generated after them.
 *
 *   qvl_text_rotary_table, qvl_qk_norm_rotary   per-head RMSNorm of q and k and the (t, h, w) position rotation, one
 *                                               pass; k and v rows go to the cache
 *   qvl_causal_worklist, qvl_causal_attention   packed prompts: causal over a sequence's own new tokens, full over the
 *                                               keys it had before; grouped heads
 *   qvl_decode_attention                        a few new tokens of each sequence over its cache; sequences may come in
 *                                               groups that share a prefix, which is read once for the whole group
 *
 * The conventions of qvl_vision.h hold (streams, no allocation, error codes, thread safety). Beside them:
 *   - q, k, v, out and the caches are views [rows, heads, head_dim] of one dtype: element (r, h, d) lies at
 *     p[r * row_stride + h * head_stride + d], strides in elements, 0 <= stride < 2^31, both multiples of 16 bytes
 *     like the pointers (QVL_ERR_MISALIGNED). So the column blocks of a qkv Dense output, a cache [rows, heads, dim]
 *     and one [heads, rows, dim] all serve as they are. Rows of k and v of the attention lie at most 64 MiB apart
 *     (QVL_ERR_UNSUPPORTED). Rows and heads of an output do not lie over one another, nor over an input.
 *   - num_heads is a multiple of num_kv_heads; query head h reads key/value head h / (num_heads / num_kv_heads).
 *   - head_dim 64 or 128, bf16 or fp32. Sums, softmax statistics and norms are held in fp32 in both; outputs are
 *     rounded once.
 *   - Offsets are 64-bit: a cache may be larger than 4 GiB. Counts of tokens, tokens x (num_heads / num_kv_heads) and keys
 *     of a sequence stay below 2^30, heads below 4096, sequences and groups of a decode call below 65536 (QVL_ERR_UNSUPPORTED;
 *     lengths that lie on the device: NaN).
 *   - What a call computes depends on its inputs alone, bit for bit: no atomics, and parts are joined in a fixed order.
 */
#ifndef QVL_DECODER_H
#define QVL_DECODER_H

#include "qvl_vision.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The rotation of qvl_qk_norm_rotary as a host table [head_dim / 2][2] uint64, copied to the device by the caller:
 * entry j holds theta^(-2j / head_dim) / 2pi as a binary fraction of 2^64 turns per position, and the axis (0 t, 1 h,
 * 2 w) whose position drives it. `section` counts the frequencies of each axis: one after the other (they sum to
 * head_dim / 2), or interleaved: frequency j follows axis j % 3 while j < 3 * section[j % 3], else t. head_dim a
 * multiple of 4, at most 256; theta finite, > 1. */
int qvl_text_rotary_table(int32_t head_dim, double theta, const int32_t* h_section, int32_t interleaved,
                          uint64_t* h_table);

/* For each token n: y = x * rsqrt(mean(x^2) + eps) * w over each head of q (w = q_norm) and of k (k_norm), fp32 [head_dim],
 * then the rotation of dims (j, j + head_dim/2) by the angle of frequency j at the position
 * d_positions[axis * pos_stride + n] (int32; pos_stride 0: one position for the three axes), all in fp32 and rounded
 * once. The angle is reduced in 64-bit fixed point, so positions of any int32 keep full precision.
 * q goes to q_out row n; k to k_out and v (copied as it is) to v_out at row d_rows[n] (int64; NULL: row n), and a token
 * whose row lies outside [0, out_rows) writes neither. v and v_out may be NULL together. Rows should differ: the row of
 * two tokens holds values of either. Outputs may be their inputs (same pointer and strides, d_rows NULL); other overlaps
 * are not allowed. */
int qvl_qk_norm_rotary(void* stream, int32_t dtype,
                       const void* d_q, int64_t q_row_stride, int64_t q_head_stride,
                       const void* d_k, int64_t k_row_stride, int64_t k_head_stride,
                       const void* d_v, int64_t v_row_stride, int64_t v_head_stride,
                       const float* d_q_norm, const float* d_k_norm, float eps,
                       const int32_t* d_positions, int64_t pos_stride, const uint64_t* d_table,
                       const int64_t* d_rows, int64_t out_rows,
                       void* d_q_out, int64_t qo_row_stride, int64_t qo_head_stride,
                       void* d_k_out, int64_t ko_row_stride, int64_t ko_head_stride,
                       void* d_v_out, int64_t vo_row_stride, int64_t vo_head_stride,
                       int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim);

/* Work list of qvl_causal_attention (host): sequence i brings h_new[i] query tokens (packed one sequence after the other)
 * and has h_len[i] keys, the new tokens' own among them, in cache rows [h_start[i], h_start[i] + h_len[i]). Query token t
 * sees keys j <= h_len - h_new + t; where h_len < h_new the first tokens see none. Items of QVL_CAUSAL_ITEM_WORDS int32,
 * dealt to 8 queues (one per XCD) and ordered by work; where tiles would leave compute units idle, they are cut along their
 * keys. The list holds n_items items, n_parts of which are parts of a tile, and after them n_joins entries for the tiles
 * that are in parts. *tile_rows: the rows (token, head) of a tile, 128 or 256 (bf16 only); 0 on entry lets a model of the
 * kernels' times choose, and the choice is written. h_items NULL: only the counts and the tile height are written;
 * capacity: the entries there is room for, n_items + n_joins at least. */
#define QVL_CAUSAL_ITEM_WORDS 10
int qvl_causal_worklist(int64_t n_seqs, const int64_t* h_new, const int64_t* h_len, const int64_t* h_start,
                        int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t n_cus,
                        int32_t* tile_rows, int32_t* h_items, int64_t capacity, int64_t* n_items, int64_t* n_parts,
                        int64_t* n_joins);

/* out = softmax(scale * q k^T, keys the token does not see left out) v, for every token of the sequences of a
 * qvl_causal_worklist list (device copy, 16-byte aligned; made for the same heads, head_dim, dtype and tile_rows). A token that sees
 * no key gets zeros; rows of no sequence are left as they are. Keys a token does not see never enter its output, whatever
 * they hold. An item whose rows leave [0, n_tokens) or [0, kv_rows) is not run. scale: finite, > 0. The workspace
 * (qvl_causal_workspace_size; 16-byte aligned) holds the parts' partial outputs: calls that overlap need one each. */
int qvl_causal_workspace_size(int32_t head_dim, int32_t tile_rows, int64_t n_parts, size_t* bytes);
int qvl_causal_attention(void* stream, int32_t dtype,
                         const void* d_q, int64_t q_row_stride, int64_t q_head_stride,
                         const void* d_k, int64_t k_row_stride, int64_t k_head_stride,
                         const void* d_v, int64_t v_row_stride, int64_t v_head_stride, int64_t kv_rows,
                         int32_t tile_rows, const int32_t* d_items, int64_t n_items, int64_t n_parts, int64_t n_joins, float scale,
                         void* d_out, int64_t out_row_stride, int64_t out_head_stride,
                         int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* d_workspace, size_t workspace_bytes);

/* Attention of new tokens over a cache whose state lies on the device, so that a captured graph replays with the lengths
 * of the moment. Sequence i brings query tokens [d_cu_q[i], d_cu_q[i+1]) (NULL: token i, n_tokens == n_seqs) and has
 * d_k_len[i] keys in cache rows from d_k_start[i], the new tokens' own among them, seen as in qvl_causal_attention.
 * With n_groups > 0, sequences [d_cu_groups[g], d_cu_groups[g+1]) also see, before their own keys, all of the
 * d_prefix_len[g] cache rows from d_prefix_start[g]; one softmax covers both; sequences of no group have no prefix.
 * d_cu_groups stays in [0, n_seqs] and d_cu_q in [0, n_tokens], neither ever falling; rows before d_cu_q[0] and from
 * d_cu_q[n_seqs] on are left as they are. A token that sees no key gets zeros. The tokens of a sequence whose keys (or prefix) leave [0, kv_rows) come out NaN; nothing outside is read.
 * max_len and max_prefix are the lengths the launch is laid out for (a captured call's largest); longer ones are still
 * right. The workspace (qvl_decode_workspace_size of the same sizes, with the same device current; 16-byte aligned) holds
 * partial outputs: calls that overlap need one each. */
int qvl_decode_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t max_len, int64_t n_groups, int64_t max_prefix,
                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, size_t* bytes);
int qvl_decode_attention(void* stream, int32_t dtype,
                         const void* d_q, int64_t q_row_stride, int64_t q_head_stride,
                         const void* d_k, int64_t k_row_stride, int64_t k_head_stride,
                         const void* d_v, int64_t v_row_stride, int64_t v_head_stride, int64_t kv_rows,
                         const int32_t* d_cu_q, int64_t n_seqs, const int64_t* d_k_start, const int32_t* d_k_len,
                         int64_t max_len, const int32_t* d_cu_groups, int64_t n_groups, const int64_t* d_prefix_start,
                         const int32_t* d_prefix_len, int64_t max_prefix, float scale,
                         void* d_out, int64_t out_row_stride, int64_t out_head_stride,
                         int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* d_workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* QVL_DECODER_H */
