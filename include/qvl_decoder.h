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
 *   qvl_paged_append, qvl_paged_unpack,         a cache in pages and 4 bits a value: new tokens' keys and values into it (norm and
 *   qvl_paged_attention                         rotation on the way), read back as rows, and attended to
 *   qvl_sample_tokens                           the next token of rows of logits: temperature, top-k, top-p, min-p
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
 *   - What a call computes depends on its inputs alone, bit for bit: no atomics but on whole numbers, and parts are joined in a
 *     fixed order.
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

/* A cache in pages of `page_rows` tokens (a power of two, 16 to 4096), 4 bits a value. A head's values go in groups of 64; of a group
 * x the scale is s = bf16(fp32(max|x| / 6)) (rounded to nearest even, twice) and each value becomes the number nearest to |x| / s of 0,
 * .5, 1, 1.5, 2, 3, 4, 6 (a tie goes to 0, 1, 2 or 4) with x's sign, and stands for s times it. A group with a NaN or an infinity, or whose
 * scale is beyond bf16, stands for NaN. What a group stands for in fp32 gives the same group again where s is 0, NaN or normal and 6 s
 * finite (a subnormal s has few bits, and 6 s of values over 3.399e38 may be beyond fp32).
 * The bytes of a page are this library's own; qvl_paged_cache_size tells how many a cache of
 * n_pages takes (64-byte aligned; any content until tokens are written).
 * Token t of sequence i lies in page d_page_table[i * table_stride + t / page_rows], slot t % page_rows. Sequences may share pages.
 * An entry outside [0, n_pages) is no page: what would be written there is dropped, what would be read there is NaN. */
int qvl_paged_cache_size(int64_t n_pages, int32_t page_rows, int32_t num_kv_heads, int32_t head_dim, size_t* bytes);

/* Keys and values of new tokens into their pages. Sequence i brings tokens [d_cu_q[i], d_cu_q[i+1]) of k and v (NULL: token i,
 * n_tokens == n_seqs) and has d_k_len[i] tokens with them: the last one's t is d_k_len[i] - 1. Tokens of no sequence, and those whose t
 * is negative or beyond the table, are dropped. With q, the norm and rotation of qvl_qk_norm_rotary run on the way: q to q_out (rows
 * of no sequence are left as they are) as there, k to 4 bits; k's norm, rotation and codes are formed in fp64. q NULL: k goes to 4 bits as it is, and
 * q_norm, k_norm, eps, positions, table, q_out and num_heads are not looked at. q_out may be q. A slot that two tokens of
 * a call are given holds any mixture of the two. */
int qvl_paged_append(void* stream, int32_t dtype,
                     const void* d_q, int64_t q_row_stride, int64_t q_head_stride,
                     const void* d_k, int64_t k_row_stride, int64_t k_head_stride,
                     const void* d_v, int64_t v_row_stride, int64_t v_head_stride,
                     const float* d_q_norm, const float* d_k_norm, double eps,
                     const int32_t* d_positions, int64_t pos_stride, const uint64_t* d_table,
                     void* d_cache, int64_t n_pages, int32_t page_rows,
                     const int32_t* d_page_table, int64_t table_width, int64_t table_stride,
                     const int32_t* d_cu_q, int64_t n_seqs, const int32_t* d_k_len,
                     void* d_q_out, int64_t qo_row_stride, int64_t qo_head_stride,
                     int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim);

/* Tokens d_first[i] <= t < d_k_len[i] (NULL: from 0) of each sequence read back as rows of k and v, token t's as row
 * d_k_start[i] + t - d_first[i], rounded to dtype once. Rows outside [0, out_rows) are dropped. max_len: the most tokens of a
 * sequence that the launch is laid out for; more are still right. */
int qvl_paged_unpack(void* stream, int32_t dtype, const void* d_cache, int64_t n_pages, int32_t page_rows,
                     const int32_t* d_page_table, int64_t table_width, int64_t table_stride, int64_t n_seqs,
                     const int32_t* d_first, const int32_t* d_k_len, int64_t max_len, const int64_t* d_k_start,
                     void* d_k, int64_t k_row_stride, int64_t k_head_stride,
                     void* d_v, int64_t v_row_stride, int64_t v_head_stride, int64_t out_rows,
                     int32_t num_kv_heads, int32_t head_dim);

/* Attention of new tokens over the pages: qvl_decode_attention (without prefixes) of the values that the pages stand for. The tokens of
 * a sequence with more tokens than its line of the table has room for, or fewer than none, come out NaN, and so does a token that sees a
 * key in no page. What pages hold behind a sequence's last key never enters its output. */
int qvl_paged_attention_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t max_len, int32_t num_heads, int32_t num_kv_heads,
                                       int32_t head_dim, size_t* bytes);
int qvl_paged_attention(void* stream, int32_t dtype,
                        const void* d_q, int64_t q_row_stride, int64_t q_head_stride,
                        const void* d_cache, int64_t n_pages, int32_t page_rows,
                        const int32_t* d_page_table, int64_t table_width, int64_t table_stride,
                        const int32_t* d_cu_q, int64_t n_seqs, const int32_t* d_k_len, int64_t max_len, float scale,
                        void* d_out, int64_t out_row_stride, int64_t out_head_stride,
                        int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                        void* d_workspace, size_t workspace_bytes);

/* The next token of each row of logits [n_rows, vocab] (fp32 or bf16, rows `row_stride` elements apart, vocab at most 2^18), to out[row].
 * With z = (x - max x) / T the weight of a token is W = round(2^44 e^z), formed in fp64. In the order of falling logits (equal ones: rising
 * index) the first top_k are kept (<= 0: all); of them those before which less than top_p of their sum of weights lies (not < 1: all); of
 * them those whose W is no less than min_p 2^44 (not > 0: all). The token is the first index at which the sum of the kept weights up to it is over
 * u times the sum of all (u of [0, 1); others count as 0, or as just below 1). T <= 0 or NaN, top_k 1, top_p <= 0 and min_p > 1: the first in the
 * order. A row with NaN or +infinity, or of -infinities alone, gives -1; tokens of -infinity are never chosen.
 * Each setting is fp32 (top_k int32) [n_rows] on the device, or, where that is NULL, the value that follows it for all rows.
 * The workspace (qvl_sample_workspace_size; 16-byte aligned) holds the rows' histograms: calls that overlap need one each. */
int qvl_sample_workspace_size(int64_t n_rows, size_t* bytes);
int qvl_sample_tokens(void* stream, int32_t dtype, const void* d_logits, int64_t row_stride, int64_t n_rows, int64_t vocab,
                      const float* d_u, const float* d_temperature, float temperature, const int32_t* d_top_k, int32_t top_k,
                      const float* d_top_p, float top_p, const float* d_min_p, float min_p, int64_t* d_out,
                      void* d_workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* QVL_DECODER_H */
