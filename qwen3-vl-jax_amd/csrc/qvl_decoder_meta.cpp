// GPU-free host side of the decoder entries: the rotation table and the causal work list. Plain C++ (no HIP), so that
// it also builds for the CPU sanitizer run.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <array>
#include <vector>

#include "qvl_decoder_items.h"

using namespace qvl;

extern "C" {

int qvl_text_rotary_table(int32_t head_dim, double theta, const int32_t* section, int32_t interleaved, uint64_t* table) {
  if (head_dim <= 0 || head_dim % 4 || head_dim > 256) return set_error(QVL_ERR_INVALID_ARG, "text_rotary_table: head_dim=%d", head_dim);
  if (!(theta > 1.0) || !isfinite(theta)) return set_error(QVL_ERR_INVALID_ARG, "text_rotary_table: theta=%g", theta);
  if (!section || !table) return set_error(QVL_ERR_INVALID_ARG, "text_rotary_table: NULL pointer");
  const int half = head_dim / 2;
  for (int a = 0; a < 3; ++a)
    if (section[a] < 0 || section[a] > half) return set_error(QVL_ERR_INVALID_ARG, "text_rotary_table: section[%d]=%d", a, section[a]);
  if (!interleaved && section[0] + section[1] + section[2] != half)
    return set_error(QVL_ERR_INVALID_ARG, "text_rotary_table: section sums to %d, not head_dim / 2 = %d",
                     section[0] + section[1] + section[2], half);
  for (int j = 0; j < half; ++j) {
    // Turns per position, below 1/2pi: 64 fraction bits hold it to 2^-64 turns, 2^31 positions of it to 2^-33.
    const long double turns = powl((long double)theta, -2.0L * j / head_dim) / 6.283185307179586476925286766559L;
    table[2 * j] = (uint64_t)roundl(ldexpl(turns, 64));
    const int a = j % 3;
    table[2 * j + 1] = interleaved ? (j < 3 * section[a] ? a : 0)
                                   : (j < section[0] ? 0 : j < section[0] + section[1] ? 1 : 2);
  }
  return QVL_OK;
}

int qvl_causal_worklist(int64_t n_seqs, const int64_t* n_new, const int64_t* len, const int64_t* start, int32_t num_heads,
                        int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t n_cus, int32_t* items,
                        int64_t capacity, int64_t* n_items, int64_t* n_whole) {
  if (!n_items || !n_whole) return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: n_items / n_whole is NULL");
  if (n_seqs < 0 || (n_seqs > 0 && (!n_new || !len || !start)))
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: sequences are NULL");
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: head_dim=%d (64 or 128)", head_dim);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: %d heads over %d key/value heads", num_heads, num_kv_heads);
  if (num_heads > kItemHeadMask) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: num_heads=%d", num_heads);
  if (n_cus <= 0) return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: n_cus=%d", n_cus);
  const int64_t group = num_heads / num_kv_heads;
  std::vector<std::array<int32_t, 8>> list;
  int64_t q0 = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    if (n_new[i] < 0 || len[i] < 0 || start[i] < 0 || start[i] > (int64_t)1 << 56)
      return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: sequence %lld: %lld new, %lld keys from row %lld", (long long)i,
                       (long long)n_new[i], (long long)len[i], (long long)start[i]);
    if (len[i] > kItemMaxLen || q0 + n_new[i] > kItemMaxLen || n_new[i] * group > kItemMaxLen)
      return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: sequence %lld is too long", (long long)i);
    for (int64_t r = 0; r < n_new[i] * group; r += kItemRows)
      for (int32_t h = 0; h < num_kv_heads; ++h)
        list.push_back({(int32_t)q0, (int32_t)n_new[i], (int32_t)len[i], (int32_t)r, h, -1,
                        (int32_t)(uint32_t)(start[i] & 0xffffffff), (int32_t)(start[i] >> 32)});
    q0 += n_new[i];
  }
  *n_items = *n_whole = (int64_t)list.size();
  if (!items) return QVL_OK;
  if (capacity < *n_items)
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist capacity %lld < %lld", (long long)capacity, (long long)*n_items);
  for (size_t k = 0; k < list.size(); ++k) std::copy(list[k].begin(), list[k].end(), items + 8 * k);
  return QVL_OK;
}

}  // extern "C"
