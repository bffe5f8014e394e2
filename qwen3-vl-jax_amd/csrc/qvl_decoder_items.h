// The work items of the causal attention, shared by the host list and the kernels.
#pragma once
#include "qvl_decoder.h"
#include "qvl_host_common.h"

namespace qvl {

// An item, QVL_CAUSAL_ITEM_WORDS int32: first query token of the sequence, its new tokens, its keys, first row of the tile,
// key/value head, slot of the partial result or -1, low and high word of the first cache row, first key tile, key tile
// after the last. After the items, for each tile that is cut into parts: the same, with the first part's slot, and in the
// last two words 0 and the number of parts. A tile's rows are (token, head of the group) pairs of one key/value head, token by token: row r is token
// r / group, head kv_head * group + r % group, so that the heads that share keys read them together.
constexpr int kItemWords = QVL_CAUSAL_ITEM_WORDS;
constexpr int kItemRows = 128;   // ... or 256 (bf16), as the list says
constexpr int kItemMaxHeads = 0xfff;
constexpr int64_t kItemMaxLen = 0x3fffffff;   // lengths, tokens and rows stay well inside int32

}  // namespace qvl
