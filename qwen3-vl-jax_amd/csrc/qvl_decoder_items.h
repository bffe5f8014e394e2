// The work items of the causal attention, shared by the host list and the kernels.
#pragma once
#include "qvl_decoder.h"
#include "qvl_host_common.h"

namespace qvl {

// An item: (first query token of the sequence, its new tokens, its keys, first row of the tile, key/value head,
// partial slot or -1, low and high word of its first cache row). A tile's rows are (token, head of the group) pairs of
// one key/value head, token by token: row r is token r / group, head kv_head * group + r % group, so that the heads
// that share keys read them together.
constexpr int kItemRows = 128;   // ... or 256 (bf16), as the list says
constexpr int kItemHeadMask = 0xfff, kItemPartShift = 12, kItemPartsShift = 20;   // the head word: head, part, parts (0: whole)
constexpr int64_t kItemMaxLen = 0x3fffffff;   // lengths, tokens and rows stay well inside int32

}  // namespace qvl
