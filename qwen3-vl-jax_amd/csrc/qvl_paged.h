// The paged 4-bit cache of the text decoder (qvl_paged_cache.hip writes it and reads it back, qvl_paged_attn.hip attends to it).
//
// A head's D values go in groups of 64: a bf16 scale s and for each value a sign and one of the numbers 0, .5, 1, 1.5, 2, 3, 4, 6
// (e2m1), which stands for s times the number: 4.25 bits a value. These numbers are exact in bf16, so the matrix products take them as
// they are; scales are applied to their sums (K) or to the weights (V) in fp32.
//
// A page holds `page_rows` tokens head by head, in blocks of 16 tokens. A block is laid out as the products' operands lie in the lanes
// of a wave (a lane is row or column r = lane % 16 of an operand and quad = lane / 16), so that a lane's share of K, and of V, is
// one read:
//   K       token by token: 8 pieces of D / 8 values; piece p holds the codes of dims [pE, pE + E) and [D/2 + pE, D/2 + pE + E),
//           E = D / 16. The lane of token r takes pieces 2 quad and 2 quad + 1.
//   V       [4 quads][16 r][4 tokens][D / 16 codes]: of tokens 4 quad + i the dims 4r + j and (D = 128) 64 + 4r + j, j < 4
//   scales  [16 tokens][D / 64] of K, then of V
#pragma once
#include "qvl_common.h"

namespace qvl {

template <int D> struct PageBlock {
  static constexpr int kTokens = 16, kGroups = D / 64, kE = D / 16;
  static constexpr int kTokenBytes = D / 2, kPieceBytes = D / 16, kCodes = kTokens * kTokenBytes, kScales = kTokens * kGroups * 2;
  static constexpr int kK = 0, kV = kCodes, kKScale = 2 * kCodes, kVScale = 2 * kCodes + kScales, kBytes = 2 * (kCodes + kScales);
  static __host__ __device__ constexpr int k_piece(int token, int p) { return kK + token * kTokenBytes + p * kPieceBytes; }
  static __host__ __device__ constexpr int v_word(int token, int r) {
    return kV + (token >> 2) * 4 * kTokenBytes + r * 4 * (D / 32) + (token & 3) * (D / 32);
  }
  static __host__ __device__ constexpr int k_scale(int token) { return kKScale + token * kGroups * 2; }
  static __host__ __device__ constexpr int v_scale(int token) { return kVScale + token * kGroups * 2; }
};

struct Pages {
  char* data;
  const int32_t* table;   // [sequences][width], rows `stride` apart: a sequence's pages
  int64_t stride;
  int width, n_pages, shift, hkv;   // 2^shift tokens a page
  // the page of a sequence's tokens [page << shift, ...); -1: none
  __device__ __forceinline__ int page(int64_t seq, int64_t i) const {
    if (i < 0 || i >= width) return -1;
    const int p = table[seq * stride + i];
    return p >= 0 && p < n_pages ? p : -1;
  }
  template <int D> __device__ __forceinline__ char* block(int page, int head, int token) const {
    return data + ((((int64_t)page * hkv + head) << (shift - 4)) + ((token & ((1 << shift) - 1)) >> 4)) * PageBlock<D>::kBytes;
  }
};

// Checks shared by the entries (qvl_paged_cache.hip).
int pages_of(const char* what, const void* data, int64_t n_pages, int32_t page_rows, const int32_t* table, int64_t table_width,
             int64_t table_stride, int64_t n_seqs, int32_t num_kv_heads, int32_t head_dim, Pages& out);

}  // namespace qvl
