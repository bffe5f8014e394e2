// CPU sanitizer driver for the decoder's GPU-free host code (qvl_decoder_meta.cpp): rotation tables and causal work lists on
// random and malformed inputs with exactly-sized buffers. Exit 0 = clean.
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "qvl_decoder.h"

static int failures = 0;
#define CHECK(cond)                                                        \
  do {                                                                     \
    if (!(cond)) {                                                         \
      fprintf(stderr, "CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      ++failures;                                                          \
    }                                                                      \
  } while (0)

static void one_list(std::mt19937& rng) {
  auto below = [&](int n) { return (int)(rng() % (uint32_t)n); };
  const int n_seqs = below(9), hkv = 1 + below(8), hq = hkv * (1 + below(7)), hd = below(2) ? 64 : 128, dt = below(2);
  const int top = 1 << below(14);
  std::vector<int64_t> n_new(n_seqs), len(n_seqs), start(n_seqs);
  for (int i = 0; i < n_seqs; ++i) {
    n_new[i] = below(top);
    len[i] = std::max<int64_t>(n_new[i] + below(3 * top) - below(top), 0);
    start[i] = (int64_t)rng() << below(20);
  }
  int32_t rows = 128 * below(dt == QVL_DTYPE_BF16 ? 3 : 2), cus = 1 + below(300);
  int64_t n = -1, parts = -1, joins = -1;
  CHECK(qvl_causal_worklist(n_seqs, n_new.data(), len.data(), start.data(), hq, hkv, hd, dt, cus, &rows, nullptr, 0, &n, &parts, &joins) == QVL_OK);
  std::vector<int32_t> items((size_t)(n + joins) * QVL_CAUSAL_ITEM_WORDS);
  CHECK(qvl_causal_worklist(n_seqs, n_new.data(), len.data(), start.data(), hq, hkv, hd, dt, cus, &rows, items.data(), n + joins, &n, &parts, &joins) == QVL_OK);
  if (n + joins > 1) {   // (no room at all would be a NULL list: a count)
    std::vector<int32_t> small((size_t)(n + joins - 1) * QVL_CAUSAL_ITEM_WORDS);
    CHECK(qvl_causal_worklist(n_seqs, n_new.data(), len.data(), start.data(), hq, hkv, hd, dt, cus, &rows, small.data(), n + joins - 1, &n, &parts, &joins) != QVL_OK);
  }
  // every tile's keys once: the parts' steps sum up to the tile's
  std::map<std::tuple<int, int, int, int>, int64_t> steps;
  int64_t with_slot = 0;
  for (int64_t k = 0; k < n; ++k) {
    const int32_t* it = items.data() + k * QVL_CAUSAL_ITEM_WORDS;
    if (it[1] == 0) continue;
    steps[{it[0], it[1], it[3], it[4]}] += it[9] - it[8];
    with_slot += it[5] >= 0;
    CHECK(it[5] < parts && it[8] >= 0 && it[9] >= it[8]);
  }
  CHECK(with_slot == parts);
  int64_t q0 = 0, tiles = 0;
  for (int i = 0; i < n_seqs; q0 += n_new[i++])
    for (int64_t r = 0; r < n_new[i] * (hq / hkv); r += rows)
      for (int h = 0; h < hkv; ++h, ++tiles) {
        const int64_t last = (std::min<int64_t>(r + rows, n_new[i] * (hq / hkv)) - 1) / (hq / hkv), step = dt == QVL_DTYPE_BF16 ? 64 : 32;
        const int64_t keys = std::max<int64_t>(std::min(len[i] - n_new[i] + 1 + last, len[i]), 0);
        auto at = steps.find({(int)q0, (int)n_new[i], (int)r, h});
        CHECK(at != steps.end() && at->second == (keys + step - 1) / step);
      }
  CHECK(tiles == (int64_t)steps.size());
}

int main() {
  std::mt19937 rng(7);
  const int cases = 300;
  for (int i = 0; i < cases; ++i) one_list(rng);
  for (int hd = 4; hd <= 256; hd += 4) {
    std::vector<uint64_t> table((size_t)hd);
    const int32_t section[3] = {hd / 2, 0, 0};
    for (double theta : {1.0001, 1e4, 5e6, 1e300})
      for (int inter : {0, 1}) CHECK(qvl_text_rotary_table(hd, theta, section, inter, table.data()) == QVL_OK);
  }
  const int64_t one = 1, far = (int64_t)1 << 57, many = (int64_t)1 << 29;
  int64_t n = 0, p = 0, j = 0;
  int32_t rows = 0;
  CHECK(qvl_causal_worklist(1, &one, &one, &far, 8, 8, 64, 1, 256, &rows, nullptr, 0, &n, &p, &j) != QVL_OK);
  CHECK(qvl_causal_worklist(1, &many, &one, &one, 64, 64, 64, 1, 256, &rows, nullptr, 0, &n, &p, &j) != QVL_OK);
  CHECK(qvl_causal_worklist(-1, &one, &one, &one, 8, 8, 64, 1, 256, &rows, nullptr, 0, &n, &p, &j) != QVL_OK);
  CHECK(qvl_causal_worklist(0, nullptr, nullptr, nullptr, 8, 8, 64, 1, 256, &rows, nullptr, 0, &n, &p, &j) == QVL_OK && n == 0 && j == 0);
  CHECK(qvl_last_error()[0] != 0);
  printf("decoder sanitizer driver: %d lists, %d failures\n", cases, failures);
  return failures ? 1 : 0;
}
