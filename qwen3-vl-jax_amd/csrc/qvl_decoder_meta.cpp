// GPU-free host side of the decoder entries: the rotation table and the causal work list. Plain C++ (no HIP), so that
// it also builds for the CPU sanitizer run.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <functional>
#include <map>
#include <new>
#include <queue>
#include <vector>

#include "qvl_decoder_items.h"

using namespace qvl;

namespace {

struct Job {
  int64_t seq;      // -1: none (padding of a queue)
  int32_t row0, head, slot;
  int32_t t0, t1;   // key tiles
  int32_t steps() const { return t1 - t0; }
};

constexpr int64_t kMaxJobs = 1 << 22;   // 5 10^8 rows

// Greedy time of jobs, longest first, on `slots` workgroup slots.
double makespan(std::vector<double> cost, int64_t slots) {
  std::sort(cost.begin(), cost.end(), std::greater<double>());
  std::priority_queue<double, std::vector<double>, std::greater<double>> free;
  for (int64_t s = 0; s < slots; ++s) free.push(0.0);
  double end = 0;
  for (double c : cost) {
    const double t = free.top() + c;
    free.pop();
    free.push(t);
    end = std::max(end, t);
  }
  return end;
}

// What the kernel of a tile height does with key tiles: workgroup slots, and in microseconds a step (one key tile of 64, fp32 32,
// by the tile's rows) with every slot busy, one where each compute unit has a single workgroup, what a job costs beside its
// steps, and what a cut costs: the join's launch, and each part's rows written and joined. Fitted on MI355X (head_dim 128; 64
// takes 0.6 of a step).
struct Kernel {
  int64_t slots, cus;
  double step, alone, job, join, part;
};

Kernel kernel_of(int32_t tile_rows, int32_t dtype, int32_t head_dim, int64_t n_cus) {
  const double half = head_dim == 64 ? 0.6 : 1.0;
  if (dtype == QVL_DTYPE_F32) return {2 * n_cus, n_cus, 8.5 * half, 4.3 * half, 2.5, 5.0, 0.03 * half};
  if (tile_rows == 256) return {n_cus, n_cus, 1.55 * half, 1.55 * half, 9.0, 5.0, 0.06 * half};
  return {(head_dim == 64 ? 3 : 2) * n_cus, n_cus, 1.75 * half, 1.25 * half, 4.5, 5.0, 0.03 * half};
}

// Where the jobs do not fill the slots evenly (few rows over many keys, or a prompt of a few tiles whose last one is the
// longest), their keys are cut: those of a sequence every `length` steps or a little less, so that its longest tile's parts are
// alike, and all its tiles at the same keys, which their workgroups then read together. (Cut where a slot's share ends, wherever
// that was, the slots came out even and the time no better: 278 us against 269 with every key read from further away.)
constexpr int32_t kMinPart = 4;

std::vector<Job> cut(const std::vector<Job>& jobs, const std::vector<int32_t>& longest, int32_t length) {
  std::vector<Job> out;
  for (const Job& j : jobs) {
    const int32_t most = longest[j.seq], n = std::max((most + length - 1) / length, 1), each = std::max((most + n - 1) / n, kMinPart);
    Job one = j;
    for (; j.t1 - one.t0 >= each + kMinPart; one.t0 = one.t1) {
      one.t1 = one.t0 + each;
      out.push_back(one);
    }
    one.t1 = j.t1;
    out.push_back(one);
  }
  return out;
}

bool whole(const Job& piece, const std::vector<Job>& pieces, size_t k) {
  const auto same = [&](const Job& o) { return o.seq == piece.seq && o.row0 == piece.row0 && o.head == piece.head; };
  return !(k > 0 && same(pieces[k - 1])) && !(k + 1 < pieces.size() && same(pieces[k + 1]));
}

// Jobs whole or in pieces, by the least modelled time, which is returned. Lengths tried: the mean load of a slot, and
// fractions and a little more of it.
double best_cut(std::vector<Job>& jobs, int64_t n_seqs, const Kernel& K) {
  double best = -1;
  std::vector<Job> kept;
  const auto attempt = [&](std::vector<Job> pieces) {
    std::vector<double> cost;
    double all = 0;
    int64_t parts = 0;
    const double step = (int64_t)pieces.size() <= K.cus ? K.alone : K.step;
    for (size_t k = 0; k < pieces.size(); ++k) {
      cost.push_back(pieces[k].steps() * step + K.job);
      all += cost.back();
      parts += !whole(pieces[k], pieces, k);
    }
    const double joined = parts ? K.join + K.part * parts : 0.0;
    if (best >= 0 && all / K.slots + joined >= best) return;
    const double t = makespan(std::move(cost), K.slots) + joined;
    if (best >= 0 && t >= best) return;
    best = t;
    kept.swap(pieces);
  };
  attempt(jobs);
  if ((int64_t)jobs.size() > 8 * K.slots) return best;   // (kept: the jobs as they were)
  std::vector<int32_t> longest((size_t)n_seqs);
  int64_t total = 0;
  for (const Job& j : jobs) {
    longest[j.seq] = std::max(longest[j.seq], j.steps());
    total += j.steps();
  }
  int32_t tried = 0;
  for (double f : {1.35, 1.2, 1.1, 1.0, 0.85, 0.75, 0.6, 0.5, 0.4, 0.334, 0.25, 0.167, 0.125}) {
    const int32_t length = std::max((int32_t)std::ceil((double)total / K.slots * f), kMinPart);
    if (length == tried) continue;
    tried = length;
    std::vector<Job> pieces = cut(jobs, longest, length);
    if (pieces.size() != jobs.size()) attempt(std::move(pieces));
  }
  jobs.swap(kept);
  return best;
}

// Jobs dealt to 8 queues, one per XCD (the dispatcher gives workgroup k to XCD k % 8): the jobs of one sequence and
// key/value head go to one queue, whose L2 then holds their keys, the longest such group to the queue with least to do;
// where queues come out unlike, jobs of the fullest move to the emptiest. A queue's longest jobs come first; short queues
// are padded.
std::vector<Job> deal(const std::vector<Job>& jobs, const Kernel& K) {
  const int32_t beside = (int32_t)(K.job / K.step);
  if (jobs.empty()) return {};
  std::map<std::pair<int64_t, int32_t>, std::vector<Job>> by_group;
  for (const Job& j : jobs) by_group[{j.seq, j.head}].push_back(j);
  std::vector<std::pair<int64_t, std::vector<Job>*>> groups;
  for (auto& g : by_group) {
    int64_t w = 0;
    for (const Job& j : g.second) w += j.steps() + beside;
    groups.push_back({w, &g.second});
  }
  std::stable_sort(groups.begin(), groups.end(),
                   [](const std::pair<int64_t, std::vector<Job>*>& a, const std::pair<int64_t, std::vector<Job>*>& b) { return a.first > b.first; });
  std::array<std::vector<Job>, kAttnQueues> queue;
  std::array<int64_t, kAttnQueues> load{};
  int64_t all = 0;
  for (auto& g : groups) {
    const size_t q = std::min_element(load.begin(), load.end()) - load.begin();
    load[q] += g.first;
    all += g.first;
    queue[q].insert(queue[q].end(), g.second->begin(), g.second->end());
  }
  auto longer = [](const Job& a, const Job& b) { return a.steps() > b.steps(); };
  for (auto& q : queue) std::stable_sort(q.begin(), q.end(), longer);
  for (int round = 0; round < 64; ++round) {
    const size_t hi = std::max_element(load.begin(), load.end()) - load.begin();
    const size_t lo = std::min_element(load.begin(), load.end()) - load.begin();
    const int64_t half = (load[hi] - load[lo]) / 2;
    if (half <= all / 400) break;
    // every other job of the fullest queue, so that what is left and what moves are alike, up to half the difference
    std::vector<Job> keep, move;
    int64_t moved = 0;
    for (size_t k = 0; k < queue[hi].size(); ++k) {
      const Job& j = queue[hi][k];
      if (k % 2 == 1 && moved + j.steps() + beside <= half) {
        move.push_back(j);
        moved += j.steps() + beside;
      } else {
        keep.push_back(j);
      }
    }
    if (move.empty()) break;
    queue[hi].swap(keep);
    queue[lo].insert(queue[lo].end(), move.begin(), move.end());
    std::stable_sort(queue[lo].begin(), queue[lo].end(), longer);
    load[hi] -= moved;
    load[lo] += moved;
  }
  // The first workgroups go to one slot of each compute unit, the next to the second: those in reverse, so that a long job
  // shares its compute unit with a short one (1181 tokens, 16/8 heads of 128, fp32: 66 us and not 73).
  const int64_t cus = std::max<int64_t>(K.cus / kAttnQueues, 1);
  for (auto& q : queue)
    for (int64_t s = 1; s < K.slots / K.cus; s += 2)
      std::reverse(q.begin() + std::min<int64_t>(s * cus, q.size()), q.begin() + std::min<int64_t>((s + 1) * cus, q.size()));
  size_t longest = 0;
  for (auto& q : queue) longest = std::max(longest, q.size());
  std::vector<Job> out(longest * kAttnQueues, Job{-1, 0, 0, -1, 0, 0});
  for (size_t k = 0; k < out.size(); ++k)
    if (k / kAttnQueues < queue[k % kAttnQueues].size()) out[k] = queue[k % kAttnQueues][k / kAttnQueues];
  return out;
}

int causal_worklist(int64_t n_seqs, const int64_t* n_new, const int64_t* len, const int64_t* start, int32_t num_heads,
                    int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t n_cus, int32_t* tile_rows,
                    int32_t* items, int64_t capacity, int64_t* n_items, int64_t* n_parts, int64_t* n_joins) {
  if (!n_items || !n_parts || !n_joins || !tile_rows)
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: n_items / n_parts / n_joins / tile_rows is NULL");
  if (n_seqs < 0 || (n_seqs > 0 && (!n_new || !len || !start)))
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: sequences are NULL");
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: head_dim=%d (64 or 128)", head_dim);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: %d heads over %d key/value heads", num_heads, num_kv_heads);
  if (num_heads > kItemMaxHeads) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: num_heads=%d", num_heads);
  if (n_cus <= 0 || n_cus > 65536) return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: n_cus=%d", n_cus);
  if (*tile_rows != 0 && *tile_rows != 128 && *tile_rows != 256) return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: tile_rows=%d", *tile_rows);
  if (*tile_rows == 256 && dtype == QVL_DTYPE_F32) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: tiles of 256 rows are bf16 only");
  const int64_t group = num_heads / num_kv_heads;
  const int64_t step_keys = dtype == QVL_DTYPE_BF16 ? 64 : 32;
  std::vector<int64_t> q_first;
  int64_t q0 = 0, n_jobs = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    if (n_new[i] < 0 || len[i] < 0 || start[i] < 0 || start[i] > (int64_t)1 << 56)
      return set_error(QVL_ERR_INVALID_ARG, "causal_worklist: sequence %lld: %lld new, %lld keys from row %lld", (long long)i,
                       (long long)n_new[i], (long long)len[i], (long long)start[i]);
    if (len[i] > kItemMaxLen || q0 + n_new[i] > kItemMaxLen || n_new[i] * group > kItemMaxLen)
      return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: sequence %lld is too long", (long long)i);
    q_first.push_back(q0);
    q0 += n_new[i];
    n_jobs += (n_new[i] * group + kItemRows - 1) / kItemRows * num_kv_heads;
    if (n_jobs > kMaxJobs) return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: more than %lld tiles", (long long)kMaxJobs);
  }
  // the tile height (where the caller leaves it open) and the cut of least modelled time
  std::vector<Job> jobs;
  int32_t height = 0;
  Kernel kernel{};
  double best = 0;
  for (int32_t rows : {128, 256}) {
    if (*tile_rows ? rows != *tile_rows : rows == 256 && dtype == QVL_DTYPE_F32) continue;
    std::vector<Job> mine;
    for (int64_t i = 0; i < n_seqs; ++i)
      for (int64_t r = 0; r < n_new[i] * group; r += rows) {
        const int64_t last = (std::min(r + rows, n_new[i] * group) - 1) / group;
        const int64_t keys = std::max<int64_t>(std::min(len[i] - n_new[i] + 1 + last, len[i]), 0);
        const int32_t steps = (int32_t)((keys + step_keys - 1) / step_keys);
        for (int32_t h = 0; h < num_kv_heads; ++h) mine.push_back({i, (int32_t)r, h, -1, 0, steps});
      }
    const Kernel K = kernel_of(rows, dtype, head_dim, n_cus);
    const double t = best_cut(mine, n_seqs, K);
    if (kernel.slots == 0 || t < best) {
      best = t;
      kernel = K;
      height = rows;
      jobs.swap(mine);
    }
  }
  *tile_rows = height;
  // slots and joins of the tiles that are in pieces, which lie one after the other
  std::vector<Job> joins;
  int32_t slots = 0;
  for (size_t k = 0; k < jobs.size(); ++k) {
    if (whole(jobs[k], jobs, k)) continue;
    if (jobs[k].t0 == 0) joins.push_back({jobs[k].seq, jobs[k].row0, jobs[k].head, slots, 0, 0});
    ++joins.back().t1;
    jobs[k].slot = slots++;
  }
  std::vector<Job> list = deal(jobs, kernel);
  while (!list.empty() && list.back().seq < 0) list.pop_back();
  *n_items = (int64_t)list.size();
  *n_parts = slots;
  *n_joins = (int64_t)joins.size();
  if (!items) return QVL_OK;
  list.insert(list.end(), joins.begin(), joins.end());
  if (capacity < (int64_t)list.size())
    return set_error(QVL_ERR_INVALID_ARG, "causal_worklist capacity %lld < %zu", (long long)capacity, list.size());
  for (size_t k = 0; k < list.size(); ++k) {
    const Job& j = list[k];
    int32_t* it = items + kItemWords * k;
    memset(it, 0, kItemWords * sizeof(int32_t));
    if (j.seq < 0) continue;
    it[0] = (int32_t)q_first[j.seq];
    it[1] = (int32_t)n_new[j.seq];
    it[2] = (int32_t)len[j.seq];
    it[3] = j.row0;
    it[4] = j.head;
    it[5] = j.slot;
    it[6] = (int32_t)(uint32_t)(start[j.seq] & 0xffffffff);
    it[7] = (int32_t)(start[j.seq] >> 32);
    it[8] = j.t0;
    it[9] = j.t1;
  }
  return QVL_OK;
}

}  // namespace

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
                        int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t n_cus, int32_t* tile_rows,
                        int32_t* items, int64_t capacity, int64_t* n_items, int64_t* n_parts, int64_t* n_joins) {
  // (a list too long for the host's memory is an error like any other, not an exception through a C call)
  try {
    return causal_worklist(n_seqs, n_new, len, start, num_heads, num_kv_heads, head_dim, dtype, n_cus, tile_rows, items, capacity,
                           n_items, n_parts, n_joins);
  } catch (const std::bad_alloc&) {
    return set_error(QVL_ERR_UNSUPPORTED, "causal_worklist: out of host memory");
  }
}

}  // extern "C"
