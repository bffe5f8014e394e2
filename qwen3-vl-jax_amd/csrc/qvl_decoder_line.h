// The streaming launch of the decode attention kernels (qvl_decode.hip: rows of a cache; qvl_paged_attn.hip: pages of a packed
// one): the key blocks of all sequences as one line that is cut into equal runs, and the join of a workgroup's four waves.
#pragma once
#include "qvl_decoder_core.h"

namespace qvl {

// A job of the streaming launch whose last block lies in this run and whose first does not: what its join needs.
struct SplitJob {
  int64_t token0;
  int rows, row0, first, parts;   // parts == 0: none
};

struct DecodeState {
  const int32_t* cu_q;
  const int64_t* k_start;   // NULL: 0
  const int32_t* k_len;
  const int32_t* cu_groups;
  const int64_t* prefix_start;
  const int32_t* prefix_len;
  int n_seqs, n_groups;
  int own_parts, own_chunk, prefix_parts, prefix_chunk, prefix_tiles;   // with prefixes: parts of so many keys each
  SplitJob* split;                                                      // streaming: [runs]
  int slot_rows;                                                        // streaming: rows a part's slot has
  int tile;                                                             // rows of a tile: 32, or 16 (FewWave)
  int shift = 5;                                                        // streaming: 2^shift keys a block of the line
  int pad = 0;                                                          // blocks that a job counts for beside its own
  int keep = -1;                                                        // blocks of a job that stays whole; -1: a run's share
};

// A barrier for what lies in LDS alone: __syncthreads also waits until stores to memory are through (3 us of a launch of 20).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// LDS of the join below, over the tiles (tiles of ROWS rows).
template <typename T, int D, int ROWS = 32> constexpr int kJoinBytes = 4 * ROWS * (D * 4 + 16);

// The four waves' results of the same rows joined in LDS and written: to the output, or as
// a part, row r of which is row at(r) of the part buffers. `ka`: the first key of the range the waves covered.
template <typename T, int D, typename W, typename F>
__device__ __forceinline__ void join_waves(const AttnParams& P, const Unit& u, W& w, char* smem, int first_row, int ka, bool part,
                                           F&& at) {
  // Rows of kPitch bytes: 16 more than a row, so that neither rows nor chunks meet in a bank and every address is one lane's
  // base and a constant (each line of code that runs once costs a workgroup some 800 cycles of fetching it).
  constexpr int kC = D / 4, kPitch = D * 4 + 16, kWave = W::kRows * kPitch;
  __shared__ float sm[4][32], sl[4][32];
  __shared__ int slim[32];
  const int lane = threadIdx.x & 63, lr = lane & (W::kRows - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = min(W::kRows, u.rows - first_row);
  const float lw = w.core.row_sum();
  if (lane < W::kRows) {
    sm[wave][lr] = w.m;
    sl[wave][lr] = lw;
    slim[lr] = w.lim;
  }
  lds_barrier();                               // every wave is past its tiles
  if (lr < n) {
    char* row = smem + wave * kWave + lr * kPitch;
    w.core.each4([&](int d, const f32x4& x) { *reinterpret_cast<f32x4*>(row + d * 4) = x; });
  }
  lds_barrier();
  for (int i = threadIdx.x; i < n * kC; i += 256) {
    const int r = i / kC, c = i % kC;
    float M = sm[0][r];
#pragma unroll
    for (int x = 1; x < 4; ++x) M = fmaxf(M, sm[x][r]);
    const float shift = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = __builtin_amdgcn_exp2f(sm[x][r] - shift);
      l += f * sl[x][r];
      // a wave that saw none of the row's keys has zeros; one whose maximum is far below the others' may hold infinities
      const f32x4 o = *reinterpret_cast<const f32x4*>(smem + x * kWave + r * kPitch + c * 16);
      if (f != 0.f) acc += f * o;
    }
    const bool sees = slim[r] > ka;
    if (part) {
      const int64_t a = at(r);
      *reinterpret_cast<f32x4*>(P.part_o + a * D + c * 4) = acc;
      if (c == 0) P.part_ml[a] = part_state(M, l, sees);
    } else {
      const float inv = 1.0f / l;
      store4<T>(out_row<T, D>(P, u, first_row + r), c * 4, sees ? acc * inv : f32x4{0.f, 0.f, 0.f, 0.f});
    }
  }
  lds_barrier();                               // the tiles may be written again
}

// The token range of sequences [s0, s1), empty where it is none of [0, n_tokens).
__device__ __forceinline__ int64_t tokens_of(const AttnParams& P, const DecodeState& S, int s0, int s1, int64_t& first) {
  const int64_t a = S.cu_q ? S.cu_q[s0] : s0, b = S.cu_q ? S.cu_q[s1] : s1;
  first = a;
  return a < 0 || b > P.n_tokens || b < a ? 0 : b - a;
}

__device__ __forceinline__ bool bad_keys(const AttnParams& P, int64_t start, int len) {
  return len < 0 || len > kItemMaxLen || start < 0 || start > P.kv_rows - len;
}

// ---------------------------------------------------------------------------------------------
// streaming
// ---------------------------------------------------------------------------------------------
// What the line holds of a sequence: its jobs (tiles of S.tile rows), and the blocks of 2^S.shift keys of each, one where there is
// nothing to read, for the rows' zeros (or NaN), and S.pad before them.
struct Sequence {
  int64_t token0, start;
  int tokens, len, jobs, blocks;
};

__device__ __forceinline__ Sequence sequence_of(const AttnParams& P, const DecodeState& S, int seq) {
  Sequence q;
  q.tokens = (int)tokens_of(P, S, seq, seq + 1, q.token0);
  q.start = S.k_start ? S.k_start[seq] : 0;   // (a page table has rows of its own)
  q.len = S.k_len[seq];
  q.jobs = (int)(((int64_t)q.tokens * P.group + S.tile - 1) / S.tile);
  q.blocks = (bad_keys(P, q.start, q.len) ? 1 : max((int)((q.len + (1ll << S.shift) - 1) >> S.shift), 1)) + S.pad;
  return q;
}

// Exclusive sums of v over the workgroup, in excl[0..256] (excl[256]: the total).
__device__ __forceinline__ void scan256(int64_t v, int64_t* excl) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ int64_t waves[4];
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += waves[i];
  excl[threadIdx.x + 1] = x;
  if (threadIdx.x == 0) excl[0] = 0;
  __syncthreads();
}

__device__ __forceinline__ Sequence uniform(Sequence q) {
  q.token0 = uniform(q.token0);
  q.start = uniform(q.start);
  q.tokens = uniform(q.tokens);
  q.len = uniform(q.len);
  q.jobs = uniform(q.jobs);
  q.blocks = uniform(q.blocks);
  return q;
}

// Where run i of n begins: an equal share of the line, moved to a job's end where the job is no longer than a share (or a
// block for each wave), so that short jobs stay whole. `base`: where the jobs of the sequence that the share begins in do.
__device__ __forceinline__ int64_t share(int64_t total, int i, int n) { return total / n * i + total % n * i / n; }
__device__ __forceinline__ int64_t run_start(int64_t total, int64_t pos, int n, int64_t base, int blocks, int pad, int keep) {
  const int in = (int)((pos - base) % blocks);
  if (in <= pad) return pos - in;             // no run begins inside the padding
  return blocks > max((int64_t)4, keep < 0 ? total / n : keep) ? pos : pos - in + (2 * in < blocks ? 0 : blocks);
}

// The line as one workgroup sees it. Up to 64 sequences: one a lane, and each wave finds its way without the others. More: a
// run of `per` sequences a thread, summed up in LDS, then one run again.
struct Line {
  int64_t excl[257], work[257];
  int hit;
};

__device__ __forceinline__ void locate(const AttnParams& P, const DecodeState& S, Line& L, int64_t pos, int per, int& seq, int64_t& base) {
  if (L.excl[threadIdx.x] <= pos && pos < L.excl[threadIdx.x + 1]) L.hit = threadIdx.x;
  __syncthreads();
  const int run = L.hit;
  seq = run * per;
  base = L.excl[run];
  if (per == 1) {                              // a thread's run is one sequence (96 of 300 keys in pages: 20.4 us, not 22.6)
    seq = uniform(seq);
    base = uniform(base);
    __syncthreads();
    return;
  }
  __syncthreads();
  const int s = seq + (int)threadIdx.x;
  int64_t mine = 0;
  if ((int)threadIdx.x < per && s < S.n_seqs) {
    const Sequence q = sequence_of(P, S, s);
    mine = (int64_t)q.jobs * q.blocks;
  }
  scan256(mine, L.work);
  if (L.work[threadIdx.x] <= pos - base && pos - base < L.work[threadIdx.x + 1]) L.hit = threadIdx.x;
  __syncthreads();
  seq = uniform(seq + L.hit);
  base = uniform(base + L.work[L.hit]);
  __syncthreads();
}

// The run [pos, end) of workgroup `run` of at most `runs`, how many there are (n), and the sequence that pos lies in, whose
// jobs begin at `base`. pos >= end: nothing to do.
__device__ __forceinline__ void find_run(const AttnParams& P, const DecodeState& S, Line& L, int run, int runs, int64_t& total, int& n,
                                         int64_t& pos, int64_t& end, int& seq, int64_t& base, Sequence& q) {
  const int lane = threadIdx.x & 63;
  pos = end = 0;
  if (S.n_seqs <= 64) {
    Sequence mine{};
    if (lane < S.n_seqs) mine = sequence_of(P, S, lane);
    // in 32 bits where the line is that short (2^30 blocks: 2^35 keys): a few instructions for each division, not a hundred,
    // and code that runs once is paid by its length
    const int own = (int)min((int64_t)mine.jobs * mine.blocks, (int64_t)1 << 25);
    int x = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d);
      x += lane >= d ? y : 0;
    }
    const uint32_t sum = (uint32_t)__builtin_amdgcn_readlane(x, 63);
    if (__builtin_amdgcn_ballot_w64((int64_t)mine.jobs * mine.blocks != own) == 0) {
      total = sum;
      n = (int)min((uint32_t)runs, sum);   // no run of a split job is empty
      if (run >= n) return;
      const uint32_t each = sum / (uint32_t)n, rest = sum - each * (uint32_t)n;
      auto start = [&](int i, int& at) {
        const uint32_t p = each * (uint32_t)i + rest * (uint32_t)i / (uint32_t)n;
        at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64((uint32_t)(x - own) <= p && p < (uint32_t)x)) - 1;
        if (i == n) return (int64_t)sum;
        const uint32_t blocks = (uint32_t)__builtin_amdgcn_readlane(mine.blocks, at);
        const uint32_t in = (p - (uint32_t)__builtin_amdgcn_readlane(x - own, at)) % blocks;
        if (in <= (uint32_t)S.pad) return (int64_t)(p - in);
        return (int64_t)(blocks > max(4u, S.keep < 0 ? each : (uint32_t)S.keep) ? p : p - in + (2 * in < blocks ? 0 : blocks));
      };
      int other = 0;
      end = start(run + 1, other);
      pos = start(run, seq);
      base = __builtin_amdgcn_readlane(x - own, seq);
      auto lane64 = [&](int64_t v) {
        return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), seq) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)v, seq));
      };
      q.token0 = lane64(mine.token0);
      q.start = lane64(mine.start);
      q.tokens = __builtin_amdgcn_readlane(mine.tokens, seq);
      q.len = __builtin_amdgcn_readlane(mine.len, seq);
      q.jobs = __builtin_amdgcn_readlane(mine.jobs, seq);
      q.blocks = __builtin_amdgcn_readlane(mine.blocks, seq);
      return;
    }
  }
  const int per = (S.n_seqs + 255) / 256;
  int64_t mine = 0;
  for (int s = threadIdx.x * per; s < min((int)(threadIdx.x + 1) * per, S.n_seqs); ++s) {
    const Sequence one = sequence_of(P, S, s);
    mine += (int64_t)one.jobs * one.blocks;
  }
  scan256(mine, L.excl);
  total = uniform(L.excl[256]);
  n = (int)min((int64_t)runs, total);
  if (run >= n) return;
  auto start = [&](int i, int& at, int64_t& first) {
    const int64_t p = share(total, i, n);
    if (p >= total) return total;
    locate(P, S, L, p, per, at, first);
    return run_start(total, p, n, first, uniform(sequence_of(P, S, at).blocks), S.pad, S.keep);
  };
  int other = 0;
  int64_t other_base = 0;
  pos = start(run, seq, base);
  end = start(run + 1, other, other_base);
  q = uniform(sequence_of(P, S, seq));
}

}  // namespace qvl
