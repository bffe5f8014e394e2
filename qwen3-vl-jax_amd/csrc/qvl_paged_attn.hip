// Attention of a few new tokens of each sequence over its pages of the 4-bit cache (qvl_paged.h), the sequences' state read on the
// device: bound by reading the pages once, 136 bytes a key and head of 128, K and V together (bf16 rows: 512).
//
// The launch is qvl_decode.hip's stream: the key blocks of all sequences are one line that is cut into equal runs, a workgroup a run
// and key/value head, and a second launch joins jobs that cross runs. A wave takes a block of 32 keys at a time and up to 16 rows
// (token, query head). S^T = K Q^T by v_mfma_f32_16x16x32_bf16 puts a row in a lane (column lane % 16) with keys
// 4 (lane / 16) + i of each half of the block; an instruction's 32 dims lie in one group, so a group's sum takes the key's
// scale in fp32. O^T = V^T P^T takes the weights as they lie, times V's scale of the key and group, rounded to bf16.
// K and V come from memory in the lanes that use them (16 bytes a lane and 16 keys, whole lines): no LDS, no barrier, and the
// codes become bf16 by one conversion for two of them. V's are nibbles of one token in a row; four bit operations turn 16 of
// two tokens into pairs.
//
// fp32: q and the weights are split in three bf16 parts (24 bits); the codes are exact, so three products give the fp32 one.
#include "qvl_decoder.h"
#include "qvl_decoder_line.h"
#include "qvl_paged.h"

namespace qvl {

// x rounded to `PARTS` bf16 parts, the largest first (PARTS 3: exact).
template <int PARTS, int N> __device__ __forceinline__ void bf16_parts(const float (&x)[N], bf16x8 (&out)[PARTS]) {
  static_assert(N == 8, "an operand");
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pack_bf16x2(rest[2 * j], rest[2 * j + 1]);
      if (p + 1 < PARTS) {
        rest[2 * j] -= bf16_lo(w[j]);
        rest[2 * j + 1] -= bf16_hi(w[j]);
      }
    }
    out[p] = __builtin_bit_cast(bf16x8, w);
  }
}

// byte `I` of w: two codes as bf16
template <int I> __device__ __forceinline__ uint32_t numbers(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, I));
}
__device__ __forceinline__ bf16x8 numbers8(uint32_t w) {
  return __builtin_bit_cast(bf16x8, u32x4{numbers<0>(w), numbers<1>(w), numbers<2>(w), numbers<3>(w)});
}

__device__ __forceinline__ f32x4 product(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T, int D> struct PagedCore {
  using B = PageBlock<D>;
  static constexpr int kRows = 16, kParts = std::is_same<T, float>::value ? 3 : 1, kG = B::kGroups, kSteps = D / 32, kDB = D / 16;
  static constexpr int kWords = D / 32;        // words of K, of V and of either's scales that a lane has of 16 keys
  bf16x8 q[kSteps][kParts];                    // step 2 g + s (D = 64: s): the dims of group g in piece 2 quad + s
  f32x4 o[kDB];                                // D = 128: dims 64 (db / 4) + 4 r + db % 4, r = 4 quad + i; D = 64: 4 r + db
  float l;

  static __device__ __forceinline__ int quad() { return (threadIdx.x & 63) >> 4; }
  __device__ __forceinline__ void init(const char* qrow) {
    constexpr int E = D / 16;
    const T* x = reinterpret_cast<const T*>(qrow);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int d = (2 * quad() + s) * E;
      float lo[E], hi[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        lo[j] = (float)x[d + j];
        hi[j] = (float)x[D / 2 + d + j];
      }
      if constexpr (D == 128) {
        bf16_parts<kParts>(lo, q[s]);
        bf16_parts<kParts>(hi, q[2 + s]);
      } else {
        const float both[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        bf16_parts<kParts>(both, q[s]);
      }
    }
#pragma unroll
    for (auto& y : o) y = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
  }
  __device__ __forceinline__ void rescale(float a) {
#pragma unroll
    for (auto& y : o) y *= a;
    l *= a;
  }
  __device__ __forceinline__ float row_sum() const {
    const float x = l + __shfl_xor(l, 16);
    return x + __shfl_xor(x, 32);
  }
  template <typename F> __device__ __forceinline__ void each4(F&& f) const {
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) f(64 * g + 16 * quad() + 4 * i, f32x4{o[4 * g][i], o[4 * g + 1][i], o[4 * g + 2][i], o[4 * g + 3][i]});
  }

  // What a lane holds of 16 keys.
  struct Keys {
    uint32_t k[kWords], v[kWords], ks[kWords], vs[kWords];
    static __device__ __forceinline__ void load(uint32_t (&w)[kWords], const char* p) {
      if constexpr (kWords == 4) *reinterpret_cast<u32x4*>(w) = *reinterpret_cast<const u32x4*>(p);
      else *reinterpret_cast<u32x2*>(w) = *reinterpret_cast<const u32x2*>(p);
    }
    __device__ __forceinline__ void load(const char* block) {
      const int r = threadIdx.x & 15;
      load(k, block + B::k_piece(r, 2 * quad()));
      load(v, block + B::v_word(4 * quad(), r));
      load(ks, block + B::k_scale(4 * quad()));
      load(vs, block + B::v_scale(4 * quad()));
    }
    // scale of token i of the quad, group g
    static __device__ __forceinline__ float scale(const uint32_t (&w)[kWords], int i, int g) {
      const int at = i * kG + g;
      return at & 1 ? bf16_hi(w[at >> 1]) : bf16_lo(w[at >> 1]);
    }
  };

  __device__ __forceinline__ f32x4 scores(const Keys& x) const {
    f32x4 s;
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const bf16x8 k = numbers8(x.k[kG * st + g]);
#pragma unroll
        for (int p = kParts - 1; p >= 0; --p) acc = product(k, q[2 * g + st][p], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float sc = Keys::scale(x.ks, i, g);
        s[i] = g == 0 ? sc * acc[i] : __builtin_fmaf(sc, acc[i], s[i]);
      }
    }
    return s;
  }

  // bytes whose low nibble is a code of a and whose high one is b's of the same dim: the even dims, the odd ones
  static __device__ __forceinline__ uint32_t even_pairs(uint32_t a, uint32_t b) { return (a & 0x0f0f0f0fu) | (b << 4 & 0xf0f0f0f0u); }
  static __device__ __forceinline__ uint32_t odd_pairs(uint32_t a, uint32_t b) { return (a >> 4 & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u); }

  // o += V^T P^T of two blocks of 16 keys, weights w (scaled below); `seen`: a bit for each key that the row sees, where EDGE
  template <bool EDGE> __device__ __forceinline__ void values(const Keys (&x)[2], const f32x4 (&w)[2], uint32_t seen) {
    uint32_t even[2][2], odd[2][2];            // [block][tokens (0, 1), (2, 3)]
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      l += (w[b][0] + w[b][1]) + (w[b][2] + w[b][3]);
      if constexpr (D == 128) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          even[b][h] = even_pairs(x[b].v[2 * h], x[b].v[2 * h + 1]);
          odd[b][h] = odd_pairs(x[b].v[2 * h], x[b].v[2 * h + 1]);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {          // two tokens a word: the second's codes are 16 bits on
          even[b][h] = even_pairs(x[b].v[h], x[b].v[h] >> 16);
          odd[b][h] = odd_pairs(x[b].v[h], x[b].v[h] >> 16);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      float p[8];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[4 * b + i] = w[b][i] * Keys::scale(x[b].vs, i, g);
          if (EDGE) p[4 * b + i] = (seen >> (4 * b + i)) & 1 ? p[4 * b + i] : 0.f;   // an unseen key's scale may be anything
        }
      bf16x8 pw[kParts];
      bf16_parts<kParts>(p, pw);
      auto add = [&](int db, uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, u32x4{a0, a1, b0, b1});
#pragma unroll
        for (int q = kParts - 1; q >= 0; --q) o[db] = product(v, pw[q], o[db]);
      };
      if (g == 0) {                            // bytes 0 and 1: dims 4 r + (0, 1), (2, 3) of the first group
        add(0, numbers<0>(even[0][0]), numbers<0>(even[0][1]), numbers<0>(even[1][0]), numbers<0>(even[1][1]));
        add(1, numbers<0>(odd[0][0]), numbers<0>(odd[0][1]), numbers<0>(odd[1][0]), numbers<0>(odd[1][1]));
        add(2, numbers<1>(even[0][0]), numbers<1>(even[0][1]), numbers<1>(even[1][0]), numbers<1>(even[1][1]));
        add(3, numbers<1>(odd[0][0]), numbers<1>(odd[0][1]), numbers<1>(odd[1][0]), numbers<1>(odd[1][1]));
      } else {
        add(4, numbers<2>(even[0][0]), numbers<2>(even[0][1]), numbers<2>(even[1][0]), numbers<2>(even[1][1]));
        add(5, numbers<2>(odd[0][0]), numbers<2>(odd[0][1]), numbers<2>(odd[1][0]), numbers<2>(odd[1][1]));
        add(6, numbers<3>(even[0][0]), numbers<3>(even[0][1]), numbers<3>(even[1][0]), numbers<3>(even[1][1]));
        add(7, numbers<3>(odd[0][0]), numbers<3>(odd[0][1]), numbers<3>(odd[1][0]), numbers<3>(odd[1][1]));
      }
    }
  }
};

// One wave: 16 rows over blocks of 32 keys.
template <typename T, int D> struct PagedWave : RowState<PagedCore<T, D>> {
  using C = PagedCore<T, D>;
  using Keys = typename C::Keys;
  using RowState<C>::core;
  using RowState<C>::lim;
  using RowState<C>::lim_lo;

  // 32 keys from kb on; bad: which of the two blocks of 16 lies in a page outside the cache (its keys' scores are NaN)
  template <bool EDGE> __device__ __forceinline__ void step(const Keys (&x)[2], int kb, float scale, int bad) {
    f32x4 s[2];
    uint32_t seen = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = core.scores(x[b]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[b][i] *= scale;
        if (bad & (1 << b)) s[b][i] = NAN;
        if (EDGE) {
          const bool in = kb + 16 * b + 4 * C::quad() + i < lim;
          seen |= (in ? 1u : 0u) << (4 * b + i);
          s[b][i] = in ? s[b][i] : -INFINITY;
        }
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    this->cover(mx);
    const float shift = this->shift();
    f32x4 w[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[b][i] = __builtin_amdgcn_exp2f(s[b][i] + shift);
    core.template values<EDGE>(x, w, seen);
  }
};

// Where a wave's blocks of 16 keys lie: of its next 32 steps' 64 blocks, one a lane.
template <int D> struct PageWalk {
  const Pages& pages;
  int64_t seq;
  int kvh, last;                               // the last block of 16 that holds a key
  const char* at;                              // the lane's block; NULL: its page is none
  __device__ __forceinline__ void look(int t) {   // steps t, t + 4, ..., of two blocks each
    const int lane = threadIdx.x & 63;
    const int b = min(2 * (t + 4 * (lane >> 1)) + (lane & 1), last);
    const int page = pages.page(seq, b >> (pages.shift - 4));
    at = page < 0 ? nullptr : pages.block<D>(page, kvh, b << 4);
  }
  __device__ __forceinline__ const char* block(int i) const {
    const uint64_t p = (uint64_t)at;
    return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)p, i));
  }
};

// A workgroup's four waves over blocks [t0, t1) of 32 keys, every fourth to a wave, a step's loads one step ahead.
template <typename T, int D>
__device__ __forceinline__ void paged_run(const AttnParams& P, const Pages& pages, int seq, const Unit& u, PagedWave<T, D>& w, int t0, int t1) {
  using Keys = typename PagedCore<T, D>::Keys;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int t = t0 + wave;
  if (t >= t1) return;
  PageWalk<D> walk{pages, seq, u.kvh, (u.len - 1) >> 4, nullptr};
  Keys x[2][2];
  int bad[2], n = 0;
  auto fetch = [&](int t, Keys (&y)[2], int& out) {
    if ((n & 31) == 0) walk.look(t);
    out = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const char* block = walk.block(2 * (n & 31) + b);
      if (block) y[b].load(block);
      else {
        out |= 1 << b;
        y[b] = Keys{};
      }
    }
    ++n;
  };
  auto use = [&](int t, const Keys (&y)[2], int out) {
    if (t * 32 + 32 > w.lim_lo) w.template step<true>(y, t * 32, P.scale, out);
    else w.template step<false>(y, t * 32, P.scale, out);
  };
  fetch(t, x[0], bad[0]);
  for (;;) {
    if (t + 4 < t1) fetch(t + 4, x[1], bad[1]);
    use(t, x[0], bad[0]);
    if ((t += 4) >= t1) break;
    if (t + 4 < t1) fetch(t + 4, x[0], bad[0]);
    use(t, x[1], bad[1]);
    if ((t += 4) >= t1) break;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void paged_stream_kernel(AttnParams P, DecodeState S, Pages pages) {
  using W = PagedWave<T, D>;
  __shared__ __attribute__((aligned(16))) char smem[kJoinBytes<T, D, 16>];
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
    const int64_t into = pos - base;
    const int job = (int)(into / blocks), b0 = (int)(into % blocks);
    const int b1 = (int)min((int64_t)blocks, b0 + (end - pos));
    const Unit u{nullptr, nullptr, q.len, q.len - q.tokens + 1, q.token0, q.tokens * P.group, job * W::kRows, kvh};
    const int n_rows = min(W::kRows, u.rows - u.row0);
    const bool whole = b0 == 0 && b1 == blocks;
    if (bad_keys(P, 0, u.len)) {
      for (int i = threadIdx.x; i < n_rows * (D / 4); i += 256)
        store4<T>(out_row<T, D>(P, u, u.row0 + i / (D / 4)), i % (D / 4) * 4, f32x4{NAN, NAN, NAN, NAN});
    } else {
      W w;
      w.init(P, u, u.row0);
      paged_run<T, D>(P, pages, seq, u, w, b0, min(b1, (u.len + 31) >> 5));
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

// Part p of a split job, as in qvl_decode.hip.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnParams P, DecodeState S) {
  const SplitJob j = S.split[blockIdx.x];
  if (j.parts == 0) return;
  const int kvh = blockIdx.y;
  const Unit u{nullptr, nullptr, 0, 0, j.token0, j.rows, j.row0, kvh};
  const int n = min(S.tile, j.rows - j.row0), per = (n + gridDim.z - 1) / gridDim.z, r0 = blockIdx.z * per;
  join_parts<T, D>(P, r0, min(r0 + per, n), j.parts,
                   [&](int r, int p) { return ((int64_t)(2 * (j.first + p) + (p == 0)) * P.hkv + kvh) * S.slot_rows + r; },
                   [&](int r) { return out_row<T, D>(P, u, j.row0 + r); });
}

// How a launch is laid out: from the sizes alone, so that the workspace can be told beforehand.
struct PagedPlan {
  int runs, slot_rows;
  size_t part_rows, split_bytes;
};

static int paged_plan(const char* what, int64_t n_tokens, int64_t n_seqs, int64_t max_len, int32_t num_heads, int32_t num_kv_heads, PagedPlan& D) {
  if (n_tokens < 0 || n_seqs < 0 || max_len < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_seqs > 65535 || max_len > kItemMaxLen) return set_error(QVL_ERR_UNSUPPORTED, "%s: sequences or lengths", what);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(QVL_ERR_INVALID_ARG, "%s: %d heads over %d key/value heads", what, num_heads, num_kv_heads);
  const int64_t rows = n_tokens * (num_heads / num_kv_heads);
  if (num_heads > kItemMaxHeads || n_tokens > kItemMaxLen || rows > kItemMaxLen) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  D = PagedPlan{};
  const int64_t slots = (int64_t)gemm_device_cus() * 2;
  const int64_t own_rows = (rows + std::max<int64_t>(n_seqs, 1) - 1) / std::max<int64_t>(n_seqs, 1);
  const int64_t tiles = std::max<int64_t>((own_rows + 15) / 16, 1), jobs = n_seqs * tiles, blocks = jobs * ((max_len + 31) / 32);
  D.runs = (int)std::max<int64_t>(std::min(slots / num_kv_heads, std::max((blocks + 3) / 4, jobs)), 1);
  D.slot_rows = (int)std::min<int64_t>(16, std::max<int64_t>(rows, 1));
  D.part_rows = (size_t)D.runs * num_kv_heads * 2 * D.slot_rows;
  D.split_bytes = round_up(D.runs * sizeof(SplitJob), 16);
  return QVL_OK;
}

static size_t workspace_bytes_of(const PagedPlan& D, int32_t head_dim) { return D.split_bytes + D.part_rows * ((size_t)head_dim + 2) * sizeof(float); }

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_paged_attention_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t max_len, int32_t num_heads, int32_t num_kv_heads,
                                       int32_t head_dim, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "paged_attention_workspace_size: bytes is NULL");
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "paged_attention_workspace_size: head_dim=%d", head_dim);
  PagedPlan plan;
  QVL_TRY_RC(paged_plan("paged_attention_workspace_size", n_tokens, n_seqs, max_len, num_heads, num_kv_heads, plan));
  *bytes = workspace_bytes_of(plan, head_dim);
  return QVL_OK;
}

int qvl_paged_attention(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* cache, int64_t n_pages,
                        int32_t page_rows, const int32_t* page_table, int64_t table_width, int64_t table_stride, const int32_t* cu_q,
                        int64_t n_seqs, const int32_t* k_len, int64_t max_len, float scale, void* out, int64_t out_row, int64_t out_head,
                        int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, void* workspace,
                        size_t workspace_bytes) {
  AttnParams P{};
  Pages pages;
  QVL_TRY_RC(pages_of("paged_attention", cache, n_pages, page_rows, page_table, table_width, table_stride, n_seqs, num_kv_heads, head_dim, pages));
  QVL_TRY_RC(attn_params("paged_attention", dtype, q, q_row, q_head, nullptr, 0, 0, nullptr, 0, 0, 0, out, out_row, out_head, n_tokens,
                         num_heads, num_kv_heads, head_dim, scale, P));
  PagedPlan plan;
  QVL_TRY_RC(paged_plan("paged_attention", n_tokens, n_seqs, max_len, num_heads, num_kv_heads, plan));
  if (!cu_q && n_tokens != n_seqs) return set_error(QVL_ERR_INVALID_ARG, "paged_attention: %lld tokens of %lld sequences without cu_q", (long long)n_tokens, (long long)n_seqs);
  if (n_tokens == 0 || n_seqs == 0) return QVL_OK;
  if (!k_len) return set_error(QVL_ERR_INVALID_ARG, "paged_attention: NULL pointer");
  if ((uintptr_t)k_len % 4 || (uintptr_t)cu_q % 4) return set_error(QVL_ERR_MISALIGNED, "paged_attention: the sequences' state");
  const size_t need = workspace_bytes_of(plan, head_dim);
  if (workspace_bytes < need || !workspace) return set_error(QVL_ERR_WORKSPACE, "paged_attention: workspace %zu < %zu", workspace_bytes, need);
  if ((uintptr_t)workspace % 16) return set_error(QVL_ERR_MISALIGNED, "paged_attention: workspace");
  P.kv_rows = (int64_t)pages.width << pages.shift;   // of a sequence: it has no more rows than its line of the table names
  P.part_o = (float*)((char*)workspace + plan.split_bytes);
  P.part_ml = (f32x2*)(P.part_o + plan.part_rows * head_dim);
  DecodeState S{};
  S.cu_q = cu_q;
  S.k_len = k_len;
  S.n_seqs = (int)n_seqs;
  S.split = (SplitJob*)workspace;
  S.slot_rows = plan.slot_rows;
  S.tile = 16;
  QVL_ATTN_LAUNCH(paged_stream_kernel, dim3((unsigned)(plan.runs * num_kv_heads)), P, S, pages);
  QVL_TRY_RC(check_launch("paged_stream"));
  if (plan.runs == 1) return QVL_OK;
  QVL_ATTN_LAUNCH(paged_join_kernel, dim3((unsigned)plan.runs, (unsigned)num_kv_heads, (unsigned)plan.slot_rows), P, S);
  return check_launch("paged_join");
}

}  // extern "C"
