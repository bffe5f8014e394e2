// Attention tiles of 256 rows (bf16): 64 rows a wave, two sets of 32, so that each K and V fragment read from LDS serves two
// products and each tile's bytes twice the rows of the 128-row units. One wave a SIMD with all 512 registers: matrix and
// vector work overlap within the wave, by the order they are issued in. A tile takes 3000 cycles, 2048 of them the matrix
// cores'; the units of 128 rows, two on a compute unit, 3400 for as many rows.
//
// A tile of 64 keys is four units, (set A, keys 0..31), (B, 0..31), (A, 32..63), (B, 32..63), each with its scores' products
// Q0..Q3, its weights and its products with V, P0..P3, D / 16 instructions a group. They are issued as
//   Q0  Q1  Q2  P0  Q3  P1  P2  P3
// and the 16 weights of each lane and unit, one by one, among Q1..P2: unit u's are complete when Pu begins, and while
// they are formed the matrix cores work on another unit. LDS reads stand a group before their use; the next tile's
// first K fragments are read during P3, from a third stage of the ring, so that no wait for LDS follows the barrier. The
// tile's DMAs stand apart, four products between two (one takes the CU's address unit long enough to hold the wave), and in
// the tile's first half, so that they are there when it ends.
//
// No running maximum: a row's weights are 2^(s - m) with m the largest score of its first tile, whatever comes later, so that
// the loop has no branch and no pass over the accumulators. fp32 sums lose nothing by that until they overflow. A part of a
// cut tile has to be joined besides: by 2^(m - M), which the exponential makes 0 below 2^-126, so that a sum held against an m
// so far below the others' M may not be large. Where a row's sum of weights, both its lanes', reaches 2^60 (a later score 41
// nats above the first 64), where a row's first scores are all -inf (weights without a shift, and a part that counts as empty
// in a join), or where V holds what is not finite, the workgroup runs once more: rows of the first two kinds, from a sum of
// 2^30 on, with their true maximum, and with values that a row does not see kept from it. What a join then drops is below
// 2^-66 of the row.
#pragma once
#include <algorithm>
#include <utility>

#include "qvl_decoder_core.h"

namespace qvl {

// f(0), f(1), ... with constant arguments.
template <typename F, int... I> __device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>{}), ...);
}

template <int D> struct WideUnit {
  using W = Wave<bf16, D>;
  using C = Core<bf16, D>;
  static constexpr int kRows = 256, kBN = 64, kG = D / 16, kDB = D / 32;
  static constexpr int kTile = kBN * C::kRowBytes, kDmas = kTile / 1024 / 4, kLds = 3 * 2 * kTile;
  static_assert(kLds >= 4 * kWriteLds, "rows are written through the tiles' LDS");
  static_assert(2 * kDmas == kG, "a DMA beside each product of one group");
  static constexpr float kMostSum = 0x1p60f;

  static __device__ __forceinline__ float shift_of(const W& w) { return w.m == -INFINITY ? 0.f : -w.m; }
  static __device__ __forceinline__ bf16x8 k_frag(const char* k, int b, int ks) {
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
    return *reinterpret_cast<const bf16x8*>(k + (b * 32 + l32) * C::kRowBytes + (((ks * 2 + hh) ^ C::k_swz(l32)) << 4));
  }

  // A tile; EDGE: some row may not see it whole, and its keys start at kb. k0: K's fragments of its first 32 keys; the next
  // tile's on return.
  template <bool EDGE, typename F>
  static __device__ __forceinline__ void tile(W& A, W& B, const char* k, const char* v, const char* knext, bf16x8 (&k0)[kG], int kb,
                                              float scale, F&& dma) {
    f32x16 s[4];
    u32x4 pw[4][2];
    bf16x8 k1[kG], v0[2 * kDB], v1[2 * kDB];
    const float sa = shift_of(A), sb = shift_of(B);
    const int first = kb + 4 * (int)((threadIdx.x & 63) >> 5), la = A.lim - first, lb = B.lim - first;
    float even;
    auto weight = [&](int p) {                  // score p & 15 of unit p >> 4; packed by twos
      const int u = p >> 4, i = p & 15;
      float x = s[u][i];
      if (EDGE) x = 32 * (u >> 1) + 8 * (i >> 2) + (i & 3) < (u & 1 ? lb : la) ? x : -INFINITY;
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, u & 1 ? sb : sa));
      (u & 1 ? B.core.l : A.core.l) += a;
      if (i & 1) pw[u][i >> 3][(i >> 1) & 3] = pack_bf16x2(even, a);
      else even = a;
    };
    auto product = [&](W& w, int u, const bf16x8 (&vf)[2 * kDB], int i) {
      const int e = i / kDB, db = i % kDB;
      w.core.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i], __builtin_bit_cast(bf16x8, pw[u][e]), w.core.o[db], 0, 0, 0);
    };
    auto score = [&](W& w, int u, const bf16x8& kf, int i) {
      s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, w.core.q[i], i ? s[u] : f32x16{}, 0, 0, 0);
    };
    each_of(std::make_integer_sequence<int, 8 * kG>{}, [&](auto at) {
      constexpr int slot = decltype(at)::value, g = slot / kG, i = slot % kG;
      if constexpr (g == 0) {
        score(A, 0, k0[i], i);
      } else if constexpr (g == 1) {
        k1[i] = k_frag(k, 1, i);
        score(B, 1, k0[i], i);
      } else if constexpr (g == 2) {
        v0[i] = A.core.v_frag(v, i % kDB, i / kDB);
        score(A, 2, k1[i], i);
      } else if constexpr (g == 3) {
        product(A, 0, v0, i);
      } else if constexpr (g == 4) {
        score(B, 3, k1[i], i);
      } else if constexpr (g == 5) {
        v1[i] = A.core.v_frag(v, i % kDB, 2 + i / kDB);
        product(B, 1, v0, i);
      } else if constexpr (g == 6) {
        product(A, 2, v1, i);
      } else {
        k0[i] = k_frag(knext, 0, i);
        product(B, 3, v1, i);
      }
      if constexpr (slot % 4 == 1 && slot / 4 < kG) dma(slot / 4);
      // the weights whose turn it is: 64 over the six groups from slot kG on
      constexpr int in = slot - kG, upto = in < 0 ? 0 : std::min(((in + 1) * 64 + 6 * kG - 1) / (6 * kG), 64);
      constexpr int from = in < 0 ? 0 : std::min((in * 64 + 6 * kG - 1) / (6 * kG), 64);
      each_of(std::make_integer_sequence<int, upto - from>{}, [&](auto p) { weight(from + decltype(p)::value); });
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  // 32 keys of a tile for one set of rows, with values that a row does not see kept from it.
  static __device__ __forceinline__ void block_safe(W& w, const char* k, const char* v, int b, int kb, float scale) {
    if (kb >= w.lim_hi) return;
    f32x16 s = w.core.scores(k, b);
    const uint32_t seen = w.mask(s, kb);
    const float shift = shift_of(w);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale, shift));
    if (kb + 32 > w.lim_lo) w.core.pv_safe(v, b, s, seen);
    else w.core.pv(v, b, s);
  }
  // The largest score of a tile, into m where it is larger. k0: K's fragments of its first 32 keys.
  static __device__ __forceinline__ void raise(W& A, W& B, const char* k, const bf16x8 (&k0)[kG], int kb, float scale) {
    f32x16 s[4] = {};                           // four chains of products, so that one hides another's latency
#pragma unroll
    for (int i = 0; i < kG; ++i) {
      const bf16x8 k1 = k_frag(k, 1, i);
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0[i], A.core.q[i], s[0], 0, 0, 0);
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0[i], B.core.q[i], s[1], 0, 0, 0);
      s[2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1, A.core.q[i], s[2], 0, 0, 0);
      s[3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1, B.core.q[i], s[3], 0, 0, 0);
    }
    if (kb + kBN > min(A.lim_lo, B.lim_lo)) {
      A.mask(s[0], kb);
      B.mask(s[1], kb);
      A.mask(s[2], kb + 32);
      B.mask(s[3], kb + 32);
    }
    float ma = fmaxf(s[0][0], s[2][0]), mb = fmaxf(s[1][0], s[3][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) {
      ma = fmaxf(fmaxf(ma, s[0][r]), s[2][r]);
      mb = fmaxf(fmaxf(mb, s[1][r]), s[3][r]);
    }
    A.m = fmaxf(A.m, across_halves(ma) * scale);
    B.m = fmaxf(B.m, across_halves(mb) * scale);
  }

  struct Tiles {
    Loader<bf16, D, false> lk;
    Loader<bf16, D, true> lv;
    const AttnParams& P;
    const Unit& u;
    uint32_t lds;
    int wave, t1;
    __device__ __forceinline__ Tiles(const AttnParams& P, const Unit& u, const char* smem, int t1)
        : lk(P.k), lv(P.v), P(P), u(u), lds(lds_addr_of(smem)), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), t1(t1) {}
    __device__ __forceinline__ void aim(int t) {
      const int left = t < t1 ? u.len - t * kBN : 0;
      lk.at(u.k + (int64_t)(t * kBN) * P.k.row, left);
      lv.at(u.v + (int64_t)(t * kBN) * P.v.row, left);
    }
    // DMA i < 2 kDmas of this wave's share of the tile aimed at
    __device__ __forceinline__ void load(int i, int stage) const {
      if (i < kDmas) lk(wave * kDmas + i, lds + stage * 2 * kTile);
      else lv(wave * kDmas + i - kDmas, lds + stage * 2 * kTile + kTile);
    }
    __device__ __forceinline__ void load_all(int t, int stage) {
      aim(t);
#pragma unroll
      for (int i = 0; i < 2 * kDmas; ++i) load(i, stage);
    }
  };

  // Rows [row0, row0 + 256) of the unit over tiles [t0, t1): tile t in stage (t - t0) % 3, two tiles ahead.
  static __device__ __forceinline__ void run(const AttnParams& P, const Unit& u, W& A, W& B, int row0, char* smem, int t0, int t1) {
    Tiles T(P, u, smem, t1);
    T.load_all(t0, 0);
    A.init(P, u, row0 + T.wave * 64);
    B.init(P, u, row0 + T.wave * 64 + 32);
    T.load_all(t0 + 1, 1);
    A.core.pin();
    B.core.pin();
    wait_dma();
    __syncthreads();
    if (t0 >= t1) return;
    bf16x8 k0[kG];
#pragma unroll
    for (int i = 0; i < kG; ++i) k0[i] = k_frag(smem, 0, i);
    raise(A, B, smem, k0, t0 * kBN, P.scale);
    // Two loops, so that the accumulators stay where they are in the first and its weights need no comparisons; a wave may
    // pass a barrier of one while another does of the other.
    const int whole = min(A.lim_lo, B.lim_lo) / kBN, some = max(A.lim_hi, B.lim_hi);
    int st = 0, t = t0;
    const auto after = [&](int n) { return smem + (st + n >= 3 ? st + n - 3 : st + n) * 2 * kTile; };
    const auto step = [&](auto edge) {
      const int to = st == 0 ? 2 : st - 1;      // of tile t + 2
      T.aim(t + 2);
      if (!decltype(edge)::value || t * kBN < some)
        tile<decltype(edge)::value>(A, B, after(0), after(0) + kTile, after(1), k0, t * kBN, P.scale, [&](int i) { T.load(i, to); });
      else
        for (int i = 0; i < 2 * kDmas; ++i) T.load(i, to);
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      st = st == 2 ? 0 : st + 1;
      ++t;
    };
    while (t < min(whole, t1)) step(std::false_type{});
    while (t < t1) step(std::true_type{});
  }
  // Once more, a tile at a time, after a run that left sums that are not finite.
  static __device__ __forceinline__ void run_safe(const AttnParams& P, const Unit& u, W& A, W& B, char* smem, int t0, int t1) {
    Tiles T(P, u, smem, t1);
    const float la = A.core.row_sum(), lb = B.core.row_sum();
    const float ma = A.m, mb = B.m;
    A.core.clear();
    B.core.clear();
    for (int t = t0; t < t1; ++t) {
      T.load_all(t, 0);
      wait_dma();
      __syncthreads();
      bf16x8 k0[kG];
#pragma unroll
      for (int i = 0; i < kG; ++i) k0[i] = k_frag(smem, 0, i);
      raise(A, B, smem, k0, t * kBN, P.scale);
      __syncthreads();
    }
    if (la < 0x1p30f && ma != -INFINITY) A.m = ma;
    if (lb < 0x1p30f && mb != -INFINITY) B.m = mb;
    for (int t = t0; t < t1; ++t) {
      T.load_all(t, 0);
      wait_dma();
      __syncthreads();
      for (int b = 0; b < 2; ++b) {
        block_safe(A, smem, smem + kTile, b, t * kBN + 32 * b, P.scale);
        block_safe(B, smem, smem + kTile, b, t * kBN + 32 * b, P.scale);
      }
      __syncthreads();
    }
  }
  static __device__ __forceinline__ void run_all(const AttnParams& P, const Unit& u, W& A, W& B, int row0, char* smem, int t0, int t1) {
    run(P, u, A, B, row0, smem, t0, t1);
    const auto good = [&](const W& w) {
      const float l = w.core.row_sum();         // (an exchange between lanes: every lane takes part)
      return w.finite() & (l < kMostSum) & (w.m != -INFINITY || w.lim <= t0 * kBN);
    };
    const bool ok = good(A) & good(B);
    if (__builtin_expect(__syncthreads_or(!ok), 0)) run_safe(P, u, A, B, smem, t0, t1);
  }
};

}  // namespace qvl
