// Device side shared by the decoder's attention kernels (qvl_causal.hip, qvl_decode.hip): out = softmax(scale q k^T) v over the
// keys a token sees, grouped heads, bf16 or fp32, head_dim 64 or 128.
//
// A row is one (token, query head); the rows of one key/value head that see the same keys are handled together. One
// pass over the keys holds the running maximum m, the sum l of 2^(s - m) and the unnormalised output.
#pragma once
#include <math.h>
#include <type_traits>

#include "qvl_decoder_items.h"
#include "qvl_kernels.h"

namespace qvl {

struct AttnView {
  const char* p;
  int64_t row, head;   // strides in bytes
};

struct AttnParams {
  AttnView q, k, v, out;
  int64_t kv_rows, n_tokens;
  int hkv, group;          // key/value heads, query heads of each
  float scale;             // of the scores, times log2(e): the softmax runs on powers of two
  float* part_o;           // partial results: unnormalised outputs and (m, l) of rows
  f32x2* part_ml;
};

// A value that is the same in every lane, in scalar registers (a DMA's descriptor and a workgroup's branches have to be).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}

// The larger of the two lanes of a row.
__device__ __forceinline__ float across_halves(float x) {
  const u32x2 p = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// What one wave does with 32 rows and a block of 32 keys in LDS. S^T = K Q^T puts a row in a lane (column lane % 32) with
// 16 of the block's keys: register r is key 8 (r / 4) + 4 (lane / 32) + r % 4. The second product O^T = V^T P^T takes P as
// it lies in those registers, as its B operand; only V has to come transposed.
//
// bf16: v_mfma_f32_32x32x16. K and V lie in LDS row by row as they come from memory. A lane's 8 keys of a 16-key group
// are two runs of 4, so V^T is read by two transposing reads of 4 keys (ds_read_b64_tr_b16: 16 lanes give 4 rows of 16
// values, and each gets a column). The weights are rounded to bf16 for that product, the type of the instruction's operands:
// outputs are 1.7e-3 to 2.3e-3 off, 1.3e-3 to 1.7e-3 of which is their own rounding; weights in two bf16 parts would take the
// rest away for half as many matrix instructions again, in kernels bound by those. The row sums are plain fp32 additions of
// the weights before their rounding: a dot instruction that adds two rounded ones waits for the matrix cores (52 cycles
// beside a product of 32).
// 16-byte chunks are XOR-swizzled by the row so that neither read meets a bank twice: 16 rows of one chunk for K, 4 rows
// of 64 bytes for V.
template <typename T, int D> struct Core;

template <int D> struct Core<bf16, D> {
  static constexpr int kRows = 32, kRowBytes = D * 2, kDB = D / 32;
  static constexpr int kChunks = kRowBytes / 16;
  bf16x8 q[D / 16];
  f32x16 o[kDB];
  float l;

  static __device__ __forceinline__ int k_swz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int v_swz(int row) { return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

  __device__ __forceinline__ void init(const char* qrow) {
    const int lane = threadIdx.x & 63, hh = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) q[ks] = *reinterpret_cast<const bf16x8*>(qrow + (ks * 16 + hh * 8) * 2);
    clear();
  }
  // Uses the rows, so that the wait for their loads stands here, behind the first DMAs' issue: at their first use in the loop
  // it would be a wait for every DMA in flight, tile by tile.
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (auto& x : q) asm volatile("" : "+v"(x));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] = f32x16{};
    l = 0.f;
  }
  // keys block b of the tile at `lds` (one sum: D / 16 additions, each of 16 exact products)
  template <int SUMS = 1> __device__ __forceinline__ f32x16 scores(const char* lds, int b) const {
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
    f32x16 s = f32x16{};
    const char* row = lds + (b * 32 + l32) * kRowBytes;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const bf16x8 k = *reinterpret_cast<const bf16x8*>(row + (((ks * 2 + hh) ^ k_swz(l32)) << 4));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[ks], s, 0, 0, 0);
    }
    return s;
  }
  // V^T rows 32 db + lane % 32, the lane's 8 keys of 16-key group g (keys 16 g on)
  __device__ __forceinline__ bf16x8 v_frag(const char* lds, int db, int g) const {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const int lane = threadIdx.x & 63, hh = lane >> 5, i = lane & 15;
    const int r = 4 * hh + (i >> 2);                       // row of the first run; the second is 8 rows on (same swizzle)
    const int c = db * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
    const char* p = lds + (16 * g + r) * kRowBytes + ((c ^ v_swz(r)) << 4) + (i & 1) * 8;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * kRowBytes));
    return __builtin_bit_cast(bf16x8, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
  }
  __device__ __forceinline__ void pv(const char* lds, int b, const f32x16& p) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      u32x4 pw;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pw[j] = pack_bf16x2(p[8 * e + 2 * j], p[8 * e + 2 * j + 1]);
        l += p[8 * e + 2 * j];
        l += p[8 * e + 2 * j + 1];
      }
      const bf16x8 pf = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_frag(lds, db, 2 * b + e), pf, o[db], 0, 0, 0);
    }
  }
  // The scores of both blocks of a tile of 64 keys: a block's fragments are read ahead of its products.
  // `beside(i)`, i < 8, runs among the products.
  template <typename F> __device__ __forceinline__ void scores2(const char* lds, f32x16 (&s)[2], F&& beside) const {
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
    const char* row = lds + l32 * kRowBytes;
    bf16x8 a[D / 16], c[D / 16];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) a[ks] = *reinterpret_cast<const bf16x8*>(row + (((ks * 2 + hh) ^ k_swz(l32)) << 4));
    __builtin_amdgcn_sched_barrier(0);
    s[0] = f32x16{};
    s[1] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      c[ks] = *reinterpret_cast<const bf16x8*>(row + 32 * kRowBytes + (((ks * 2 + hh) ^ k_swz(l32)) << 4));
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[ks], q[ks], s[0], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (ks % (D / 64) == D / 64 - 1) beside(ks / (D / 64));
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c[ks], q[ks], s[1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (ks % (D / 64) == D / 64 - 1) beside(4 + ks / (D / 64));
    }
  }
  __device__ __forceinline__ void v_group(const char* lds, int g, bf16x8 (&v)[kDB]) const {
#pragma unroll
    for (int db = 0; db < kDB; ++db) v[db] = v_frag(lds, db, g);
  }
  __device__ __forceinline__ u32x4 pack8(const f32x16& s, int e, float scale, float shift) {
    float p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * e + r], scale, shift));
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pack_bf16x2(p[2 * j], p[2 * j + 1]);
      l += p[2 * j];
      l += p[2 * j + 1];
    }
    return w;
  }
  // Weights and their product with V, 16 keys at a time: a group's weights are formed and its V read beside the products of
  // the group before. v0: V's first group.
  __device__ __forceinline__ void pv2(const char* lds, bf16x8 (&v0)[kDB], const f32x16 (&s)[2], float scale, float shift) {
    u32x4 pw = pack8(s[0], 0, scale, shift);
    bf16x8 v1[kDB];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 (&now)[kDB] = g & 1 ? v1 : v0;
      bf16x8 (&next)[kDB] = g & 1 ? v0 : v1;
      if (g < 3) v_group(lds, g + 1, next);
      const bf16x8 pf = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now[db], pf, o[db], 0, 0, 0);
      if (g < 3) pw = pack8(s[(g + 1) >> 1], (g + 1) & 1, scale, shift);
      if (g < 3) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * kDB, 0);
#pragma unroll
        for (int db = 0; db < kDB; ++db) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 24 / kDB, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // The same where some rows do not see all of the block's keys and V may hold infinities or NaN, which a weight of zero
  // does not silence: V's non-finite values are left out of the product and counted, row by row, among the keys that the
  // row sees (+inf as 1, -inf as 2^8, NaN as 2^16: sums of 16 keys stay exact), and the counts put back what they stand for.
  __device__ __forceinline__ void pv_safe(const char* lds, int b, const f32x16& p, uint32_t seen) {
    for (int e = 0; e < 2; ++e) {
      u32x4 pw, sw;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 8 * e + 2 * j;
        pw[j] = pack_bf16x2(p[r], p[r + 1]);
        l += p[r];
        l += p[r + 1];
        sw[j] = ((seen >> r) & 1 ? 0x3f80u : 0u) | ((seen >> (r + 1)) & 1 ? 0x3f800000u : 0u);
      }
      const bf16x8 pf = __builtin_bit_cast(bf16x8, pw), sf = __builtin_bit_cast(bf16x8, sw);
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        u32x4 v = __builtin_bit_cast(u32x4, v_frag(lds, db, 2 * b + e)), bad;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t clean = 0, mark = 0;
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            const uint32_t x = (v[j] >> h) & 0xffffu;
            const bool ok = (x & 0x7f80u) != 0x7f80u;
            clean |= (ok ? x : 0u) << h;
            mark |= (ok ? 0u : x == 0x7f80u ? 0x3f80u : x == 0xff80u ? 0x4380u : 0x4780u) << h;
          }
          v[j] = clean;
          bad[j] = mark;
        }
        __builtin_amdgcn_sched_barrier(0);   // one output block at a time: registers
        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), pf, o[db], 0, 0, 0);
        const f32x16 n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, bad), sf, f32x16{}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t c = (uint32_t)n[r];
          if (c & 0xffu) o[db][r] += INFINITY;
          if (c & 0xff00u) o[db][r] -= INFINITY;
          if (c >> 16) o[db][r] = NAN;
        }
      }
    }
  }
  __device__ __forceinline__ void rescale(float a) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] *= a;
    l *= a;
  }
  // the row's sum, in both of its lanes
  __device__ __forceinline__ float row_sum() const { return l + __shfl_xor(l, 32); }
  // f(first dim, 4 values) for each run of 4 dims this lane holds of its row
  template <typename F> __device__ __forceinline__ void each4(F&& f) const {
    const int hh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f(db * 32 + 8 * k + 4 * hh, f32x4{o[db][4 * k], o[db][4 * k + 1], o[db][4 * k + 2], o[db][4 * k + 3]});
  }
};

// fp32: v_mfma_f32_32x32x2_f32, one value a lane and operand. The two lanes of a row take dims (or keys) 4 apart, so that K
// is read 16 bytes at a time; a lane of V^T takes the dims kDB i + db of its row i, which lie together in V's row: one
// read serves all of a key's output blocks. P needs no packing.
template <int D> struct Core<float, D> {
  static constexpr int kRows = 32, kRowBytes = D * 4, kDB = D / 32;
  static constexpr int kChunks = kRowBytes / 16;
  f32x4 q[D / 8];
  f32x16 o[kDB];
  float l;

  static __device__ __forceinline__ int k_swz(int row) { return row & 15; }
  static __device__ __forceinline__ int v_swz(int) { return 0; }

  __device__ __forceinline__ void init(const char* qrow) {
    const int hh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) q[j] = *reinterpret_cast<const f32x4*>(qrow + (j * 8 + hh * 4) * 4);
    clear();
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (auto& x : q) asm volatile("" : "+v"(x));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] = f32x16{};
    l = 0.f;
  }
  // SUMS sums of D / SUMS products each, added in pairs: of a score of 128 products one sum is off by 3.4 2^-24 in the root
  // mean square, two by 2.5, four by 1.9.
  template <int SUMS> __device__ __forceinline__ f32x16 scores(const char* lds, int b) const {
    static_assert(SUMS == 1 || SUMS == 2 || SUMS == 4, "sums of a score");
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
    f32x16 s[SUMS] = {};
    const char* row = lds + (b * 32 + l32) * kRowBytes;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const f32x4 k = *reinterpret_cast<const f32x4*>(row + (((j * 2 + hh) ^ k_swz(l32)) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e % SUMS] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[j][e], s[e % SUMS], 0, 0, 0);
    }
    if constexpr (SUMS == 4) return (s[0] + s[1]) + (s[2] + s[3]);
    else if constexpr (SUMS == 2) return s[0] + s[1];
    else return s[0];
  }
  // dims kDB (lane % 32) + db of the lane's key in register r of block b
  __device__ __forceinline__ void v_frag(const char* lds, int b, int r, float (&v)[kDB]) const {
    const int lane = threadIdx.x & 63;
    const char* p = lds + (b * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * kRowBytes + (lane & 31) * kDB * 4;
    if constexpr (kDB == 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
      for (int db = 0; db < 4; ++db) v[db] = x[db];
    } else {
      const f32x2 x = *reinterpret_cast<const f32x2*>(p);
      v[0] = x[0];
      v[1] = x[1];
    }
  }
  __device__ __forceinline__ void pv(const char* lds, int b, const f32x16& p) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v[kDB];
      v_frag(lds, b, r, v);
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[db], p[r], o[db], 0, 0, 0);
      l += p[r];
    }
  }
  __device__ __forceinline__ void pv_safe(const char* lds, int b, const f32x16& p, uint32_t seen) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      f32x16 n = f32x16{};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v[kDB];
        v_frag(lds, b, r, v);
        const bool ok = fabsf(v[db]) < INFINITY;
        const float mark = ok ? 0.f : v[db] == INFINITY ? 1.f : v[db] == -INFINITY ? 256.f : 65536.f;
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(ok ? v[db] : 0.f, p[r], o[db], 0, 0, 0);
        n = __builtin_amdgcn_mfma_f32_32x32x2f32(mark, (seen >> r) & 1 ? 1.f : 0.f, n, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t c = (uint32_t)n[r];
        if (c & 0xffu) o[db][r] += INFINITY;
        if (c & 0xff00u) o[db][r] -= INFINITY;
        if (c >> 16) o[db][r] = NAN;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) l += p[r];
  }
  __device__ __forceinline__ void rescale(float a) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] *= a;
    l *= a;
  }
  __device__ __forceinline__ float row_sum() const { return l + __shfl_xor(l, 32); }
  template <typename F> __device__ __forceinline__ void each4(F&& f) const {
    const int hh = (threadIdx.x & 63) >> 5;
    if constexpr (kDB == 4) {
#pragma unroll
      for (int r = 0; r < 16; ++r) f(4 * (8 * (r >> 2) + 4 * hh + (r & 3)), f32x4{o[0][r], o[1][r], o[2][r], o[3][r]});
    } else {
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        f(2 * (8 * (r >> 2) + 4 * hh + (r & 3)), f32x4{o[0][r], o[1][r], o[0][r + 1], o[1][r + 1]});
    }
  }
};

// 4 values rounded to T at dim d of a row.
template <typename T> __device__ __forceinline__ void store4(char* row, int d, const f32x4& x) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<f32x4*>(row + 4 * d) = x;
  else *reinterpret_cast<u32x2*>(row + 2 * d) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
}

// Keys of one unit of work for one key/value head: cache rows from `k`, `v`, rows of the unit [row0, rows) as (token, head)
// pairs, token by token; token t sees keys below lim0 + t, and never more than `len`.
struct Unit {
  const char *k, *v;
  int len, lim0;       // lim0 + t: keys that token t sees (len - 1 and more: all of them)
  int64_t token0;      // the sequence's (or group's) first token
  int rows, row0, kvh;
};

// The rows of one wave, one a lane (and more lanes of the same row), and what they see.
template <typename C> struct RowState {
  static constexpr int kRows = C::kRows;
  C core;
  float m;             // running maximum of the lane's row, in powers of two; -inf before the first key it sees
  int lim, lim_lo;     // keys the lane's row sees; the fewest any row of the wave does
  int lim_hi;          // the most

  __device__ __forceinline__ void init(const AttnParams& P, const Unit& u, int first_row) {
    const int row = min(first_row + (int)(threadIdx.x & (kRows - 1)), u.rows - 1);
    const int t = (int)((uint32_t)row / (uint32_t)P.group), g = row - t * P.group;
    const char* q = P.q.p + (u.token0 + t) * P.q.row + (int64_t)(u.kvh * P.group + g) * P.q.head;
    lim = max(min(u.lim0 + t, u.len), 0);
    const int lo = min(first_row, u.rows - 1), hi = min(first_row + kRows - 1, u.rows - 1);
    lim_lo = max(min(u.lim0 + (int)((uint32_t)lo / (uint32_t)P.group), u.len), 0);
    lim_hi = max(min(u.lim0 + (int)((uint32_t)hi / (uint32_t)P.group), u.len), 0);
    m = -INFINITY;
    core.init(q);
  }
  // The maximum moved to cover mx, the largest score of a step (times the scale). It moves only where it grew by more than
  // 2^8: until then weights of up to 2^8 lose nothing (fp32 sums, and bf16 weights of the same relative rounding), and the
  // accumulators need no pass. Row by row, so that a row's result does not depend on the others of its wave.
  __device__ __forceinline__ void cover(float mx) {
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {
      const float mn = mx > m + 8.f ? mx : m;
      // (nothing to rescale before a row's first key)
      if (__builtin_amdgcn_ballot_w64(m != -INFINITY) != 0) core.rescale(__builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn)));
      m = mn;
    }
  }
  __device__ __forceinline__ float shift() const { return m == -INFINITY ? 0.f : -m; }
};

// The online softmax of one wave: 32 rows over the keys it is given. SUMS: Core's, fp32 (4000 keys, head_dim 128: 1.12e-6 off
// with one, 6.5e-7 with two, 4.6e-7 with four, no slower; head_dim 64 has no registers for four).
template <typename T, int D, int SUMS = D == 128 ? 4 : 2> struct Wave : RowState<Core<T, D>> {
  using RowState<Core<T, D>>::core;
  using RowState<Core<T, D>>::m;
  using RowState<Core<T, D>>::lim;
  using RowState<Core<T, D>>::lim_lo;

  // Scores of 32 keys from kb on that the lane's row does not see become -inf; returns which it sees, a bit per register.
  __device__ __forceinline__ uint32_t mask(f32x16& s, int kb) const {
    const int base = lim - kb - 4 * (int)((threadIdx.x & 63) >> 5);
    uint32_t seen = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool in = 8 * (r >> 2) + (r & 3) < base;
      seen |= (in ? 1u : 0u) << r;
      s[r] = in ? s[r] : -INFINITY;
    }
    return seen;
  }
  // NB blocks of 32 keys from key kb on; K and V tiles in LDS. `between(i)`, i < 8, runs beside the scores' products, or
  // after them, once they are read out of K's tile; `before_v` before V's is read.
  // SAFE: V may hold what is not finite.
  template <int NB, bool SAFE, typename F, typename G>
  __device__ __forceinline__ void step(const char* klds, const char* vlds, int kb, float scale, F&& between, G&& before_v) {
    f32x16 s[NB];
    constexpr bool kAhead = NB == 2 && !SAFE && std::is_same<T, bf16>::value;
    bf16x8 v0[D / 32];
    if constexpr (kAhead) {
      core.scores2(klds, s, between);
      core.v_group(vlds, 0, v0);
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) s[b] = core.template scores<SUMS>(klds, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) between(i);
    }
    const bool edge = kb + 32 * NB > lim_lo;
    uint32_t seen[NB];
    if (edge) {
#pragma unroll
      for (int b = 0; b < NB; ++b) seen[b] = mask(s[b], kb + 32 * b);
    }
    float m4[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      m4[c] = s[0][c];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = b ? 0 : 4; r < 16; r += 4) m4[c] = fmaxf(m4[c], s[b][r + c]);
    }
    const float mx = across_halves(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))) * scale;
    this->cover(mx);
    const float shift = this->shift();
    if constexpr (kAhead) {
      core.pv2(vlds, v0, s, scale, shift);
      return;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], scale, shift));
    before_v();
    if (SAFE && edge) {
#pragma unroll
      for (int b = 0; b < NB; ++b) core.pv_safe(vlds, b, s[b], seen[b]);
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) core.pv(vlds, b, s[b]);
    }
  }
  __device__ __forceinline__ bool finite() const {
    bool ok = true;
    core.each4([&](int, const f32x4& x) {
#pragma unroll
      for (int e = 0; e < 4; ++e) ok = ok & (fabsf(x[e]) < INFINITY);
    });
    return ok;
  }
};

// fp32 and at most 16 rows, on v_mfma_f32_16x16x4_f32: half the products of a tile of 32 rows, 4096 cycles a block of 32 keys
// at head_dim 128. A row has four lanes (column lane % 16 of S^T = K Q^T); of half b of the block, register r of a lane is
// key 16 b + 4 (lane / 16) + r. Its lanes take dims 16 j + 4 (lane / 16) + e of K and Q; a lane of V^T takes dims
// 64 h + 4 (lane % 16) + e. K and V lie in LDS as for Core<float, D>.
template <int D> struct FewCore {
  using C = Core<float, D>;
  static constexpr int kRows = 16, kDB = D / 16;
  f32x4 q[D / 16], o[kDB];
  float l;

  static __device__ __forceinline__ int quad() { return (threadIdx.x & 63) >> 4; }
  static __device__ __forceinline__ int l16() { return threadIdx.x & 15; }
  __device__ __forceinline__ void init(const char* qrow) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = *reinterpret_cast<const f32x4*>(qrow + (j * 16 + quad() * 4) * 4);
#pragma unroll
    for (auto& x : o) x = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (auto& x : q) asm volatile("" : "+v"(x));
  }
  // Four sums of a quarter of the products each, as in Core<float, D>: 2310 keys and one sum 1.15e-6 off, four 4.0e-7.
  __device__ __forceinline__ void scores(const char* lds, f32x4 (&s)[2]) const {
    f32x4 t[2][4] = {};
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      f32x4 k[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int row = 16 * b + l16();
        k[b] = *reinterpret_cast<const f32x4*>(lds + row * C::kRowBytes + (((j * 4 + quad()) ^ C::k_swz(row)) << 4));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int b = 0; b < 2; ++b) t[b][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[b][e], q[j][e], t[b][e], 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = (t[b][0] + t[b][1]) + (t[b][2] + t[b][3]);
  }
  static __device__ __forceinline__ f32x4 v_frag(const char* lds, int b, int r, int h) {
    return *reinterpret_cast<const f32x4*>(lds + (16 * b + 4 * quad() + r) * C::kRowBytes + (16 * h + l16()) * 16);
  }
  __device__ __forceinline__ void pv(const char* lds, const f32x4 (&p)[2]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = p[i >> 2][i & 3];
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        const f32x4 v = v_frag(lds, i >> 2, i & 3, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], w, o[4 * h + e], 0, 0, 0);
      }
      l += w;
    }
  }
  __device__ __forceinline__ void pv_safe(const char* lds, const f32x4 (&p)[2], uint32_t seen) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      f32x4 n = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = v_frag(lds, i >> 2, i & 3, db >> 2)[db & 3];
        const bool ok = fabsf(v) < INFINITY;
        const float mark = ok ? 0.f : v == INFINITY ? 1.f : v == -INFINITY ? 256.f : 65536.f;
        o[db] = __builtin_amdgcn_mfma_f32_16x16x4f32(ok ? v : 0.f, p[i >> 2][i & 3], o[db], 0, 0, 0);
        n = __builtin_amdgcn_mfma_f32_16x16x4f32(mark, (seen >> i) & 1 ? 1.f : 0.f, n, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t c = (uint32_t)n[r];
        if (c & 0xffu) o[db][r] += INFINITY;
        if (c & 0xff00u) o[db][r] -= INFINITY;
        if (c >> 16) o[db][r] = NAN;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) l += p[i >> 2][i & 3];
  }
  __device__ __forceinline__ void rescale(float a) {
#pragma unroll
    for (auto& x : o) x *= a;
    l *= a;
  }
  __device__ __forceinline__ float row_sum() const {
    const float two = l + __shfl_xor(l, 16);
    return two + __shfl_xor(two, 32);
  }
  template <typename F> __device__ __forceinline__ void each4(F&& f) const {
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        f(64 * h + 4 * (4 * quad() + r), f32x4{o[4 * h][r], o[4 * h + 1][r], o[4 * h + 2][r], o[4 * h + 3][r]});
  }
};

template <int D> struct FewWave : RowState<FewCore<D>> {
  using RowState<FewCore<D>>::core;
  using RowState<FewCore<D>>::lim;
  using RowState<FewCore<D>>::lim_lo;

  // Wave::step for a block of 32 keys
  template <int NB, bool SAFE, typename F, typename G>
  __device__ __forceinline__ void step(const char* klds, const char* vlds, int kb, float scale, F&& between, G&& before_v) {
    static_assert(NB == 1, "a block at a time");
    f32x4 s[2];
    core.scores(klds, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) between(i);
    const bool edge = kb + 32 > lim_lo;
    uint32_t seen = 0;
    if (edge) {
      const int base = lim - kb - 4 * core.quad();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = 16 * (i >> 2) + (i & 3) < base;
        seen |= (in ? 1u : 0u) << i;
        s[i >> 2][i & 3] = in ? s[i >> 2][i & 3] : -INFINITY;
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
    mx = across_halves(mx);
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    this->cover(mx * scale);
    const float shift = this->shift();
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][i & 3], scale, shift));
    before_v();
    if (SAFE && edge) core.pv_safe(vlds, s, seen);
    else core.pv(vlds, s);
  }
};

// One DMA fills 1 KiB of a tile: lane j chunk j % kChunks of row j / kChunks, from the logical chunk that the swizzle maps
// there. A K or V tile takes a whole number of them; `Loader` does the i-th.
template <typename T, int D, bool V> struct Loader {
  using C = Core<T, D>;
  static constexpr int kRows = 1024 / C::kRowBytes;   // rows of one DMA
  u32x4 rsrc;
  uint32_t stride, row_off, chunk;

  __device__ __forceinline__ Loader(const AttnView& x) {
    const int lane = threadIdx.x & 63;
    stride = (uint32_t)x.row;
    row_off = (uint32_t)(lane / C::kChunks) * stride;
    chunk = (uint32_t)((lane % C::kChunks) ^ swz(lane / C::kChunks)) << 4;
  }
  static __device__ __forceinline__ int swz(int row) { return V ? C::v_swz(row) : C::k_swz(row); }
  // `left` rows from `base` on; past them zeros arrive (copies, where rows lie closer than a row is long)
  __device__ __forceinline__ void at(const char* base, int left) {
    rsrc = rsrc_words((const char*)uniform((int64_t)base),
                      (uint32_t)uniform((int)(left > 0 ? (uint32_t)((int64_t)(min(left, 64) - 1) * stride + C::kRowBytes) : 0u)));
  }
  // rows [kRows i, kRows (i + 1)) of the tile at `lds`. (A DMA's rows lie in one aligned run of kRows, so the swizzle of
  // row kRows i + r is that of kRows i XOR that of r.)
  __device__ __forceinline__ void operator()(int i, uint32_t lds) const {
    const uint32_t r = (uint32_t)(i * kRows);
    dma16(rsrc, row_off + r * stride + (chunk ^ ((uint32_t)swz(r & 31) << 4)), 0, lds + r * C::kRowBytes);
  }
};

// A row's result: rounded to its place, or unnormalised with (m, l) into a partial buffer.
template <typename T, int D>
__device__ __forceinline__ char* out_row(const AttnParams& P, const Unit& u, int row) {
  const int t = (int)((uint32_t)row / (uint32_t)P.group), g = row - t * P.group;
  return const_cast<char*>(P.out.p) + (u.token0 + t) * P.out.row + (int64_t)(u.kvh * P.group + g) * P.out.head;
}

// 128 rows a workgroup, 32 a wave; the four waves share each tile of 64 (fp32: 32) keys, which comes by LDS DMA into one of
// two stages while the other is computed on.
template <typename T, int D> struct RowsUnit {
  static constexpr int kNB = std::is_same<T, float>::value ? 1 : 2, kBN = 32 * kNB;
  static constexpr int kTile = kBN * Core<T, D>::kRowBytes, kLds = 4 * kTile;

  static constexpr int kDmas = kTile / 1024 / 4;   // of each wave and tile

  // Tiles [t0, t1) of the unit. The next tile's DMAs stand among this one's products: issued together they would hold the
  // wave for as long as they take to address (8 of them: 900 cycles of 3850 a tile).
  template <typename W>
  static __device__ __forceinline__ void run(const AttnParams& P, const Unit& u, W& w, char* smem, int t0, int t1) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds0 = lds_addr_of(smem);
    Loader<T, D, false> lk(P.k);
    Loader<T, D, true> lv(P.v);
    const auto aim = [&](int t) {
      const int kb = t * kBN, left = t < t1 ? u.len - kb : 0;
      lk.at(u.k + (int64_t)kb * P.k.row, left);
      lv.at(u.v + (int64_t)kb * P.v.row, left);
    };
    const auto load = [&](int i, int stage) {   // i < 2 kDmas
      if (i < kDmas) lk(wave * kDmas + i, lds0 + stage * 2 * kTile);
      else if (i < 2 * kDmas) lv(wave * kDmas + i - kDmas, lds0 + stage * 2 * kTile + kTile);
    };
    aim(t0);
#pragma unroll
    for (int i = 0; i < 2 * kDmas; ++i) load(i, 0);
    w.core.pin();
    wait_dma();
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int stage = (t - t0) & 1;
      const char* k = smem + stage * 2 * kTile;
      aim(t + 1);
      if (t * kBN < w.lim_hi) {
        w.template step<kNB, false>(k, k + kTile, t * kBN, P.scale, [&](int i) { load(i, stage ^ 1); }, [] {});
      } else {
#pragma unroll
        for (int i = 0; i < 2 * kDmas; ++i) load(i, stage ^ 1);
      }
      wait_dma();
      __syncthreads();
    }
  }
  // The same, telling apart what a row sees where V is not finite; a tile at a time.
  template <typename W>
  static __device__ __forceinline__ void run_safe(const AttnParams& P, const Unit& u, W& w, char* smem, int t0, int t1) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds0 = lds_addr_of(smem);
    Loader<T, D, false> lk(P.k);
    Loader<T, D, true> lv(P.v);
    for (int t = t0; t < t1; ++t) {
      lk.at(u.k + (int64_t)(t * kBN) * P.k.row, u.len - t * kBN);
      lv.at(u.v + (int64_t)(t * kBN) * P.v.row, u.len - t * kBN);
      for (int i = wave * kDmas; i < (wave + 1) * kDmas; ++i) {
        lk(i, lds0);
        lv(i, lds0 + kTile);
      }
      wait_dma();
      __syncthreads();
      if (t * kBN < w.lim_hi) w.template step<kNB, true>(smem, smem + kTile, t * kBN, P.scale, [](int) {}, [] {});
      __syncthreads();
    }
  }
};

// Up to 32 rows a workgroup (W: Wave, or FewWave of 16); the four waves take every fourth block of 32 keys, each through LDS of its own: while a block's
// weights are formed the next block's keys arrive, while its scores are formed the next values do. Joined in LDS at the end.
template <typename T, int D> struct KeysUnit {
  static constexpr int kTile = 32 * Core<T, D>::kRowBytes, kLds = 4 * 2 * kTile;
  static constexpr int kDmas = kTile / 1024;

  template <typename W>
  static __device__ __forceinline__ void run(const AttnParams& P, const Unit& u, W& w, char* smem, int t0, int t1) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* k = smem + wave * 2 * kTile;
    const uint32_t kl = lds_addr_of(k), vl = kl + kTile;
    Loader<T, D, false> lk(P.k);
    Loader<T, D, true> lv(P.v);
    const auto load_k = [&](int t) {
      lk.at(u.k + (int64_t)(t * 32) * P.k.row, u.len - t * 32);
#pragma unroll
      for (int i = 0; i < kDmas; ++i) lk(i, kl);
    };
    const auto load_v = [&](int t) {
      lv.at(u.v + (int64_t)(t * 32) * P.v.row, u.len - t * 32);
#pragma unroll
      for (int i = 0; i < kDmas; ++i) lv(i, vl);
    };
    t0 += wave;
    if (t0 >= t1) return;
    load_k(t0);
    load_v(t0);
    w.core.pin();
    // In flight, oldest first: K(t), V(t) at the top; V(t), K(t + 1) before V is read.
    int t = t0;
    const auto each = [&](auto safe) {
      const bool more = t + 4 < t1;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDmas) : "memory");
      w.template step<1, decltype(safe)::value>(k, k + kTile, t * 32, P.scale,
                                                [&](int i) {
                                                  if (i) return;
                                                  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                                                  if (more) load_k(t + 4);
                                                },
                                                [&] {
                                                  if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kDmas) : "memory");
                                                  else wait_dma();
                                                });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) load_v(t + 4);
      t += 4;
    };
    // blocks that every row sees whole, or that only end inside (what lies behind the keys reads as zeros, unless V's rows lie
    // closer than a row is long: then it is a copy of keys before); then the rest
    const int whole = w.lim_lo < u.len || P.v.row < Core<T, D>::kRowBytes ? min(w.lim_lo / 32, t1) : t1;
    while (t < whole) each(std::false_type{});
    while (t < t1) each(std::true_type{});
  }
};


// (m, l) of a part as the combine reads it: no key seen (-inf, 0), only keys of score -inf (-inf, -0).
__device__ __forceinline__ f32x2 part_state(float m, float l, bool sees) { return f32x2{m, l == 0.f && sees ? -0.f : l}; }

// LDS of one wave that writes 32 rows.
constexpr int kWriteLds = 32 * (256 + 16);

// A wave's 32 rows of D values E, f of the 4 that a lane holds at a time, to where each lane's row goes (dst; nullptr:
// nowhere). They are turned in LDS so that the stores cover whole rows: a lane's own 8 bytes of 32 rows at a time kept the
// CU's address unit for 7900 cycles a tile of 256 rows, so it takes 5500.
template <typename E, int D, typename W, typename F>
__device__ __forceinline__ void store_rows(const W& w, char* dst, char* lds, F&& f) {
  constexpr int kBytes = D * (int)sizeof(E) < 256 ? D * (int)sizeof(E) : 256, kPieces = D * (int)sizeof(E) / kBytes, kDims = D / kPieces;
  constexpr int kPitch = kBytes + 16, kChunks = kBytes / 16;      // the row's address stands behind its bytes
  const int lane = threadIdx.x & 63, l32 = lane & 31;
  char* mine = lds + l32 * kPitch;
  if (lane < 32) *reinterpret_cast<char**>(mine + kBytes) = dst;
#pragma unroll
  for (int piece = 0; piece < kPieces; ++piece) {
    w.core.each4([&](int d, const f32x4& x) {
      if (d / kDims == piece) store4<E>(mine, d % kDims, f(x));
    });
    __builtin_amdgcn_wave_barrier();
    char* to[kChunks / 2];
    u32x4 x[kChunks / 2];
#pragma unroll
    for (int i = 0; i < kChunks / 2; ++i) {                       // 64 / kChunks rows each
      const char* row = lds + (i * (64 / kChunks) + lane / kChunks) * kPitch;
      to[i] = *reinterpret_cast<char* const*>(row + kBytes);
      x[i] = *reinterpret_cast<const u32x4*>(row + lane % kChunks * 16);
    }
#pragma unroll
    for (int i = 0; i < kChunks / 2; ++i)
      if (to[i]) *reinterpret_cast<u32x4*>(to[i] + piece * kBytes + lane % kChunks * 16) = x[i];
    __builtin_amdgcn_wave_barrier();
  }
}

// One wave writes its 32 rows, through kWriteLds bytes of LDS that no other wave uses: to the output, or as a part.
template <typename T, int D, typename W>
__device__ __forceinline__ void write_rows(const AttnParams& P, const Unit& u, const W& w, char* lds, int row, float* po,
                                           f32x2* pml, bool sees) {
  const float l = w.core.row_sum();
  if (po) {
    store_rows<float, D>(w, row < u.rows ? (char*)po : nullptr, lds, [](const f32x4& x) { return x; });
    if (row < u.rows && (threadIdx.x & 63) < 32) *pml = part_state(w.m, l, sees);
  } else {
    const float inv = 1.0f / l;
    store_rows<T, D>(w, row < u.rows ? out_row<T, D>(P, u, row) : nullptr, lds,
                     [&](const f32x4& x) { return sees ? x * inv : f32x4{0.f, 0.f, 0.f, 0.f}; });
  }
}

// Parts of rows joined: out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p, in an order that only the number of parts
// sets. A workgroup takes 256 / (lanes x split) rows at once: D / 4 lanes hold a row, 16 bytes each, and `split` groups of
// them share its parts, 8 in flight each, so that a row of 64 parts costs one trip to memory and not 64. `at(r, p)` is part
// p's row index in P.part_ml / P.part_o, `out(r)` where row r goes.
__device__ __host__ constexpr int join_split(int parts) { return parts <= 8 ? 1 : parts <= 16 ? 2 : parts <= 32 ? 4 : 8; }

template <typename T, int D, typename At, typename Out>
__device__ __forceinline__ void join_parts(const AttnParams& P, int row0, int row1, int parts, At&& at, Out&& out) {
  constexpr int kLanes = D / 4, kSlots = 256 / kLanes, kFlight = 8;
  __shared__ f32x4 so[kSlots][kLanes];
  __shared__ float sm[kSlots], sl[kSlots];
  __shared__ int ss[kSlots];
  const int split = join_split(parts), slot = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, g = slot % split;
  for (int base = row0; base < row1; base += kSlots / split) {
    const int r = base + slot / split;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    bool sees = false;
    if (r < row1) {
      for (int p0 = g; p0 < parts; p0 += kFlight * split) {
        f32x2 st[kFlight];
        f32x4 o[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const int p = p0 + i * split;
          const int64_t a = at(r, p < parts ? p : p0);
          st[i] = P.part_ml[a];
          o[i] = *reinterpret_cast<const f32x4*>(P.part_o + a * D + lane * 4);
          if (p >= parts) st[i] = f32x2{-INFINITY, 0.f};
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) mn = fmaxf(mn, st[i].x);
        const float shift = mn == -INFINITY ? 0.f : mn;
        const float a = __builtin_amdgcn_exp2f(m - shift);
        l *= a;
        acc *= a;
        m = mn;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const float w = __builtin_amdgcn_exp2f(st[i].x - shift);
          l += w * st[i].y;
          sees = sees || __float_as_uint(st[i].y) != 0;
          if (w != 0.f) acc += w * o[i];   // a part without keys has written no output
        }
      }
    }
    if (split > 1) {
      __syncthreads();
      so[slot][lane] = acc;
      if (lane == 0) {
        sm[slot] = m;
        sl[slot] = l;
        ss[slot] = sees;
      }
      __syncthreads();
      if (g == 0) {
        for (int x = 1; x < split; ++x) m = fmaxf(m, sm[slot + x]);
        const float shift = m == -INFINITY ? 0.f : m;
        l = 0.f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < split; ++x) {
          const float w = __builtin_amdgcn_exp2f(sm[slot + x] - shift);
          l += w * sl[slot + x];
          sees = sees || ss[slot + x];
          if (w != 0.f) acc += w * so[slot + x][lane];
        }
      }
    }
    if (g == 0 && r < row1) {
      const float inv = 1.0f / l;
      store4<T>(out(r), lane * 4, sees ? acc * inv : f32x4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// The item of a work list (qvl_decoder_items.h) that this workgroup computes; false if it is none or leaves its bounds.
struct Item {
  Unit u;
  int slot, t0, t1;   // slot < 0: whole
};
__device__ __forceinline__ bool item_of(const AttnParams& P, const int32_t* items, int n_parts, int rows, int keys, Item& x) {
  const int32_t* it = items + kItemWords * (int64_t)blockIdx.x;
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4], slot = it[5];
  const int64_t start = (int64_t)(((uint64_t)(uint32_t)it[7] << 32) | (uint32_t)it[6]);
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || len < 0 ||
      len > kItemMaxLen || start < 0 || start > P.kv_rows - len || row0 >= n_new * P.group || slot >= n_parts) return false;
  x.u = Unit{P.k.p + start * P.k.row + kvh * P.k.head, P.v.p + start * P.v.row + kvh * P.v.head, len, len - n_new + 1, q0,
             n_new * P.group, row0, kvh};
  x.slot = slot;
  const int last = min(row0 + rows, x.u.rows) - 1;
  const int k_hi = max(min(x.u.lim0 + (int)((uint32_t)last / (uint32_t)P.group), len), 0);
  x.t0 = max(it[8], 0);
  x.t1 = min(it[9], (k_hi + keys - 1) / keys);
  return true;
}

// Checks shared by the entries, and the views (qvl_causal.hip).
int attn_params(const char* what, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int64_t kv_rows, const void* out,
                int64_t out_row, int64_t out_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads,
                int32_t head_dim, float scale, AttnParams& P);

// KERNEL<T, D> of the entry's dtype and head_dim.
#define QVL_ATTN_LAUNCH(KERNEL, GRID, ...)                                                                              \
  do {                                                                                                                  \
    const dim3 grid = GRID;                                                                                             \
    hipStream_t st = (hipStream_t)stream;                                                                               \
    if (dtype == QVL_DTYPE_BF16) {                                                                                      \
      if (head_dim == 128) hipLaunchKernelGGL((KERNEL<bf16, 128>), grid, dim3(256), 0, st, __VA_ARGS__);                \
      else hipLaunchKernelGGL((KERNEL<bf16, 64>), grid, dim3(256), 0, st, __VA_ARGS__);                                 \
    } else {                                                                                                            \
      if (head_dim == 128) hipLaunchKernelGGL((KERNEL<float, 128>), grid, dim3(256), 0, st, __VA_ARGS__);               \
      else hipLaunchKernelGGL((KERNEL<float, 64>), grid, dim3(256), 0, st, __VA_ARGS__);                                \
    }                                                                                                                   \
  } while (0)

}  // namespace qvl
