// What the kernels that normalise and rotate heads share (qvl_text_rotary.hip, qvl_paged_cache.hip): the sines and cosines of
// fixed-point angles, and a lane's values in memory and as fp32.
#pragma once
#include <type_traits>

#include "qvl_kernels.h"

namespace qvl {

struct HeadsView {
  char* p;
  int64_t row, head;   // strides in bytes
};

// cos and sin of f / 2^64 turns. The nearest quarter turn leaves r in [-1/8, 1/8] turns; x = 2 pi r as a sum xh + xl
// (the product's rounding error and 2 pi's own), then the Taylor sums to x^9 and x^10: |x| <= pi/4 leaves 2e-9.
__device__ __forceinline__ void sincos_turns(uint64_t f, float& c, float& s) {
  const uint32_t quarter = (uint32_t)((f + (1ull << 61)) >> 62);
  const int64_t r = (int64_t)(f - ((uint64_t)quarter << 62));
  const float rt = __builtin_fmaf((float)(uint32_t)r, 0x1p-64f, (float)(int32_t)(r >> 32) * 0x1p-32f);
  constexpr float kTwoPi = 6.2831855f, kTwoPiLow = -1.7484556e-7f;   // 2 pi = kTwoPi + kTwoPiLow
  const float xh = rt * kTwoPi;
  const float xl = __builtin_fmaf(rt, kTwoPiLow, __builtin_fmaf(rt, kTwoPi, -xh));
  const float z = xh * xh;
  float ps = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040);
  ps = __builtin_fmaf(ps, z, 1.0f / 120);
  ps = __builtin_fmaf(ps, z, -1.0f / 6);
  float pc = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  pc = __builtin_fmaf(pc, z, -1.0f / 720);
  pc = __builtin_fmaf(pc, z, 1.0f / 24);
  pc = __builtin_fmaf(pc, z, -0.5f);
  const float sx = __builtin_fmaf(xh * z, ps, xh), cx = __builtin_fmaf(pc, z, 1.0f);
  const float sn = __builtin_fmaf(xl, cx, sx), cs = __builtin_fmaf(-xl, sx, cx);
  const float a = (quarter & 1) ? cs : sn, b = (quarter & 1) ? sn : cs;
  s = (quarter & 2) ? -a : a;
  c = ((quarter + 1) & 2) ? -b : b;
}

// N words at p, 16 bytes at a time (8 where there are no more).
template <int N> __device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[N]) {
  if constexpr (N == 2) *reinterpret_cast<u32x2*>(w) = *reinterpret_cast<const u32x2*>(p);
  else
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<u32x4*>(w + i) = *reinterpret_cast<const u32x4*>(p + 4 * i);
}
template <int N> __device__ __forceinline__ void store_words(char* p, const uint32_t (&w)[N]) {
  if constexpr (N == 2) *reinterpret_cast<u32x2*>(p) = *reinterpret_cast<const u32x2*>(w);
  else
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<u32x4*>(p + 4 * i) = *reinterpret_cast<const u32x4*>(w + i);
}

// E values of T in words as fp32, and back to memory (bf16 rounds to nearest even).
template <typename T, int E, int N> __device__ __forceinline__ void values_of(const uint32_t (&w)[N], float (&x)[E]) {
  static_assert(N * 4 == E * (int)sizeof(T), "E values");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      x[i] = __uint_as_float(w[i]);
    } else {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
}

template <typename T, int E> __device__ __forceinline__ void store_vals(char* p, const float (&x)[E]) {
  uint32_t w[E * sizeof(T) / 4];
#pragma unroll
  for (int i = 0; i < (int)(E * sizeof(T) / 4); ++i) {
    if constexpr (std::is_same<T, float>::value) w[i] = __float_as_uint(x[i]);
    else w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  }
  store_words(p, w);
}

}  // namespace qvl
