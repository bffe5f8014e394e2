// Per-head RMSNorm of queries and keys and the (t, h, w) position rotation in one pass, keys and values written to cache
// rows. For a head x of D values at a token: y = x * rsqrt(mean(x^2) + eps) * w, then for j < D/2
//   (y_j, y_{j+D/2}) -> (y_j cos a_j - y_{j+D/2} sin a_j, y_{j+D/2} cos a_j + y_j sin a_j),  a_j = 2 pi pos f_j,
// f_j turns per position. pos * f_j is formed modulo 1 as a 64-bit integer product, which is exact to pos * 2^-64 turns;
// fp32 angles are off by whole radians from position 2^24 on and by 2^-9 of one at 2^15.
//
// Bound by memory: each value is read and written once. Eight lanes hold a head (both halves of each rotated pair in
// one lane, so the rotation crosses no lanes), a wave eight heads of one token; its 64 lanes compute the token's D/2
// sines and cosines once and pass them through LDS. 18011 tokens of 32 + 8 + 8 heads of 128, bf16: 84 us, 5.3 TB/s (a
// large copy: 4.9); 64 tokens: 3.8 us.
#include <type_traits>

#include "qvl_decoder.h"
#include "qvl_kernels.h"

namespace qvl {

struct HeadsView {
  char* p;
  int64_t row, head;   // strides in bytes
};

struct QkNormRotaryParams {
  HeadsView q, k, v, qo, ko, vo;
  const float *qw, *kw;
  float eps;
  const int32_t* pos;
  int64_t pos_stride;
  const uint64_t* table;
  const int64_t* rows;
  int64_t out_rows, n_tokens;
  int hq, hkv, heads, chunks;   // heads = hq + hkv (+ hkv with v), chunks = ceil(heads / 8)
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

template <typename T, int D>
__global__ __launch_bounds__(256) void qk_norm_rotary_kernel(QkNormRotaryParams P) {
  constexpr int E = D / 16;                   // values of each half a lane holds
  constexpr int kHalfBytes = D / 2 * (int)sizeof(T);
  __shared__ f32x2 cs_all[4][D / 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= P.n_tokens * P.chunks) return;
  const int64_t n = unit / P.chunks;
  const int head = (int)(unit % P.chunks) * 8 + (lane >> 3), part = lane & 7;
  const bool is_v = head >= P.hq + P.hkv, is_k = head >= P.hq && !is_v, live = head < P.heads;
  const HeadsView in = is_v ? P.v : is_k ? P.k : P.q, to = is_v ? P.vo : is_k ? P.ko : P.qo;
  const int h = is_v ? head - P.hq - P.hkv : is_k ? head - P.hq : head;
  const char* src = in.p + n * in.row + h * in.head + part * E * (int)sizeof(T);
  uint32_t lo_words[E * sizeof(T) / 4], hi_words[E * sizeof(T) / 4];
  if (live) {
    load_words(src, lo_words);
    load_words(src + kHalfBytes, hi_words);
  }
  if (lane < D / 2) {
    const uint64_t turns = P.table[2 * lane];
    const int axis = (int)min(P.table[2 * lane + 1], (uint64_t)2);
    const int32_t p = P.pos[axis * P.pos_stride + n];
    float c, s;
    sincos_turns((uint64_t)(int64_t)p * turns, c, s);
    cs_all[wave][lane] = f32x2{c, s};
  }
  __builtin_amdgcn_wave_barrier();            // the wave's own LDS: written and read in its program order
  if (!live) return;
  const int64_t row = head < P.hq || !P.rows ? n : P.rows[n];
  if (head >= P.hq && (row < 0 || row >= P.out_rows)) return;
  char* dst = to.p + row * to.row + h * to.head + part * E * (int)sizeof(T);
  if (is_v) {                                 // as bits: a conversion there and back would change a signalling NaN
    store_words(dst, lo_words);
    store_words(dst + kHalfBytes, hi_words);
    return;
  }
  float lo[E], hi[E];
  values_of<T, E>(lo_words, lo);
  values_of<T, E>(hi_words, hi);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
  ss += __shfl_xor(ss, 1);
  ss += __shfl_xor(ss, 2);
  ss += __shfl_xor(ss, 4);
  const float r = 1.0f / sqrtf(ss * (1.0f / D) + P.eps);
  const float* w = (is_k ? P.kw : P.qw) + part * E;
  uint32_t wl_words[E], wh_words[E];
  load_words(reinterpret_cast<const char*>(w), wl_words);
  load_words(reinterpret_cast<const char*>(w + D / 2), wh_words);
  float wl[E], wh[E], yl[E], yh[E];
  values_of<float, E>(wl_words, wl);
  values_of<float, E>(wh_words, wh);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const f32x2 cs = cs_all[wave][part * E + i];
    const float a = lo[i] * r * wl[i], b = hi[i] * r * wh[i];
    yl[i] = a * cs.x - b * cs.y;
    yh[i] = b * cs.x + a * cs.y;
  }
  store_vals<T, E>(dst, yl);
  store_vals<T, E>(dst + kHalfBytes, yh);
}

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_qk_norm_rotary(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k,
                       int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const float* q_norm,
                       const float* k_norm, float eps, const int32_t* positions, int64_t pos_stride,
                       const uint64_t* table, const int64_t* rows, int64_t out_rows, void* q_out, int64_t qo_row,
                       int64_t qo_head, void* k_out, int64_t ko_row, int64_t ko_head, void* v_out, int64_t vo_row,
                       int64_t vo_head, int64_t n_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "qk_norm_rotary: dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "qk_norm_rotary: head_dim=%d (64 or 128)", head_dim);
  if (n_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || out_rows < 0 || pos_stride < 0 || !(eps >= 0.f))
    return set_error(QVL_ERR_INVALID_ARG, "qk_norm_rotary: bad sizes");
  if (num_heads > 4096 || num_kv_heads > 4096 || n_tokens > 0x3fffffff)
    return set_error(QVL_ERR_UNSUPPORTED, "qk_norm_rotary: sizes");
  if (!rows && out_rows < n_tokens)
    return set_error(QVL_ERR_INVALID_ARG, "qk_norm_rotary: %lld output rows for %lld tokens", (long long)out_rows, (long long)n_tokens);
  if (!v != !v_out) return set_error(QVL_ERR_INVALID_ARG, "qk_norm_rotary: v without v_out or v_out without v");
  if (n_tokens == 0) return QVL_OK;
  if (!q || !k || !q_norm || !k_norm || !positions || !table || !q_out || !k_out)
    return set_error(QVL_ERR_INVALID_ARG, "qk_norm_rotary: NULL pointer");
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  struct { const char* what; const void* p; int64_t row, head; } views[] = {
      {"q", q, q_row, q_head}, {"k", k, k_row, k_head}, {"v", v, v_row, v_head},
      {"q_out", q_out, qo_row, qo_head}, {"k_out", k_out, ko_row, ko_head}, {"v_out", v_out, vo_row, vo_head}};
  for (auto& w : views) {
    if (!w.p) continue;
    if (w.row < 0 || w.head < 0 || w.row > 0x7fffffffLL || w.head > 0x7fffffffLL)
      return set_error(QVL_ERR_INVALID_ARG, "qk_norm_rotary: strides of %s", w.what);
    if ((uintptr_t)w.p % 16 || w.row * size % 16 || w.head * size % 16)
      return set_error(QVL_ERR_MISALIGNED, "qk_norm_rotary: %s and its strides must be multiples of 16 bytes", w.what);
  }
  if ((uintptr_t)q_norm % 16 || (uintptr_t)k_norm % 16 || (uintptr_t)table % 8 || (uintptr_t)rows % 8 || (uintptr_t)positions % 4)
    return set_error(QVL_ERR_MISALIGNED, "qk_norm_rotary: norms, table, rows or positions");
  auto view = [&](const void* p, int64_t row, int64_t head) { return HeadsView{(char*)const_cast<void*>(p), row * size, head * size}; };
  QkNormRotaryParams P{view(q, q_row, q_head), view(k, k_row, k_head), view(v, v_row, v_head), view(q_out, qo_row, qo_head),
                       view(k_out, ko_row, ko_head), view(v_out, vo_row, vo_head), q_norm, k_norm, eps, positions, pos_stride,
                       table, rows, out_rows, n_tokens, num_heads, num_kv_heads, 0, 0};
  P.heads = num_heads + (v ? 2 : 1) * num_kv_heads;
  P.chunks = (P.heads + 7) / 8;
  const int64_t blocks = (n_tokens * P.chunks + 3) / 4;
  if (blocks > 0x7fffffffLL) return set_error(QVL_ERR_UNSUPPORTED, "qk_norm_rotary: sizes");
  const dim3 grid((unsigned)blocks);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == QVL_DTYPE_BF16) {
    if (head_dim == 128) hipLaunchKernelGGL((qk_norm_rotary_kernel<bf16, 128>), grid, dim3(256), 0, st, P);
    else hipLaunchKernelGGL((qk_norm_rotary_kernel<bf16, 64>), grid, dim3(256), 0, st, P);
  } else {
    if (head_dim == 128) hipLaunchKernelGGL((qk_norm_rotary_kernel<float, 128>), grid, dim3(256), 0, st, P);
    else hipLaunchKernelGGL((qk_norm_rotary_kernel<float, 64>), grid, dim3(256), 0, st, P);
  }
  return check_launch("qk_norm_rotary");
}

}  // extern "C"
