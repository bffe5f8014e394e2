// Keys and values of new tokens into the pages of the 4-bit cache, with the per-head RMSNorm and (t, h, w) rotation of q and k on the
// way (the formulas of qvl_text_rotary.hip), and pages read back as rows.
//
// A group x of 64 values: s = bf16(fp32(max|x| / 6)), and for each value the number nearest to |x| / s; a tie goes to the even code. A
// code is a step function: an error of one rounding next to a border moves it by a whole step. So it is decided exactly for a value that
// is stored as it came, and a normalised and rotated key is formed in fp64 (sines and cosines too), so that the order of a sum can move only
// what lies within some 1e-15 of a border. fp64 runs at fp32's rate here, and only keys need it.
//
// Each value is read once, q and 4.25 bits a value of k and v are written; what keeps it from the copy's rate is the keys' fp64 (88
// registers: 5 waves a SIMD) and the lookup of the place before the stores. 18011 tokens of 32 + 8 + 8 heads of 128, bf16: 105 us, 3.7 TB/s
// (as they are, 24001 tokens of 8 + 8 heads: 37 us, 3.3 TB/s); 64 tokens: 4.7 us. Reading back: 31014 tokens of 8 + 8 heads of 128 as
// bf16 26 us, 6.0 TB/s. Eight lanes hold a head, as in
// qvl_text_rotary.hip, and a wave eight heads of one token and one kind (q, k or v), so that no wave takes two paths; the four waves of a
// workgroup take four tokens in a row, whose 4-byte pieces of V lie side by side.
#include "qvl_decoder.h"
#include "qvl_paged.h"
#include "qvl_rotary.h"

namespace qvl {

// cos and sin of f / 2^64 turns in fp64: the nearest quarter turn, then the Taylor sums to x^17 and x^16 (|x| <= pi/4 leaves 2e-18).
__device__ __forceinline__ void sincos_turns64(uint64_t f, double& c, double& s) {
  const uint32_t quarter = (uint32_t)((f + (1ull << 61)) >> 62);
  const double x = (double)(int64_t)(f - ((uint64_t)quarter << 62)) * (6.283185307179586476925 * 0x1p-64), z = x * x;
  double ps = 1.0 / 355687428096000.0, pc = 1.0 / 20922789888000.0;
  ps = __builtin_fma(ps, z, -1.0 / 1307674368000.0);
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  pc = __builtin_fma(pc, z, -0.5);
  const double sn = __builtin_fma(x * z, ps, x), cs = __builtin_fma(pc, z, 1.0);
  const double a = (quarter & 1) ? cs : sn, b = (quarter & 1) ? sn : cs;
  s = (quarter & 2) ? -a : a;
  c = ((quarter + 1) & 2) ? -b : b;
}

// The sequence that row n is a token of (cu[i] <= n < cu[i + 1]; -1: of none), and the token's place in it. Up to 63 sequences are looked
// at by a lane each, their lengths on the way; more 64 at a time.
__device__ __forceinline__ int place_of(const int32_t* cu, const int32_t* k_len, int n_seqs, int64_t n, int64_t& t) {
  const int lane = threadIdx.x & 63;
  if (!cu) {
    t = (int64_t)k_len[n] - 1;
    return (int)n;
  }
  int lo = 0, size = n_seqs + 1;
  if (size <= 64) {
    const int first = cu[min(lane, n_seqs)], length = k_len[min(lane, n_seqs - 1)];
    const int seq = __popcll(__builtin_amdgcn_ballot_w64(lane < size && first <= n)) - 1;
    if (seq < 0 || seq >= n_seqs) return -1;
    t = (int64_t)__builtin_amdgcn_readlane(length, seq) - (__builtin_amdgcn_readlane(first, seq + 1) - n);
    return seq;
  }
  for (;;) {
    const int step = (size + 63) >> 6, at = lane * step;
    const bool in = at < size && cu[lo + at] <= n;
    const int c = __popcll(__builtin_amdgcn_ballot_w64(in));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    size = min(step, size - (c - 1) * step);
    if (step == 1) break;
  }
  if (lo >= n_seqs) return -1;
  t = (int64_t)k_len[lo] - (cu[lo + 1] - n);
  return lo;
}

// v of the lane that DPP control CTRL names.
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
  return __hiloint2double((int)dpp<CTRL>((uint32_t)__double2hiint(v)), (int)dpp<CTRL>((uint32_t)__double2loint(v)));
}
// Over the 8 lanes of a head: neighbours, neighbouring pairs, the halves mirrored.
template <typename R, typename F> __device__ __forceinline__ R over_head(R v, F&& f) {
  v = f(v, dpp<0xb1>(v));
  v = f(v, dpp<0x4e>(v));
  return f(v, dpp<0x141>(v));
}

// max|x| / 6 of a group of which each of a head's lanes holds E values (N = 2: and E more), rounded to fp32; not finite where a value is not.
// The bits of fp32 values order as their absolute values do, infinities and NaN above all.
template <int E, int N> __device__ __forceinline__ float sixth(const float (&x)[N][E]) {
  uint32_t m = 0;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < E; ++i) m = max(m, __float_as_uint(x[n][i]) & 0x7fffffffu);
  return __uint_as_float(over_head(m, [](uint32_t a, uint32_t b) { return max(a, b); })) / 6.0f;
}
template <int E, int N> __device__ __forceinline__ float sixth(const double (&x)[N][E]) {
  double m = 0, wrong = 0;                     // wrong: NaN where a value is not finite
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      m = fmax(m, fabs(x[n][i]));
      wrong = __builtin_fma(x[n][i], 0.0, wrong);
    }
  m = over_head(m, [](double a, double b) { return fmax(a, b); });
  wrong = over_head(wrong, [](double a, double b) { return a + b; });
  return (float)((m + wrong) / 6.0);
}

// The group's scale as bf16 bits, NaN where the group holds what is not finite (or is beyond it).
__device__ __forceinline__ uint32_t scale_bits(float s) {
  asm volatile("" : "+v"(s));   // rounded to fp32 first: the compiler makes one rounding of the two (7 of 288000 groups differ)
  const uint32_t b = pack_bf16x2(s, 0.f) & 0xffffu;
  return b < 0x7f80u ? b : 0x7fc0u;
}

// The codes of E values x of a group of that scale, 4 bits each: x / s to the nearest of the numbers by the conversion to e2m1 (ties to
// the even code, beyond 6 to 6), from an fp32 quotient that lies on a border between two codes only where x / s does.
// fp32: the quotient rounded to nearest is such a one (s has 8 bits and a border 3, so x / s that is not a border differs from it by 2^-24 of it
// or more); q = x (1/s), then its remainder times 1/s added, is rounded so, 1/s being. Far from the ends of the exponents, that is: tiny
// groups are brought up by 2^64 first.
template <int E> __device__ __forceinline__ uint32_t codes_of(const float (&x)[E], uint32_t scale) {
  float s = __uint_as_float(scale << 16);
  const float up = s < 0x1p-60f ? 0x1p64f : 1.0f;
  s *= up;
  const float inverse = s > 0.f ? 1.0f / s : 0.f;
  uint32_t w = 0;
  float q[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float a = x[i] * up, q0 = a * inverse;
    q[i] = __builtin_fmaf(-__builtin_fmaf(q0, s, -a), inverse, q0);   // (zeros keep their sign)
  }
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.0f, 1);
  if constexpr (E == 8) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.0f, 3);
  }
  return w;
}
// fp64: cut to the upper word's 20 bits, the last of them set where anything was cut off, the quotient is exact in fp32.
template <int E> __device__ __forceinline__ uint32_t codes_of(const double (&x)[E], uint32_t scale) {
  const double s = (double)__uint_as_float(scale << 16), inverse = s > 0 ? 1.0 / s : 0.0;
  uint32_t w = 0;
  float q[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const double t = x[i] * inverse;
    q[i] = (float)__hiloint2double(__double2hiint(t) | (int)min((uint32_t)__double2loint(t), 1u), 0);
  }
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.0f, 1);
  if constexpr (E == 8) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.0f, 3);
  }
  return w;
}

struct PagedAppendParams {
  HeadsView q, k, v, qo;
  const float *qw, *kw;
  double eps;
  const int32_t* pos;
  int64_t pos_stride;
  const uint64_t* table;
  const int32_t *cu_q, *k_len;
  Pages pages;
  int64_t n_tokens;
  int n_seqs, hq, hkv, q_chunks, kv_chunks, chunks;   // chunks: of 8 heads, of q, then k, then v
};

// A lane's codes of a key or value and their scales, to its token's place.
template <int D, bool K> __device__ __forceinline__ void store_codes(char* block, int token, int p, uint32_t lo, uint32_t hi,
                                                                     uint32_t scale_lo, uint32_t scale_hi) {
  using B = PageBlock<D>;
  if constexpr (D == 128) {
    if constexpr (K) {
      *reinterpret_cast<u32x2*>(block + B::k_piece(token, p)) = u32x2{lo, hi};
    } else {
      *reinterpret_cast<uint32_t*>(block + B::v_word(token, 2 * p)) = (lo & 0xffffu) | hi << 16;
      *reinterpret_cast<uint32_t*>(block + B::v_word(token, 2 * p + 1)) = lo >> 16 | (hi & 0xffff0000u);
    }
    if (p == 0) *reinterpret_cast<uint32_t*>(block + (K ? B::k_scale(token) : B::v_scale(token))) = scale_lo | scale_hi << 16;
  } else {
    if constexpr (K) {
      *reinterpret_cast<uint32_t*>(block + B::k_piece(token, p)) = lo | hi << 16;
    } else {
      *reinterpret_cast<uint16_t*>(block + B::v_word(token, p)) = (uint16_t)lo;
      *reinterpret_cast<uint16_t*>(block + B::v_word(token, 8 + p)) = (uint16_t)hi;
    }
    if (p == 0) *reinterpret_cast<uint16_t*>(block + (K ? B::k_scale(token) : B::v_scale(token))) = (uint16_t)scale_lo;
  }
}

template <int D, bool K, typename R, int E>
__device__ __forceinline__ void pack_head(char* block, int token, int p, const R (&x)[2][E]) {
  uint32_t sl, sh;
  if constexpr (D == 128) {
    const R lo[1][E] = {{x[0][0], x[0][1], x[0][2], x[0][3], x[0][4], x[0][5], x[0][6], x[0][7]}};
    const R hi[1][E] = {{x[1][0], x[1][1], x[1][2], x[1][3], x[1][4], x[1][5], x[1][6], x[1][7]}};
    sl = scale_bits(sixth<E, 1>(lo));
    sh = scale_bits(sixth<E, 1>(hi));
  } else {
    sl = sh = scale_bits(sixth<E, 2>(x));
  }
  store_codes<D, K>(block, token, p, codes_of<E>(x[0], sl), codes_of<E>(x[1], sh), sl, sh);
}

template <typename T, int D, bool ROTATE>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams P) {
  constexpr int E = D / 16;                   // values of each half a lane holds
  constexpr int kWords = E * (int)sizeof(T) / 4, kHalfBytes = D / 2 * (int)sizeof(T);
  __shared__ double cs_all[4][D / 2][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = lane & 7;
  const int64_t n = (int64_t)(blockIdx.x / (uint32_t)P.chunks) * 4 + wave;
  const int chunk = blockIdx.x % (uint32_t)P.chunks;
  if (n >= P.n_tokens) return;
  const bool is_q = chunk < P.q_chunks, is_k = !is_q && chunk < P.q_chunks + P.kv_chunks;
  const int h = (is_q ? chunk : is_k ? chunk - P.q_chunks : chunk - P.q_chunks - P.kv_chunks) * 8 + (lane >> 3);
  const bool live = h < (is_q ? P.hq : P.hkv);
  const HeadsView in = is_q ? P.q : is_k ? P.k : P.v;
  const char* src = in.p + n * in.row + h * in.head + part * E * (int)sizeof(T);
  // everything that a lane reads is asked for before the first of it is waited for
  uint32_t lo_words[kWords], hi_words[kWords];
  if (live) {
    load_words(src, lo_words);
    load_words(src + kHalfBytes, hi_words);
  }
  const bool turn = ROTATE && (is_q || is_k);
  uint64_t turns = 0, axis = 0;
  int32_t pos[3] = {0, 0, 0};
  float w[2][E];
  if (turn) {
    const int f = min(lane, D / 2 - 1);
    turns = P.table[2 * f];
    axis = P.table[2 * f + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) pos[i] = P.pos[i * P.pos_stride + n];
    const float* weights = (is_q ? P.qw : P.kw) + part * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      w[0][i] = weights[i];
      w[1][i] = weights[D / 2 + i];
    }
  }
  int64_t t;
  const int seq = place_of(P.cu_q, P.k_len, P.n_seqs, n, t);
  if (seq < 0) return;
  char* block = nullptr;
  if (!is_q) {
    const int page = t < 0 ? -1 : P.pages.page(seq, t >> P.pages.shift);
    if (page < 0) return;
    block = P.pages.block<D>(page, min(h, P.hkv - 1), (int)t);
  }
  const int token = (int)t & 15;
  if (turn) {
    const uint64_t angle = (uint64_t)(int64_t)(axis == 0 ? pos[0] : axis == 1 ? pos[1] : pos[2]) * turns;
    if (lane < D / 2) {
      if (is_q) {
        float c, s;
        sincos_turns(angle, c, s);
        reinterpret_cast<f32x2*>(cs_all[wave])[lane] = f32x2{c, s};
      } else {
        sincos_turns64(angle, cs_all[wave][lane][0], cs_all[wave][lane][1]);
      }
    }
    __builtin_amdgcn_wave_barrier();            // the wave's own LDS: written and read in its program order
  }
  if (!live) return;
  float x[2][E];
  float(&lo)[E] = x[0], (&hi)[E] = x[1];
  values_of<T, E>(lo_words, lo);
  values_of<T, E>(hi_words, hi);
  if constexpr (ROTATE) {
    if (is_q) {                                 // as qk_norm_rotary_kernel
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
      ss += __shfl_xor(ss, 1);
      ss += __shfl_xor(ss, 2);
      ss += __shfl_xor(ss, 4);
      const float r = 1.0f / sqrtf(ss * (1.0f / D) + (float)P.eps);
      float yl[E], yh[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const f32x2 cs = reinterpret_cast<const f32x2*>(cs_all[wave])[part * E + i];
        const float a = lo[i] * r * w[0][i], b = hi[i] * r * w[1][i];
        yl[i] = a * cs.x - b * cs.y;
        yh[i] = b * cs.x + a * cs.y;
      }
      char* dst = P.qo.p + n * P.qo.row + h * P.qo.head + part * E * (int)sizeof(T);
      store_vals<T, E>(dst, yl);
      store_vals<T, E>(dst + kHalfBytes, yh);
      return;
    }
    if (is_k) {
      double ss = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += (double)lo[i] * lo[i] + (double)hi[i] * hi[i];
      ss = over_head(ss, [](double a, double b) { return a + b; });
      const double r = 1.0 / sqrt(ss * (1.0 / D) + P.eps);
      double y[2][E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const double c = cs_all[wave][part * E + i][0], s = cs_all[wave][part * E + i][1];
        const double a = lo[i] * r * w[0][i], b = hi[i] * r * w[1][i];
        y[0][i] = a * c - b * s;
        y[1][i] = b * c + a * s;
      }
      pack_head<D, true>(block, token, part, y);
      return;
    }
  }
  if (is_k) pack_head<D, true>(block, token, part, x);
  else pack_head<D, false>(block, token, part, x);
}

// A block of 16 tokens and one head a wave, 8 tokens at a time, 8 lanes a token; the lanes' codes lie as the append wrote them.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_unpack_kernel(Pages pages, const int32_t* first_, const int32_t* k_len, const int64_t* k_start,
                                                           HeadsView k, HeadsView v, int64_t out_rows) {
  using B = PageBlock<D>;
  constexpr int E = D / 16;
  const int lane = threadIdx.x & 63, p = lane & 7, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, seq = blockIdx.z;
  const int64_t first = first_ ? first_[seq] : 0, row0 = k_start[seq];
  // tokens whose rows lie in [0, out_rows); token t's is t + shift (first and t have 32 bits)
  if (row0 >= out_rows || row0 < -((int64_t)1 << 32)) return;
  const int64_t shift = row0 - first, from = max(max(first, (int64_t)0), -shift), end = min((int64_t)k_len[seq], out_rows - shift);
  for (int64_t b = (from >> 4) + blockIdx.x * 4 + wave; b * 16 < end; b += gridDim.x * 4) {
    const int page = pages.page(seq, b >> (pages.shift - 4));
    const char* block = pages.block<D>(max(page, 0), h, (int)(b << 4));
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int token = half * 8 + (lane >> 3);
      const int64_t t = b * 16 + token, row = t + shift;
      if (t < from || t >= end) continue;
      uint32_t codes[2][2] = {}, scales[2] = {0x7fc07fc0u, 0x7fc07fc0u};   // [k, v][lo, hi]; a page of none: NaN
      if (page < 0) {
      } else if constexpr (D == 128) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(block + B::k_piece(token, p));
        const uint32_t a = *reinterpret_cast<const uint32_t*>(block + B::v_word(token, 2 * p)),
                       c = *reinterpret_cast<const uint32_t*>(block + B::v_word(token, 2 * p + 1));
        codes[0][0] = w[0];
        codes[0][1] = w[1];
        codes[1][0] = (a & 0xffffu) | c << 16;
        codes[1][1] = a >> 16 | (c & 0xffff0000u);
        scales[0] = *reinterpret_cast<const uint32_t*>(block + B::k_scale(token));
        scales[1] = *reinterpret_cast<const uint32_t*>(block + B::v_scale(token));
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(block + B::k_piece(token, p));
        codes[0][0] = w;
        codes[0][1] = w >> 16;
        codes[1][0] = *reinterpret_cast<const uint16_t*>(block + B::v_word(token, p));
        codes[1][1] = *reinterpret_cast<const uint16_t*>(block + B::v_word(token, 8 + p));
        scales[0] = *reinterpret_cast<const uint16_t*>(block + B::k_scale(token)) * 0x10001u;
        scales[1] = *reinterpret_cast<const uint16_t*>(block + B::v_scale(token)) * 0x10001u;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const HeadsView& to = x ? v : k;
        char* dst = to.p + row * to.row + h * to.head + p * E * (int)sizeof(T);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float s = y ? bf16_hi(scales[x]) : bf16_lo(scales[x]);
          float f[E];
          const f32x2 n0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[x][y], 1.0f, 0);
          const f32x2 n1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[x][y], 1.0f, 1);
          f[0] = n0[0] * s;
          f[1] = n0[1] * s;
          f[2] = n1[0] * s;
          f[3] = n1[1] * s;
          if constexpr (E == 8) {
            const f32x2 n2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[x][y], 1.0f, 2);
            const f32x2 n3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[x][y], 1.0f, 3);
            f[4] = n2[0] * s;
            f[5] = n2[1] * s;
            f[6] = n3[0] * s;
            f[7] = n3[1] * s;
          }
          store_vals<T, E>(dst + y * (D / 2) * (int)sizeof(T), f);
        }
      }
    }
  }
}

int pages_of(const char* what, const void* data, int64_t n_pages, int32_t page_rows, const int32_t* table, int64_t table_width,
             int64_t table_stride, int64_t n_seqs, int32_t num_kv_heads, int32_t head_dim, Pages& out) {
  if (head_dim != 64 && head_dim != 128) return set_error(QVL_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", what, head_dim);
  if (page_rows < 16 || page_rows > 4096 || (page_rows & (page_rows - 1)))
    return set_error(QVL_ERR_UNSUPPORTED, "%s: %d rows a page (a power of two, 16 to 4096)", what, page_rows);
  if (n_pages < 0 || table_width < 0 || table_stride < 0 || n_seqs < 0 || num_kv_heads <= 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_pages > 0x7fffffffLL || table_width > 0x7fffffffLL || table_stride > (int64_t)1 << 40 || n_seqs > 65535 || num_kv_heads > 4096)
    return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (n_pages > 0 && !data) return set_error(QVL_ERR_INVALID_ARG, "%s: the cache is NULL", what);
  if (n_seqs > 0 && table_width > 0 && !table) return set_error(QVL_ERR_INVALID_ARG, "%s: the page table is NULL", what);
  if ((uintptr_t)data % 64 || (uintptr_t)table % 4) return set_error(QVL_ERR_MISALIGNED, "%s: the cache (64 bytes) or the page table", what);
  out = Pages{(char*)const_cast<void*>(data), table, table_stride, n_pages > 0 ? (int)table_width : 0, (int)n_pages,
              __builtin_ctz((unsigned)page_rows), num_kv_heads};
  return QVL_OK;
}

}  // namespace qvl

using namespace qvl;

namespace {
struct NamedView { const char* name; const void* p; int64_t row, head; };
int check_views(const char* what, int64_t size, const NamedView* views, int n) {
  for (int i = 0; i < n; ++i) {
    const NamedView& w = views[i];
    if (!w.p) return set_error(QVL_ERR_INVALID_ARG, "%s: %s is NULL", what, w.name);
    if (w.row < 0 || w.head < 0 || w.row > 0x7fffffffLL || w.head > 0x7fffffffLL)
      return set_error(QVL_ERR_INVALID_ARG, "%s: strides of %s", what, w.name);
    if ((uintptr_t)w.p % 16 || w.row * size % 16 || w.head * size % 16)
      return set_error(QVL_ERR_MISALIGNED, "%s: %s and its strides must be multiples of 16 bytes", what, w.name);
  }
  return QVL_OK;
}
}  // namespace

extern "C" {

int qvl_paged_cache_size(int64_t n_pages, int32_t page_rows, int32_t num_kv_heads, int32_t head_dim, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "paged_cache_size: bytes is NULL");
  Pages pages;
  QVL_TRY_RC(pages_of("paged_cache_size", (const void*)64, n_pages, page_rows, nullptr, 0, 0, 0, num_kv_heads, head_dim, pages));
  *bytes = (size_t)n_pages * num_kv_heads * (page_rows / 16) * (head_dim == 128 ? PageBlock<128>::kBytes : PageBlock<64>::kBytes);
  return QVL_OK;
}

int qvl_paged_append(void* stream, int32_t dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                     int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const float* q_norm, const float* k_norm, double eps,
                     const int32_t* positions, int64_t pos_stride, const uint64_t* table, void* cache, int64_t n_pages,
                     int32_t page_rows, const int32_t* page_table, int64_t table_width, int64_t table_stride, const int32_t* cu_q,
                     int64_t n_seqs, const int32_t* k_len, void* q_out, int64_t qo_row, int64_t qo_head, int64_t n_tokens,
                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  const char* what = "paged_append";
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  PagedAppendParams P{};
  QVL_TRY_RC(pages_of(what, cache, n_pages, page_rows, page_table, table_width, table_stride, n_seqs, num_kv_heads, head_dim, P.pages));
  const bool rotate = q != nullptr;
  if (n_tokens < 0 || pos_stride < 0 || (rotate && (num_heads <= 0 || !(eps >= 0)))) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_tokens > 0x3fffffff || (rotate && num_heads > 4096)) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (!cu_q && n_tokens != n_seqs)
    return set_error(QVL_ERR_INVALID_ARG, "%s: %lld tokens of %lld sequences without cu_q", what, (long long)n_tokens, (long long)n_seqs);
  if (n_tokens == 0 || n_seqs == 0) return QVL_OK;
  if (!k_len || (rotate && (!q_norm || !k_norm || !positions || !table))) return set_error(QVL_ERR_INVALID_ARG, "%s: NULL pointer", what);
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  const NamedView views[] = {{"k", k, k_row, k_head}, {"v", v, v_row, v_head}, {"q", q, q_row, q_head}, {"q_out", q_out, qo_row, qo_head}};
  QVL_TRY_RC(check_views(what, size, views, rotate ? 4 : 2));
  if ((uintptr_t)k_len % 4 || (uintptr_t)cu_q % 4 || (uintptr_t)q_norm % 4 || (uintptr_t)k_norm % 4 || (uintptr_t)positions % 4 || (uintptr_t)table % 8)
    return set_error(QVL_ERR_MISALIGNED, "%s: norms, table, positions or the sequences' state", what);
  auto view = [&](const void* p, int64_t row, int64_t head) { return HeadsView{(char*)const_cast<void*>(p), row * size, head * size}; };
  P.q = view(q, q_row, q_head);
  P.k = view(k, k_row, k_head);
  P.v = view(v, v_row, v_head);
  P.qo = view(q_out, qo_row, qo_head);
  P.qw = q_norm;
  P.kw = k_norm;
  P.eps = eps;
  P.pos = positions;
  P.pos_stride = pos_stride;
  P.table = table;
  P.cu_q = cu_q;
  P.k_len = k_len;
  P.n_tokens = n_tokens;
  P.n_seqs = (int)n_seqs;
  P.hq = rotate ? num_heads : 0;
  P.hkv = num_kv_heads;
  P.q_chunks = (P.hq + 7) / 8;
  P.kv_chunks = (num_kv_heads + 7) / 8;
  P.chunks = P.q_chunks + 2 * P.kv_chunks;
  const int64_t blocks = (n_tokens + 3) / 4 * P.chunks;
  if (blocks > 0x7fffffffLL) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  const dim3 grid((unsigned)blocks);
  hipStream_t st = (hipStream_t)stream;
#define QVL_APPEND(T, D)                                                                                    \
  do {                                                                                                      \
    if (rotate) hipLaunchKernelGGL((paged_append_kernel<T, D, true>), grid, dim3(256), 0, st, P);           \
    else hipLaunchKernelGGL((paged_append_kernel<T, D, false>), grid, dim3(256), 0, st, P);                 \
  } while (0)
  if (dtype == QVL_DTYPE_BF16) {
    if (head_dim == 128) QVL_APPEND(bf16, 128);
    else QVL_APPEND(bf16, 64);
  } else {
    if (head_dim == 128) QVL_APPEND(float, 128);
    else QVL_APPEND(float, 64);
  }
#undef QVL_APPEND
  return check_launch(what);
}

int qvl_paged_unpack(void* stream, int32_t dtype, const void* cache, int64_t n_pages, int32_t page_rows, const int32_t* page_table,
                     int64_t table_width, int64_t table_stride, int64_t n_seqs, const int32_t* first, const int32_t* k_len,
                     int64_t max_len, const int64_t* k_start, void* k, int64_t k_row, int64_t k_head, void* v, int64_t v_row,
                     int64_t v_head, int64_t out_rows, int32_t num_kv_heads, int32_t head_dim) {
  const char* what = "paged_unpack";
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  Pages pages;
  QVL_TRY_RC(pages_of(what, cache, n_pages, page_rows, page_table, table_width, table_stride, n_seqs, num_kv_heads, head_dim, pages));
  if (max_len < 0 || out_rows < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (max_len > 0x3fffffff || out_rows > (int64_t)1 << 40) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (n_seqs == 0 || out_rows == 0) return QVL_OK;
  if (!k_len || !k_start) return set_error(QVL_ERR_INVALID_ARG, "%s: NULL pointer", what);
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  const NamedView views[] = {{"k", k, k_row, k_head}, {"v", v, v_row, v_head}};
  QVL_TRY_RC(check_views(what, size, views, 2));
  if ((uintptr_t)k_len % 4 || (uintptr_t)first % 4 || (uintptr_t)k_start % 8) return set_error(QVL_ERR_MISALIGNED, "%s: the sequences' state", what);
  const HeadsView kv{(char*)k, k_row * size, k_head * size}, vv{(char*)v, v_row * size, v_head * size};
  // a wave for each block of 16 tokens, one more for a first token inside one; longer sequences go round
  const dim3 grid((unsigned)std::min<int64_t>((max_len / 16 + 2 + 3) / 4, 65535), (unsigned)num_kv_heads, (unsigned)n_seqs);
  hipStream_t st = (hipStream_t)stream;
#define QVL_UNPACK(T, D) hipLaunchKernelGGL((paged_unpack_kernel<T, D>), grid, dim3(256), 0, st, pages, first, k_len, k_start, kv, vv, out_rows)
  if (dtype == QVL_DTYPE_BF16) {
    if (head_dim == 128) QVL_UNPACK(bf16, 128);
    else QVL_UNPACK(bf16, 64);
  } else {
    if (head_dim == 128) QVL_UNPACK(float, 128);
    else QVL_UNPACK(float, 64);
  }
#undef QVL_UNPACK
  return check_launch(what);
}

}  // extern "C"
