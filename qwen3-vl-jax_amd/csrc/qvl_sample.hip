// The next token of rows of logits: temperature, top-k, top-p and min-p, from a given random number a row.
//
// With z = (x - max x) / T a token weighs W = round(2^44 e^z), a whole number: sums of them (below 2^62) do not depend on their order, so that
// atomics may form them and a row's token is a function of its inputs alone. Kept are, in the order of falling logits (equal ones:
// rising index), the first top_k; of them those before which less than top_p of their sum lies; of them those of W >= min_p 2^44.
// The token is the first index whose sum of kept weights up to it is over u times their whole sum.
//
// No row is sorted. z is cut into 2048 bins of 1/64 (beyond lie weights of 0), and a row's histogram, of counts for top-k and of weights for top-p,
// tells the bin the cut falls into; that bin's tokens (with top-k: all up to it) are listed, mostly some dozens, and
// ranked against each other. Where more than kList share it (a flat row, or equal logits) the cut is found by its bits, 8 at a
// time, over the row. The bins serve the weights too: e^z is a table's 2^44 e^(-bin / 64) times a short polynomial, in fp64 (an fp32 weight would
// be off by 2^20 of its units).
//
// Bound by reading the logits: three times where there is a cut (the maximum, the histogram, the list with the sums of segments of
// 1024 tokens), the second and third time from a cache.
#include "qvl_decoder.h"
#include "qvl_kernels.h"

namespace qvl {

constexpr int kBins = 2048, kSegment = 1024, kMaxSegments = 256, kList = 1024;
constexpr double kUnit = 17592186044416.0;   // 2^44

struct SampleParams {
  const char* x;
  int64_t row;                               // bytes
  int vocab, segments;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;        // where the pointers are NULL
  int32_t top_k1;
  int64_t* out;
};

struct Settings {
  double t, p, floor, u;                     // floor: the least weight
  int k;                                     // 0: no top-k
  bool greedy, nucleus;
};

__device__ __forceinline__ Settings settings_of(const SampleParams& P, int row) {
  Settings s;
  s.t = P.temperature ? P.temperature[row] : P.temperature1;
  s.p = P.top_p ? P.top_p[row] : P.top_p1;
  const double min_p = P.min_p ? P.min_p[row] : P.min_p1;
  s.k = max(P.top_k ? P.top_k[row] : P.top_k1, 0);
  s.u = P.u[row];
  if (!(s.u >= 0)) s.u = 0;
  s.nucleus = s.p < 1;
  s.floor = min_p > 0 ? min_p * kUnit : 0;
  // the first token in the order alone; elsewhere the rules keep it by themselves
  s.greedy = !(s.t > 0) || s.k == 1 || s.p <= 0 || min_p > 1;
  return s;
}

// Place in the order: smaller is earlier (a larger logit, then a smaller index).
__device__ __forceinline__ uint64_t place_of(float x, int index) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t key = b & 0x80000000u ? b : b ^ 0x7fffffffu;
  return (uint64_t)key << 32 | (uint32_t)index;
}
__device__ __forceinline__ float logit_of(uint64_t place) {
  const uint32_t key = (uint32_t)(place >> 32);
  return __uint_as_float(key & 0x80000000u ? key : key ^ 0x7fffffffu);
}

// Bin and weight of a logit; false: beyond the bins, weight 0 (-infinity too).
struct Weigher {
  double top, scale;                         // 64 / T
  const double* table;                       // 2^44 e^(-j / 64)
  __device__ __forceinline__ bool operator()(float x, int& bin, uint64_t& w) const {
    // (products and sums joined by hand, so that every pass over the row comes to the same weight)
    const double d = top - (double)x, y = d * scale;
    if (!(y < (double)(kBins - 1))) return false;
    bin = (int)y;
    const double r = __builtin_fma(d, scale, -(double)bin) * (-1.0 / 64);
    double e = __builtin_fma(r, 1.0 / 720, 1.0 / 120);
    e = __builtin_fma(e, r, 1.0 / 24);
    e = __builtin_fma(e, r, 1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    // (plus 2^52: rounded to a whole number, which the low bits then hold)
    w = (uint64_t)__double_as_longlong(__builtin_fma(table[bin], e, 0x1p52)) & 0xfffffffffffffull;
    return true;
  }
};

// A wave's values of a segment: element l * 64 V + lane V + e in x[l V + e], V values a load. Behind the row: -infinity.
template <typename T> struct Segment {
  static constexpr int V = 16 / (int)sizeof(T), kLoads = 16 / V;
  float x[16];
  static __device__ __forceinline__ int index(int i) { return i / V * 64 * V + (int)(threadIdx.x & 63) * V + i % V; }
  __device__ __forceinline__ void load(const char* row, int vocab, int segment) {
    const int base = segment * kSegment;
    if (base + kSegment <= vocab && ((uintptr_t)row & 15) == 0) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + (int64_t)(base + index(l * V)) * (int)sizeof(T));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (std::is_same<T, float>::value) {
            x[l * V + j] = __uint_as_float(w[j]);
          } else {
            x[l * V + 2 * j] = bf16_lo(w[j]);
            x[l * V + 2 * j + 1] = bf16_hi(w[j]);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = base + index(i);
        x[i] = at < vocab ? (float)reinterpret_cast<const T*>(row)[at] : -INFINITY;
      }
    }
  }
};

// Inclusive sums over the workgroup of NT threads; `waves`: NT / 64 words of LDS. Ends with a barrier that frees them.
template <int NT> __device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* waves, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = __shfl_up((unsigned long long)v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < wave) before += waves[i];
    total += waves[i];
  }
  __syncthreads();
  return v + before;
}

template <int NT> struct SampleLds {
  double table[kBins];
  uint64_t hist[kBins];
  uint64_t places[kList], weights[kList];
  uint64_t sums[kMaxSegments];
  uint64_t waves[NT / 64];
  uint64_t found[4];
  float tops[NT / 64];
  int n, bad, token;
};

// The largest logit of segments [s0, s1) (over the workgroup), and whether one is NaN or +infinity.
template <typename T, int NT, typename L>
__device__ __forceinline__ float largest_of(const char* row, int vocab, int s0, int s1, L& lds, bool& bad) {
  const int wave = threadIdx.x >> 6;
  float m = -INFINITY;
  bool b = false;
  for (int s = s0 + wave; s < s1; s += NT / 64) {
    Segment<T> g;
    g.load(row, vocab, s);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m = fmaxf(m, g.x[i]);
      b |= !(g.x[i] < INFINITY);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  if (threadIdx.x == 0) lds.bad = 0;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds.tops[wave] = m;
  if (b) lds.bad = 1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) m = fmaxf(m, lds.tops[i]);
  bad = lds.bad != 0;
  __syncthreads();
  return m;
}

// Runs f(x, index) for the elements of segments [s0, s1), and after(segment) behind each.
template <typename T, int NT, typename F, typename G>
__device__ __forceinline__ void over_segments(const char* row, int vocab, int s0, int s1, F&& f, G&& after) {
  for (int s = s0 + (int)(threadIdx.x >> 6); s < s1; s += NT / 64) {
    Segment<T> g;
    g.load(row, vocab, s);
#pragma unroll
    for (int i = 0; i < 16; ++i) f(g.x[i], s * kSegment + Segment<T>::index(i));
    after(s);
  }
}

template <int NT> __device__ __forceinline__ void fill_table(double* table) {
  for (int i = threadIdx.x; i < kBins; i += NT) table[i] = exp(i * (-1.0 / 64)) * kUnit;
}

// The bin that holds the cut: the first whose sum with those before reaches `enough` (the last, if none does); `before`: the sum before it.
template <int NT, typename L, typename F>
__device__ __forceinline__ int cut_bin(L& lds, uint64_t& before, F&& reached) {
  constexpr int kPer = kBins / NT;
  uint64_t own = 0, total;
#pragma unroll
  for (int j = 0; j < kPer; ++j) own += lds.hist[threadIdx.x * kPer + j];
  if (threadIdx.x == 0) {
    lds.n = kBins - 1;
    lds.found[0] = 0;
  }
  uint64_t upto = block_scan<NT>(own, lds.waves, total) - own;
  bool was = upto > 0 && reached(upto, total);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint64_t next = upto + lds.hist[threadIdx.x * kPer + j];
    const bool is = reached(next, total);
    const int bin = threadIdx.x * kPer + j;
    if ((is && !was) || (bin == kBins - 1 && !is)) {
      lds.n = bin;
      lds.found[0] = upto;
    }
    was = is;
    upto = next;
  }
  __syncthreads();
  const int bin = lds.n;
  before = lds.found[0];
  __syncthreads();
  return bin;
}

// The place of the token at which the cut lies, over the whole row, 8 bits of the place at a time: the first whose
// count (COUNT) or weight with all before it reaches what `reached` asks. Only places up to `most`.
template <typename T, int NT, bool COUNT, typename L, typename F>
__device__ __forceinline__ uint64_t cut_place(const SampleParams& P, const char* row, const Weigher& weigh, L& lds, uint64_t most, F&& reached) {
  uint64_t prefix = 0, base = 0;
  // the logit's 32 bits, then the index's 18
  for (int level = 0; level < 7; ++level) {
    const int shift = level < 4 ? 56 - 8 * level : 16 - 8 * (level - 4);
    __syncthreads();
    if (threadIdx.x < 256) lds.hist[threadIdx.x] = 0;
    __syncthreads();
    over_segments<T, NT>(row, P.vocab, 0, P.segments, [&](float x, int index) {
      int bin;
      uint64_t w;
      if (!weigh(x, bin, w)) return;
      const uint64_t at = place_of(x, index);
      if (at > most) return;
      if (level == 4 ? (at >> 32) == (prefix >> 32) : level > 0 ? (at >> (shift + 8)) == (prefix >> (shift + 8)) : true)
        atomicAdd((unsigned long long*)&lds.hist[(at >> shift) & 255], (unsigned long long)(COUNT ? 1 : w));
    }, [](int) {});
    __syncthreads();
    uint64_t total;
    const uint64_t own = threadIdx.x < 256 ? lds.hist[threadIdx.x] : 0;
    const uint64_t upto = block_scan<NT>(own, lds.waves, total);
    if (threadIdx.x == 0) lds.found[0] = 256;
    __syncthreads();
    // the first bin that reaches it (of those that hold anything, the last where none does)
    if (threadIdx.x < 256 && own > 0 && reached(base + upto)) atomicMin((unsigned long long*)&lds.found[0], (unsigned long long)threadIdx.x);
    __syncthreads();
    if (threadIdx.x == 0) lds.found[2] = 0;
    __syncthreads();
    if (lds.found[0] == 256 && threadIdx.x < 256 && own > 0) atomicMax((unsigned long long*)&lds.found[2], (unsigned long long)threadIdx.x);
    __syncthreads();
    const int bin = (int)(lds.found[0] < 256 ? lds.found[0] : lds.found[2]);
    if ((int)threadIdx.x == bin) lds.found[1] = upto - own;
    __syncthreads();
    base += lds.found[1];
    prefix |= (uint64_t)bin << shift;
  }
  __syncthreads();
  return prefix;
}

// The token of a row, once the sums of its segments' kept weights stand in lds.sums: kept are the places up to `last`
// whose weight is no less than the floor.
template <typename T, int NT, typename L>
__device__ __forceinline__ void choose(const SampleParams& P, const Settings& st, const char* row, const Weigher& weigh, uint64_t last, L& lds, int64_t* out) {
  uint64_t total, upto = 0;
  const uint64_t own = (int)threadIdx.x < P.segments ? lds.sums[threadIdx.x] : 0;
  __syncthreads();
  upto = block_scan<NT>(own, lds.waves, total);
  double t = st.u * (double)total;
  if (!(t < (double)total)) t = (double)(total - 1);
  if ((double)upto > t && !((double)(upto - own) > t)) {
    lds.n = threadIdx.x;
    lds.found[0] = upto - own;
  }
  if (threadIdx.x == 0) lds.token = 0x7fffffff;
  __syncthreads();
  const int segment = lds.n;
  uint64_t base = lds.found[0];
  for (int part = 0; part < kSegment; part += NT) {
    const int index = segment * kSegment + part + threadIdx.x;
    uint64_t w = 0, whole;
    int bin;
    if (index < P.vocab) {
      const float x = (float)reinterpret_cast<const T*>(row)[index];
      if (!weigh(x, bin, w) || place_of(x, index) > last || (double)w < st.floor) w = 0;
    }
    const uint64_t sum = base + block_scan<NT>(w, lds.waves, whole);
    if (w > 0 && (double)sum > t) atomicMin(&lds.token, index);
    base += whole;
  }
  __syncthreads();
  if (threadIdx.x == 0) *out = lds.token;
}

// The lowest index of the largest logit.
template <typename T, int NT, typename L>
__device__ __forceinline__ void choose_first(const SampleParams& P, const char* row, float top, L& lds, int64_t* out) {
  if (threadIdx.x == 0) lds.token = 0x7fffffff;
  __syncthreads();
  over_segments<T, NT>(row, P.vocab, 0, P.segments, [&](float x, int index) {
    if (x == top) atomicMin(&lds.token, index);
  }, [](int) {});
  __syncthreads();
  if (threadIdx.x == 0) *out = lds.token;
}

// Sums of the segments' kept weights: places up to `last`, weights from the floor on.
template <typename T, int NT, typename L>
__device__ __forceinline__ void segment_sums(const SampleParams& P, const Settings& st, const char* row, const Weigher& weigh, uint64_t last, L& lds) {
  uint64_t sum = 0;
  over_segments<T, NT>(row, P.vocab, 0, P.segments, [&](float x, int index) {
    int bin;
    uint64_t w;
    if (weigh(x, bin, w) && place_of(x, index) <= last && !((double)w < st.floor)) sum += w;
  }, [&](int s) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor((unsigned long long)sum, d);
    if ((threadIdx.x & 63) == 0) lds.sums[s] = sum;
    sum = 0;
  });
}

// One workgroup a row, everything by the bits of the places.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(SampleParams P) {
  __shared__ SampleLds<NT> lds;
  const char* row = P.x + (int64_t)blockIdx.x * P.row;
  int64_t* out = P.out + blockIdx.x;
  const Settings st = settings_of(P, blockIdx.x);
  bool bad;
  const float top = largest_of<T, NT>(row, P.vocab, 0, P.segments, lds, bad);
  if (bad || !(top > -INFINITY)) {           // NaN, +infinity, or nothing to choose from
    if (threadIdx.x == 0) *out = -1;
    return;
  }
  if (st.greedy) {
    choose_first<T, NT>(P, row, top, lds, out);
    return;
  }
  fill_table<NT>(lds.table);
  __syncthreads();
  const Weigher weigh{top, 64.0 / st.t, lds.table};
  uint64_t last = ~0ull;
  if (st.k > 0) last = cut_place<T, NT, true>(P, row, weigh, lds, last, [&](uint64_t n) { return n >= (uint64_t)st.k; });
  if (st.nucleus) {
    segment_sums<T, NT>(P, Settings{st.t, st.p, 0.0, st.u, st.k, false, true}, row, weigh, last, lds);
    __syncthreads();
    uint64_t whole;
    block_scan<NT>((int)threadIdx.x < P.segments ? lds.sums[threadIdx.x] : 0, lds.waves, whole);
    last = cut_place<T, NT, false>(P, row, weigh, lds, last, [&](uint64_t w) { return !((double)w < st.p * (double)whole); });
  }
  segment_sums<T, NT>(P, st, row, weigh, last, lds);
  __syncthreads();
  choose<T, NT>(P, st, row, weigh, last, lds, out);
}

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_sample_tokens(void* stream, int32_t dtype, const void* logits, int64_t row_stride, int64_t n_rows, int64_t vocab, const float* u,
                      const float* d_temperature, float temperature, const int32_t* d_top_k, int32_t top_k, const float* d_top_p,
                      float top_p, const float* d_min_p, float min_p, int64_t* out) {
  const char* what = "sample_tokens";
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (n_rows < 0 || vocab <= 0 || row_stride < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (vocab > kMaxSegments * kSegment) return set_error(QVL_ERR_UNSUPPORTED, "%s: %lld tokens (at most %d)", what, (long long)vocab, kMaxSegments * kSegment);
  if (n_rows > 0x7fffffffLL || row_stride > (int64_t)1 << 40) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (n_rows == 0) return QVL_OK;
  if (!logits || !u || !out) return set_error(QVL_ERR_INVALID_ARG, "%s: NULL pointer", what);
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  if ((uintptr_t)logits % size || (uintptr_t)out % 8 || (uintptr_t)u % 4 || (uintptr_t)d_temperature % 4 || (uintptr_t)d_top_k % 4 ||
      (uintptr_t)d_top_p % 4 || (uintptr_t)d_min_p % 4) return set_error(QVL_ERR_MISALIGNED, "%s: a pointer", what);
  const SampleParams P{(const char*)logits, row_stride * size, (int)vocab, (int)((vocab + kSegment - 1) / kSegment), u, d_temperature,
                       d_top_p, d_min_p, d_top_k, temperature, top_p, min_p, top_k, out};
  const dim3 grid((unsigned)n_rows);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == QVL_DTYPE_BF16) hipLaunchKernelGGL((sample_row_kernel<bf16, 1024>), grid, dim3(1024), 0, st, P);
  else hipLaunchKernelGGL((sample_row_kernel<float, 1024>), grid, dim3(1024), 0, st, P);
  return check_launch(what);
}

}  // extern "C"
