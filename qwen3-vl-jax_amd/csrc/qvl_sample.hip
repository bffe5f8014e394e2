// The next token of rows of logits: temperature, top-k, top-p and min-p, from a given random number a row.
//
// With z = (x - max x) / T a token weighs W = round(2^44 e^z), a whole number: sums of them (below 2^62) do not depend on their order, so that
// atomics may form them and a row's token is a function of its inputs alone. Kept are, in the order of falling logits (equal ones:
// rising index), the first top_k; of them those before which less than top_p of their sum lies; of them those of W >= min_p 2^44.
// The token is the first index whose sum of kept weights up to it is over u times their whole sum.
//
// No row is sorted. z is cut into bins of 1/32 of a power of two (beyond the last lie weights of 0), and a row's histogram, of counts for
// top-k and of weights for top-p, tells the bin that the cut falls into; that bin's tokens (with top-k: all up to it) are listed,
// mostly some dozens to hundreds, and only they are sorted. Where more than kList share it (a flat row, equal logits) the cut is
// found by the bits of its place in the order, 8 at a time, over the row. The bins serve the weights too: 2^44 e^z is one of 32 table
// entries times a short polynomial and a power of two, in fp64 (an fp32 weight would be off by 2^20 of its units).
//
// Four launches, each over (share of the vocabulary, row) but the last, which is over rows: the largest logits, the histogram, the
// list with the sums of segments of 1024 tokens, the choice. The logits are read three times where there is a cut, the second and third
// time from a cache. 256 rows of 151936, fp32, by top-p: 33 us for the largest (4.7 TB/s), 46 for the histogram (30 instructions a logit, most
// of them for its weight: 76 % of the units' time), 37 for the list, 13 for the choice. One row: 3.2 + 4.7 + 5.3 + 7.6 us; a row whose
// cut goes over it again in the last launch 170 to 210.
#include "qvl_decoder.h"
#include "qvl_kernels.h"

namespace qvl {

constexpr int kBins = 1536, kSegment = 1024, kMaxSegments = 256, kList = 4096, kShare = 1024;   // kShare: a workgroup's of the list
constexpr int kSort = 1024, kFew = 128;       // tokens that are sorted, and that are sorted without a look at parts of their bin
constexpr int kSome = 512;                   // of a segment's 1024 tokens: up to which the list's pass packs those that it weighs
constexpr int kRowsAtOnce = 1024;            // rows that share a workspace
constexpr double kUnit = 17592186044416.0;   // 2^44

// What the launches leave each other of a row.
struct SampleRow {
  uint64_t tops[kMaxSegments];               // the first place in the order of each segment
  uint64_t sums[kMaxSegments];               // sums of the segments' kept weights (list apart)
  uint64_t hist[kBins];
  uint64_t list[kList];                      // places of the cut's tokens
  uint64_t before, whole;                    // sums of weights before the list, and of all
  uint32_t n;                                // entries of the list (more than kList: not listed)
  int32_t bin;                               // the cut's
};

struct SampleParams {
  const char* x;
  int64_t row;                               // bytes
  int vocab, segments;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;        // where the pointers are NULL
  int32_t top_k1;
  int64_t* out;
  SampleRow* rows;
  int first;                                 // row 0 of this launch
};

struct Settings {
  double t, p, u;
  uint64_t floor;                            // the least weight that min-p keeps
  int k;                                     // 0: no top-k
  bool greedy, nucleus;
};

__device__ __forceinline__ Settings settings_of(const SampleParams& P, int64_t row) {
  Settings s;
  s.t = P.temperature ? P.temperature[row] : P.temperature1;
  s.p = P.top_p ? P.top_p[row] : P.top_p1;
  const double min_p = P.min_p ? P.min_p[row] : P.min_p1;
  s.k = max(P.top_k ? P.top_k[row] : P.top_k1, 0);
  // (beyond 1: the largest double below it, whose product with any sum, rounded, stays below that sum: it is half to one unit of its last place less)
  const double u = P.u[row];
  s.u = u >= 0 ? min(u, 1 - 0x1p-53) : 0;
  s.nucleus = s.p < 1;
  s.floor = min_p > 0 ? (uint64_t)ceil(min(min_p, 2.0) * kUnit) : 0;
  // the first token in the order alone; elsewhere the rules keep it by themselves
  s.greedy = !(s.t > 0) || s.k == 1 || s.p <= 0 || min_p > 1;
  return s;
}

// Place in the order: smaller is earlier (a larger logit, then a smaller index); NaN and +infinity come before all numbers.
constexpr uint32_t kNumbers = 0x00800000u;   // the first key of a number
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return x != x ? 0u : b & 0x80000000u ? b : b ^ 0x7fffffffu;
}
__device__ __forceinline__ uint64_t place_of(float x, int index) { return (uint64_t)key_of(x) << 32 | (uint32_t)index; }
__device__ __forceinline__ float logit_of(uint64_t place) {
  const uint32_t key = (uint32_t)(place >> 32);
  return __uint_as_float(key & 0x80000000u ? key : key ^ 0x7fffffffu);
}

// 2^(44 - j / 32), of five roots of 1/2 (at most four roundings: 5e-16).
struct WeightTable {
  double at[32];
  constexpr WeightTable() : at() {
    constexpr double root[5] = {0.97857206208770013451, 0.95760328069857364694, 0.91700404320467123174, 0.84089641525371454303,
                                0.70710678118654752440};
    for (int j = 0; j < 32; ++j) {
      at[j] = kUnit;
      for (int i = 0; i < 5; ++i)
        if (j >> i & 1) at[j] *= root[i];
    }
  }
};
__device__ constexpr WeightTable kWeights{};
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 32) table[threadIdx.x] = kWeights.at[threadIdx.x];
}

// Bin and weight of a logit; false: beyond the bins, weight 0 (-infinity too).
struct Weigher {
  double top, scale;                         // 32 / (T ln 2)
  const double* table;                       // LDS: 2^(44 - j / 32)
  // The bin is y to the nearest whole number, which the sum with 3 2^51 leaves in its low bits: a conversion takes four times an
  // addition's time. Products and sums are joined by hand, so that every pass over the row comes to the same bins and weights: left to the
  // compiler, one pass rounded the product before the sum and the next did not, and a token on a bin's border was in two of them or in none.
  __device__ __forceinline__ bool bin_of(float x, int& bin, double& rest) const {
    const double d = top - (double)x, y = d * scale;
    const double whole = __builtin_fma(d, scale, 0x1.8p52);
    bin = (int)__double2loint(whole);
    rest = __builtin_fma(d, scale, -(whole - 0x1.8p52));
    return y < kBins - 1;
  }
  __device__ __forceinline__ uint64_t weight(int bin, double r) const {
    // 2^(-r / 32), |r| <= 1/2: the exponential's sum to the fifth power of c r, c = ln 2 / 32 (the sixth is 2e-15)
    constexpr double c = -0.69314718055994530942 / 32, c2 = c * c, c3 = c2 * c;
    double e = __builtin_fma(r, c3 * c2 / 120, c2 * c2 / 24);
    e = __builtin_fma(e, r, c3 / 6);
    e = __builtin_fma(e, r, c2 / 2);
    e = __builtin_fma(e, r, c);
    e = __builtin_fma(e, r, 1.0);
    e *= table[bin & 31];
    e = __hiloint2double(__double2hiint(e) - ((bin & ~31) << 15), __double2loint(e));   // 2^(bin / 32) less: 2^-4 at least
    // (plus 2^52: rounded to a whole number, which the low bits then hold)
    return (uint64_t)__double_as_longlong(e + 0x1p52) & 0xfffffffffffffull;
  }
  // A number that no logit of bins up to `bin` lies below: the border, less what its own sums and its rounding to fp32 may be off by.
  __device__ __forceinline__ float least(int bin) const {
    const double down = (bin + 0.5) / scale;
    return (float)(top - down - (fabs(top) + down) * 0x1p-22);
  }
  __device__ __forceinline__ bool operator()(float x, int& bin, uint64_t& w) const {
    double r;
    if (!bin_of(x, bin, r)) return false;
    w = weight(bin, r);
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

// v of the lane that DPP control CTRL names, 0 where there is none (or where MASK leaves the row out).
template <int CTRL, int MASK = 0xf> __device__ __forceinline__ uint64_t dpp_or_zero(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, MASK, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, MASK, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}
// Inclusive sums over the wave: within rows of 16 lanes, then each row's last lane to the next row, then the first half's to the second.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += dpp_or_zero<0x111>(v);
  v += dpp_or_zero<0x112>(v);
  v += dpp_or_zero<0x114>(v);
  v += dpp_or_zero<0x118>(v);
  v += dpp_or_zero<0x142, 0xa>(v);
  v += dpp_or_zero<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
// The smallest over the wave, in its last lane: ~v's largest, so that lanes that are none count as 0.
__device__ __forceinline__ uint64_t wave_min(uint64_t v) {
  v = ~v;
  v = max(v, dpp_or_zero<0x111>(v));
  v = max(v, dpp_or_zero<0x112>(v));
  v = max(v, dpp_or_zero<0x114>(v));
  v = max(v, dpp_or_zero<0x118>(v));
  v = max(v, dpp_or_zero<0x142, 0xa>(v));
  v = max(v, dpp_or_zero<0x143, 0xc>(v));
  return last_lane(~v);
}

// Inclusive sums over the workgroup of NT threads; `waves`: NT / 64 words of LDS. Ends with a barrier that frees them. (Short code here
// and in the choice: what runs once is paid by its length, as a workgroup waits for each line of it.)
template <int NT> __device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* waves, uint64_t& total) {
  const int wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if ((threadIdx.x & 63) == 63) waves[wave] = v;
  __syncthreads();
  uint64_t w[NT / 64], before = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) w[i] = waves[i];
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    before = i == wave ? total : before;
    total += w[i];
  }
  __syncthreads();
  return v + before;
}

// The elements of segments [s0, s1), every NT / 64th to a wave, a segment's loads ahead of the work on the one before; the first ones are
// under way once the walk is made.
template <typename T, int NT> struct Walk {
  const char* row;
  int vocab, s, s1;
  Segment<T> g;
  __device__ __forceinline__ Walk(const char* row, int vocab, int s0, int s1) : row(row), vocab(vocab), s(s0 + (int)(threadIdx.x >> 6)), s1(s1) {
    if (s < s1) g.load(row, vocab, s);
  }
  // f(values, segment) for each segment of the wave
  template <typename F> __device__ __forceinline__ void segments(F&& f) {
    for (; s < s1; s += NT / 64) {
      Segment<T> next;
      if (s + NT / 64 < s1) next.load(row, vocab, s + NT / 64);
      f(g.x, s);
      g = next;
    }
  }
  // f(x, index) for each, after(segment) behind each
  template <typename F, typename G> __device__ __forceinline__ void run(F&& f, G&& after) {
    segments([&](const float (&x)[16], int s) {
#pragma unroll
      for (int i = 0; i < 16; ++i) f(x[i], s * kSegment + Segment<T>::index(i));
      after(s);
    });
  }
};

// The smallest place of a row; over the workgroup of NT threads.
template <int NT> __device__ __forceinline__ uint64_t first_place(const SampleRow& r, int segments, uint64_t* waves) {
  uint64_t m = ~0ull;
  for (int i = threadIdx.x; i < segments; i += NT) m = min(m, r.tops[i]);
  m = wave_min(m);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) m = min(m, waves[i]);
  __syncthreads();
  return m;
}
// whether a row has no token: NaN, +infinity, or nothing but -infinity
__device__ __forceinline__ bool no_token(uint64_t first) { return (uint32_t)(first >> 32) < kNumbers || logit_of(first) == -INFINITY; }

__device__ __forceinline__ Weigher weigher_of(uint64_t first, const Settings& st, const double* table) {
  return Weigher{logit_of(first), 32 / 0.69314718055994530942 / st.t, table};
}

// -------------------------------------------------------------------------------------------------------------------
// the launches over shares of rows: workgroup x takes segments [x per, (x + 1) per)
// -------------------------------------------------------------------------------------------------------------------
// The first place of each segment, and the row's sums cleared.
template <typename T>
__global__ __launch_bounds__(256) void sample_tops_kernel(SampleParams P, int per) {
  SampleRow& r = P.rows[blockIdx.y];
  const char* row = P.x + (P.first + (int64_t)blockIdx.y) * P.row;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < kBins; i += gridDim.x * 256) r.hist[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) r.n = 0;
  const int s0 = blockIdx.x * per, s1 = min(s0 + per, P.segments);
  Walk<T, 256>(row, P.vocab, s0, s1).segments([&](const float (&x)[16], int s) {
    float most = -INFINITY;                  // (a lane of nothing more: whichever of its tokens, none can be chosen)
    int at = 0;
    bool wrong = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      wrong = wrong || x[i] != x[i];
      at = x[i] > most ? i : at;
      most = x[i] > most ? x[i] : most;
    }
    const uint64_t m = wave_min(place_of(wrong ? NAN : most, s * kSegment + Segment<T>::index(at)));
    if ((threadIdx.x & 63) == 0) r.tops[s] = m;
  });
}

// The row's histogram: counts where top-k cuts, else weights where top-p does.
template <typename T>
__global__ __launch_bounds__(256) void sample_histogram_kernel(SampleParams P, int per) {
  __shared__ uint64_t hist[kBins], waves[4];
  __shared__ double table[32];
  SampleRow& r = P.rows[blockIdx.y];
  const int64_t at = P.first + (int64_t)blockIdx.y;
  const Settings st = settings_of(P, at);
  if (st.greedy || (st.k == 0 && !st.nucleus)) return;
  const int s0 = blockIdx.x * per, s1 = min(s0 + per, P.segments);
  Walk<T, 256> walk(P.x + at * P.row, P.vocab, s0, s1);
  fill_table(table);
  for (int i = threadIdx.x; i < kBins; i += 256) hist[i] = 0;
  const uint64_t first = first_place<256>(r, P.segments, waves);
  if (no_token(first)) return;
  const Weigher weigh = weigher_of(first, st, table);
  walk.run([&](float x, int) {
    int bin;
    if (st.k > 0) {
      double rest;
      if (weigh.bin_of(x, bin, rest)) atomicAdd((uint32_t*)&hist[bin], 1u);
    } else {
      uint64_t w;
      if (weigh(x, bin, w)) atomicAdd((unsigned long long*)&hist[bin], (unsigned long long)w);
    }
  }, [](int) {});
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (hist[i]) atomicAdd((unsigned long long*)&r.hist[i], (unsigned long long)hist[i]);
}

// The bin that holds the cut: the first whose sum with those before reaches `enough(sum, whole)` (the last, if none does); the sum before it
// and the whole.
struct Cut {
  int bin;
  uint64_t before, whole;
};
template <typename F> __device__ __forceinline__ Cut cut_bin(const uint64_t (&h)[kBins / 256], uint64_t* waves, Cut* found, F&& enough) {
  constexpr int kPer = kBins / 256;
  uint64_t own = 0, whole;
#pragma unroll
  for (int j = 0; j < kPer; ++j) own += h[j];
  uint64_t upto = block_scan<256>(own, waves, whole) - own;
  bool was = upto > 0 && enough(upto, whole);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int bin = threadIdx.x * kPer + j;
    const bool is = enough(upto + h[j], whole);
    if (bin == 0 ? is : is && !was) *found = Cut{bin, upto, whole};
    else if (bin == kBins - 1 && !is) *found = Cut{bin, upto, whole};
    was = is;
    upto += h[j];
  }
  __syncthreads();
  return *found;
}

// The tokens of the cut's bin (of top-k: all up to it) into the list, and the sums of the segments' weights before it (without a cut: of all).
template <typename T>
__global__ __launch_bounds__(256) void sample_list_kernel(SampleParams P, int per) {
  __shared__ uint64_t waves[4], list[kShare];
  __shared__ f32x2 kept[4][kSome];
  __shared__ double table[32];
  __shared__ Cut found;
  __shared__ uint32_t n, base;
  SampleRow& r = P.rows[blockIdx.y];
  const int64_t at = P.first + (int64_t)blockIdx.y;
  const Settings st = settings_of(P, at);
  if (st.greedy) return;
  const int s0 = blockIdx.x * per, s1 = min(s0 + per, P.segments);
  Walk<T, 256> walk(P.x + at * P.row, P.vocab, s0, s1);
  uint64_t h[kBins / 256];                   // the histogram, 6 bins a thread
#pragma unroll
  for (int j = 0; j < kBins / 256; ++j) h[j] = r.hist[threadIdx.x * (kBins / 256) + j];
  fill_table(table);
  if (threadIdx.x == 0) n = 0;
  const uint64_t first = first_place<256>(r, P.segments, waves);
  if (no_token(first)) return;
  const Weigher weigh = weigher_of(first, st, table);
  Cut cut{kBins, 0, 0};
  if (st.k > 0) cut = cut_bin(h, waves, &found, [&](uint64_t c, uint64_t) { return c >= (uint64_t)st.k; });
  else if (st.nucleus) cut = cut_bin(h, waves, &found, [&](uint64_t w, uint64_t whole) { return !((double)w < st.p * (double)whole); });
  uint64_t sum = 0;
  const auto take = [&](float x, int index) {
    int bin;
    double rest;
    if (!weigh.bin_of(x, bin, rest) || bin > cut.bin) return;
    if (st.k > 0 || bin == cut.bin) {
      // (a share may hold them all: the rest goes straight to the row's list)
      const uint32_t i = atomicAdd(&n, 1u);
      if (i < kShare) list[i] = place_of(x, index);
      else {
        const uint32_t j = atomicAdd(&r.n, 1u);
        if (j < kList) r.list[j] = place_of(x, index);
      }
    } else {
      const uint64_t w = weigh.weight(bin, rest);
      sum += w < st.floor ? 0 : w;
    }
  };
  // Most cuts leave few of a segment: those are put side by side first, and their weights formed 64 at a time (256 rows by top-p: 37 us,
  // not 54; where more than half are left, or there is no cut, all in their places)
  const float least = weigh.least(min(cut.bin, kBins - 1));
  f32x2* const some = kept[threadIdx.x >> 6];
  walk.segments([&](const float (&x)[16], int s) {
    int left = cut.bin < kBins ? 0 : kSome + 1;
    if (left == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) left += __popcll(__builtin_amdgcn_ballot_w64(x[i] >= least));
    if (left <= kSome) {
      int upto = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(x[i] >= least);
        const int to = upto + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
        if (x[i] >= least) some[to] = f32x2{x[i], __uint_as_float((uint32_t)(s * kSegment + Segment<T>::index(i)))};
        upto += __popcll(lanes);
      }
      __builtin_amdgcn_wave_barrier();         // the wave's own LDS: written and read in its program order
      for (int j = threadIdx.x & 63; j < left; j += 64) take(some[j].x, (int)__float_as_uint(some[j].y));
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) take(x[i], s * kSegment + Segment<T>::index(i));
    }
    if (st.k == 0) {
      const uint64_t all = wave_scan(sum);
      if ((threadIdx.x & 63) == 63) r.sums[s] = all;
      sum = 0;
    }
  });
  __syncthreads();
  const uint32_t own = min(n, (uint32_t)kShare);
  if (threadIdx.x == 0) {
    base = own > 0 ? atomicAdd(&r.n, own) : 0;
    if (blockIdx.x == 0) {
      r.before = cut.before;
      r.whole = cut.whole;
      r.bin = cut.bin;
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < own; i += 256)
    if (base + i < kList) r.list[base + i] = list[i];
}

// -------------------------------------------------------------------------------------------------------------------
// the choice: a workgroup a row
// -------------------------------------------------------------------------------------------------------------------
constexpr int kChoosers = 512;               // threads of the choice
struct SampleLds {
  double table[32];
  uint64_t hist[kBins];
  uint64_t list[kList];
  uint64_t sort[kSort];
  uint64_t sums[kMaxSegments];
  uint64_t waves[kChoosers / 64];
  uint64_t found[2];
  int n, token;
};

// Sorted, rising: value j of thread i is number 512 j + i of `size`, a power of two. Neighbours up to a wave apart meet in registers.
template <int E> __device__ __forceinline__ void sort_values(uint64_t (&v)[E], int size, uint64_t* lds) {
  constexpr int NT = kChoosers;
  const int i = threadIdx.x;
#pragma unroll 1
  for (int k = 2; k <= size; k <<= 1) {
#pragma unroll 1
    for (int d = k >> 1; d > 0; d >>= 1) {
      if (E > 1 && d == NT) {
        const uint64_t a = min(v[0], v[E - 1]), b = max(v[0], v[E - 1]);   // (the last merge: rising)
        v[0] = a;
        v[E - 1] = b;
        continue;
      }
      if (d >= 64) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j) lds[j * NT + i] = v[j];
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint64_t o = d >= 64 ? lds[j * NT + (i ^ d)] : __shfl_xor((unsigned long long)v[j], d);
        const bool low = ((i & d) == 0) == (((j * NT + i) & k) == 0);
        v[j] = low ? min(v[j], o) : max(v[j], o);
      }
    }
  }
}

// The first of hist[0..n) (n a multiple of the threads) whose sum with `base` and those before it `enough` says is reached, the last that holds
// anything where none is; its sum before.
template <typename F> __device__ __forceinline__ int cut_of(SampleLds& lds, int n, uint64_t& base, F&& enough) {
  const int per = n / kChoosers, at = threadIdx.x * per;
  uint64_t own = 0, whole;
  for (int j = 0; j < per; ++j) own += lds.hist[at + j];
  uint64_t upto = base + block_scan<kChoosers>(own, lds.waves, whole) - own;
  whole += base;
  const bool none = !enough(whole);
  for (int j = 0; j < per; ++j) {
    const uint64_t h = lds.hist[at + j];
    if (h > 0 && (none ? upto + h == whole : enough(upto + h) && !enough(upto))) {
      lds.n = at + j;
      lds.found[0] = upto;
    }
    upto += h;
  }
  __syncthreads();
  base = lds.found[0];
  const int bin = lds.n;
  __syncthreads();
  return bin;
}

// The cut's place among the tokens of one bin that `each(f)` runs f(x, place, bin, rest) over: the first whose count (COUNT) or weight with all
// before it, `base` of them in earlier bins, is enough (the last, where none is). Where kSort share the bin, and then a 512th of it,
// false: they are equal, or nearly.
template <bool COUNT, typename Each, typename F>
__device__ __forceinline__ bool cut_place(const Weigher& weigh, SampleLds& lds, bool many, int in, uint64_t base, uint64_t most, uint64_t& last, Each&& each, F&& enough) {
  constexpr int NT = kChoosers;
  const int i = threadIdx.x;
  const auto gather = [&](int sub) {
    __syncthreads();
    if (i == 0) lds.n = 0;
    __syncthreads();
    each([&](uint64_t place, int bin, double rest) {
      if (bin != in || place > most || (sub >= 0 && min(max((int)((rest + 0.5) * NT), 0), NT - 1) != sub)) return;
      const int j = atomicAdd(&lds.n, 1);
      if (j < kSort) lds.sort[j] = place;
    });
    __syncthreads();
    return lds.n;
  };
  int n = many ? kFew + 1 : gather(-1);
  if (n > kFew) {
    __syncthreads();
    lds.hist[i] = 0;
    __syncthreads();
    each([&](uint64_t place, int bin, double rest) {
      if (bin != in || place > most) return;
      const int sub = min(max((int)((rest + 0.5) * NT), 0), NT - 1);
      atomicAdd((unsigned long long*)&lds.hist[sub], (unsigned long long)(COUNT ? 1 : weigh.weight(bin, rest)));
    });
    __syncthreads();
    n = gather(cut_of(lds, NT, base, enough));
    if (n > kSort) return false;
  }
  int size = 64;
  while (size < n) size <<= 1;
  uint64_t v[2], upto[2], w[2], whole, rest;
#pragma unroll
  for (int j = 0; j < 2; ++j) v[j] = j * NT + i < n ? lds.sort[j * NT + i] : ~0ull;
  __syncthreads();
  if (size <= NT) {
    uint64_t one[1] = {v[0]};
    sort_values<1>(one, size, lds.sort);
    v[0] = one[0];
  } else {
    sort_values<2>(v, size, lds.sort);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int bin;
    w[j] = 0;
    if (j * NT + i < n && (COUNT || weigh(logit_of(v[j]), bin, w[j])) && COUNT) w[j] = 1;
  }
  upto[0] = base + block_scan<NT>(w[0], lds.waves, whole);
  upto[1] = base + whole + block_scan<NT>(w[1], lds.waves, rest);
  if (i == 0) lds.found[1] = ~0ull;
  __syncthreads();
  uint64_t mine = ~0ull;
#pragma unroll
  for (int j = 1; j >= 0; --j)
    if (j * NT + i < n && (enough(upto[j]) || j * NT + i == n - 1)) mine = v[j];
  if (mine != ~0ull) atomicMin((unsigned long long*)&lds.found[1], (unsigned long long)mine);
  __syncthreads();
  last = lds.found[1];
  return true;
}

// A thread's additions to sums in LDS: what follows in the same one is added up first, as equal logits do for four levels below (a row of
// 151936 of them: 760 us a call, not 1110). Where sums change all the time, as in the other passes, it costs more than it saves.
struct Sums {
  uint64_t* to;
  int entry = 0;
  uint64_t sum = 0;
  __device__ __forceinline__ void put() {
    if (sum > 0) atomicAdd((unsigned long long*)&to[entry], (unsigned long long)sum);
  }
  __device__ __forceinline__ void add(int e, uint64_t w) {
    if (e != entry) {
      put();
      entry = e;
      sum = 0;
    }
    sum += w;
  }
};

// The same whatever the bin holds, 8 bits of the place at a time.
template <bool COUNT, typename Each, typename F>
__device__ __forceinline__ uint64_t cut_bits(const Weigher& weigh, SampleLds& lds, int in, uint64_t base, uint64_t most, Each&& each, F&& enough) {
  uint64_t prefix = 0;
  for (int level = 0; level < 7; ++level) {   // the logit's 32 bits, then the index's 18
    const int shift = level < 4 ? 56 - 8 * level : 16 - 8 * (level - 4);
    const int above = level == 4 ? 32 : shift + 8;
    __syncthreads();
    lds.hist[threadIdx.x] = 0;
    __syncthreads();
    Sums sums{lds.hist};
    each([&](uint64_t place, int bin, double rest) {
      if (bin == in && place <= most && (level == 0 || (place >> above) == (prefix >> above)))
        sums.add((int)(place >> shift) & 255, COUNT ? 1 : weigh.weight(bin, rest));
    });
    sums.put();
    __syncthreads();
    prefix |= (uint64_t)cut_of(lds, kChoosers, base, enough) << shift;
  }
  return prefix;
}

template <typename T>
__global__ __launch_bounds__(kChoosers) void sample_choose_kernel(SampleParams P) {
  constexpr int NT = kChoosers;
  static_assert(NT >= kMaxSegments && kSort == 2 * NT && kBins % NT == 0 && NT >= 256, "entries a thread");
  __shared__ SampleLds lds;
  const int64_t at = P.first + (int64_t)blockIdx.x;
  const SampleRow& r = P.rows[blockIdx.x];
  const char* row = P.x + at * P.row;
  int64_t* out = P.out + at;
  const int i = threadIdx.x;
  const uint64_t sum = i < P.segments ? r.sums[i] : 0;
  const int n = (int)min(r.n, (uint32_t)kList + 1);
  const Settings st = settings_of(P, at);
  fill_table(lds.table);
  const uint64_t first = first_place<NT>(r, P.segments, lds.waves);
  if (no_token(first) || st.greedy) {
    if (i == 0) *out = no_token(first) ? -1 : (int64_t)(uint32_t)first;
    return;
  }
  const Weigher weigh = weigher_of(first, st, lds.table);
  uint64_t last = ~0ull;                     // the last place that is kept
  if (i < P.segments) lds.sums[i] = st.k > 0 ? 0 : sum;
  if (i == 0) lds.found[1] = 0;
  if ((st.k > 0 || st.nucleus) && n <= kFew) {
    // the list sorted: with top-k all that can be kept, else the bin of top-p's cut
    uint64_t v[1] = {i < n ? r.list[i] : ~0ull}, w = 0, part;
    sort_values<1>(v, n <= 64 ? 64 : kFew, lds.sort);
    int bin;
    double rest;
    if (i < n && (st.k == 0 || i < st.k) && weigh.bin_of(logit_of(v[0]), bin, rest)) w = weigh.weight(bin, rest);
    const uint64_t upto = block_scan<NT>(w, lds.waves, part);
    const double enough = st.p * (double)(st.k > 0 ? part : r.whole);
    __syncthreads();
    if (w > 0 && !(st.nucleus && !((double)((st.k > 0 ? 0 : r.before) + upto - w) < enough))) {
      atomicMax((unsigned long long*)&lds.found[1], (unsigned long long)v[0]);
      if (w >= st.floor) atomicAdd((unsigned long long*)&lds.sums[(uint32_t)v[0] / kSegment], (unsigned long long)w);
    }
    __syncthreads();
    last = lds.found[1];
  } else if (st.k > 0 || st.nucleus) {
    const bool listed = n <= kList;
    if (listed)
      for (int j = i; j < n; j += NT) lds.list[j] = r.list[j];
    // f(place, bin, rest) for the list's tokens, or where there were too many for it all of the row's
    const auto each = [&](auto&& f) {
      if (listed) {
        for (int j = i; j < n; j += NT) {
          int bin;
          double rest;
          weigh.bin_of(logit_of(lds.list[j]), bin, rest);
          f(lds.list[j], bin, rest);
        }
      } else {
        Walk<T, NT>(row, P.vocab, 0, P.segments).run([&](float x, int index) {
          int bin;
          double rest;
          if (weigh.bin_of(x, bin, rest)) f(place_of(x, index), bin, rest);
        }, [](int) {});
      }
    };
    __syncthreads();
    uint64_t before = r.before, whole = r.whole;
    int bin = r.bin;
    if (st.k > 0) {
      const auto enough = [&](uint64_t c) { return c >= (uint64_t)st.k; };
      if (!cut_place<true>(weigh, lds, false, bin, before, last, last, each, enough)) last = cut_bits<true>(weigh, lds, bin, before, last, each, enough);
    }
    if (st.nucleus) {
      if (st.k > 0) {                        // the weights of what top-k kept, by bins
        const uint64_t most = last;
        __syncthreads();
        for (int j = i; j < kBins; j += NT) lds.hist[j] = 0;
        __syncthreads();
        uint64_t mine = 0;
        each([&](uint64_t place, int b, double rest) {
          if (place > most) return;
          const uint64_t w = weigh.weight(b, rest);
          mine += w;
          atomicAdd((unsigned long long*)&lds.hist[b], (unsigned long long)w);
        });
        __syncthreads();
        block_scan<NT>(mine, lds.waves, whole);
        before = 0;
      }
      const auto enough = [&](uint64_t w) { return !((double)w < st.p * (double)whole); };
      if (st.k > 0) bin = cut_of(lds, kBins, before, enough);
      const uint64_t most = last;
      if (!cut_place<false>(weigh, lds, st.k == 0, bin, before, most, last, each, enough)) last = cut_bits<false>(weigh, lds, bin, before, most, each, enough);
    }
    __syncthreads();
    each([&](uint64_t place, int b, double rest) {   // without top-k the segments' sums have the bins before the cut's
      if (place > last || (st.k == 0 && b != bin)) return;
      const uint64_t w = weigh.weight(b, rest);
      if (w >= st.floor) atomicAdd((unsigned long long*)&lds.sums[(uint32_t)place / kSegment], (unsigned long long)w);
    });
  }
  __syncthreads();
  // the segment whose kept weights reach u times all, and the token in it
  if (i == 0) {
    lds.n = 0;
    lds.found[0] = 0;
  }
  uint64_t total;
  const uint64_t own = i < P.segments ? lds.sums[i] : 0, upto = block_scan<NT>(own, lds.waves, total);
  const double t = st.u * (double)total;
  if ((double)upto > t && !((double)(upto - own) > t)) {
    lds.n = i;
    lds.found[0] = upto - own;
  }
  if (i == 0) lds.token = 0x7fffffff;
  __syncthreads();
  const int index = lds.n * kSegment + 2 * i;
  uint64_t w[2], whole;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float x = index + j < P.vocab ? (float)reinterpret_cast<const T*>(row)[index + j] : -INFINITY;
    int bin;
    double rest;
    const bool is = weigh.bin_of(x, bin, rest) && place_of(x, index + j) <= last;
    w[j] = is ? weigh.weight(bin, rest) : 0;
    if (w[j] < st.floor) w[j] = 0;
  }
  const uint64_t second = lds.found[0] + block_scan<NT>(w[0] + w[1], lds.waves, whole);
  if (w[0] > 0 && (double)(second - w[1]) > t) atomicMin(&lds.token, index);
  else if (w[1] > 0 && (double)second > t) atomicMin(&lds.token, index + 1);
  __syncthreads();
  // (were no weight kept, the first place: whoever looks the token up finds one)
  if (i == 0) *out = lds.token != 0x7fffffff ? lds.token : (int64_t)(uint32_t)first;
}

}  // namespace qvl

using namespace qvl;

extern "C" {

int qvl_sample_workspace_size(int64_t n_rows, size_t* bytes) {
  if (!bytes) return set_error(QVL_ERR_INVALID_ARG, "sample_workspace_size: bytes is NULL");
  if (n_rows < 0) return set_error(QVL_ERR_INVALID_ARG, "sample_workspace_size: bad sizes");
  *bytes = (size_t)std::min<int64_t>(n_rows, kRowsAtOnce) * sizeof(SampleRow);
  return QVL_OK;
}

int qvl_sample_tokens(void* stream, int32_t dtype, const void* logits, int64_t row_stride, int64_t n_rows, int64_t vocab, const float* u,
                      const float* d_temperature, float temperature, const int32_t* d_top_k, int32_t top_k, const float* d_top_p,
                      float top_p, const float* d_min_p, float min_p, int64_t* out, void* workspace, size_t workspace_bytes) {
  const char* what = "sample_tokens";
  if (dtype != QVL_DTYPE_F32 && dtype != QVL_DTYPE_BF16) return set_error(QVL_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (n_rows < 0 || vocab <= 0 || row_stride < 0) return set_error(QVL_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (vocab > kMaxSegments * kSegment) return set_error(QVL_ERR_UNSUPPORTED, "%s: %lld tokens (at most %d)", what, (long long)vocab, kMaxSegments * kSegment);
  if (n_rows > 0x7fffffffLL || row_stride > (int64_t)1 << 40) return set_error(QVL_ERR_UNSUPPORTED, "%s: sizes", what);
  if (n_rows == 0) return QVL_OK;
  if (!logits || !u || !out) return set_error(QVL_ERR_INVALID_ARG, "%s: NULL pointer", what);
  const int64_t size = dtype == QVL_DTYPE_BF16 ? 2 : 4;
  if ((uintptr_t)logits % size || (uintptr_t)out % 8 || (uintptr_t)u % 4 || (uintptr_t)d_temperature % 4 || (uintptr_t)d_top_k % 4 ||
      (uintptr_t)d_top_p % 4 || (uintptr_t)d_min_p % 4 || (uintptr_t)workspace % 16) return set_error(QVL_ERR_MISALIGNED, "%s: a pointer", what);
  size_t need = 0;
  QVL_TRY_RC(qvl_sample_workspace_size(n_rows, &need));
  if (workspace_bytes < need || !workspace) return set_error(QVL_ERR_WORKSPACE, "%s: workspace %zu < %zu", what, workspace_bytes, need);
  SampleParams P{(const char*)logits, row_stride * size, (int)vocab, (int)((vocab + kSegment - 1) / kSegment), u, d_temperature,
                 d_top_p, d_min_p, d_top_k, temperature, top_p, min_p, top_k, out, (SampleRow*)workspace, 0};
  // settings that are the same for all rows may leave launches nothing to do
  const bool cuts = d_top_k || top_k > 0 || d_top_p || top_p < 1;
  const bool greedy = (!d_temperature && !(temperature > 0)) || (!d_top_k && top_k == 1) || (!d_top_p && top_p <= 0) || (!d_min_p && min_p > 1);
  hipStream_t st = (hipStream_t)stream;
  for (int64_t first = 0; first < n_rows; first += kRowsAtOnce) {
    const int64_t rows = std::min<int64_t>(n_rows - first, kRowsAtOnce);
    P.first = (int)first;
    // a segment a wave, or as many as make some 2048 workgroups of four waves: all that the GPU holds (256 rows: the three
    // launches take 117 to 119 us, 117 with 1024 and 136 with 512)
    const int shares = (int)std::max<int64_t>(std::min<int64_t>((P.segments + 3) / 4, 2048 / rows), 1);
    const int per = (P.segments + shares - 1) / shares;
    const dim3 grid((unsigned)((P.segments + per - 1) / per), (unsigned)rows);
#define QVL_SAMPLE(KERNEL, GRID, NT, ...)                                                                        \
  do {                                                                                                           \
    if (dtype == QVL_DTYPE_BF16) hipLaunchKernelGGL((KERNEL<bf16>), GRID, dim3(NT), 0, st, __VA_ARGS__);         \
    else hipLaunchKernelGGL((KERNEL<float>), GRID, dim3(NT), 0, st, __VA_ARGS__);                                \
  } while (0)
    QVL_SAMPLE(sample_tops_kernel, grid, 256, P, per);
    if (!greedy && cuts) QVL_SAMPLE(sample_histogram_kernel, grid, 256, P, per);
    if (!greedy) QVL_SAMPLE(sample_list_kernel, grid, 256, P, per);
    QVL_SAMPLE(sample_choose_kernel, dim3((unsigned)rows), kChoosers, P);
#undef QVL_SAMPLE
    QVL_TRY_RC(check_launch(what));
  }
  return QVL_OK;
}

}  // extern "C"
