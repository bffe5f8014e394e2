// Attention of a few new tokens of each sequence over its pages of the 4-bit cache (qvl_paged.h), the sequences' state read on the
// device: bound by reading the pages once, 136 bytes a key and head of 128, K and V together (bf16 rows: 512).
//
// The launch is qvl_decode.hip's stream: the key blocks of all sequences are one line that is cut into equal runs, a workgroup a run
// and key/value head, and a second launch joins jobs that cross runs. A wave takes a step of 64 keys and up to 4 rows (token, query head)
// at a time, or of 32 keys and up to 8 or 16. S^T = K Q^T by v_mfma_f32_16x16x32_bf16 puts a row in a lane (column lane % 16) with keys
// 4 (lane / 16) + i of each tile of 16; an instruction's 32 dims lie in one group, so a group's sum takes the key's
// scale in fp32. O^T = V^T P^T takes the weights as they lie, times V's scale of the key and group, rounded to bf16 (off by 2^-8 of
// each at most; the product has no other type for them).
// K and V come by DMA into a ring in LDS of each wave's own (Ring): the loop has no barrier. Codes become bf16 by one conversion for two of
// them; V's are nibbles of one token in a row, and four bit operations turn 16 of two tokens into pairs.
//
// 96 sequences of 1 to 7900 keys, 32/8 heads of 128, bf16: 85 us and 5.5 for the join, 4.9 TB/s of cache; 24 instead of 12 sequences of
// 32000 keys take 72 us more, 5.8 TB/s. One of 9001: 11.6 and 5.5 us, a chain of the state, a page's number, a tile, and the join.
// MFMA is busy 13 % of the time, VALU 43 %, and waves wait 57 % of theirs.
//
// fp32: q and the weights are split in three bf16 parts (24 bits); the codes are exact, so three products give the fp32 one.
#include "qvl_decoder.h"
#include "qvl_decoder_line.h"
#include "qvl_paged.h"

namespace qvl {

// x rounded to `PARTS` bf16 parts, the largest first (PARTS 3: exact).
template <int PARTS, int N> __device__ __forceinline__ void bf16_parts(const float (&x)[N], uint32_t (&out)[PARTS][N / 2]) {
  float rest[N];
#pragma unroll
  for (int j = 0; j < N; ++j) rest[j] = x[j];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const uint32_t w = pack_bf16x2(rest[2 * j], rest[2 * j + 1]);
      out[p][j] = w;
      if (p + 1 < PARTS) {
        rest[2 * j] -= bf16_lo(w);
        rest[2 * j + 1] -= bf16_hi(w);
      }
    }
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

// The lane `BY` lanes on in its row of 16 (round).
template <int BY> __device__ __forceinline__ float turned(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + BY, 0xf, 0xf, false));
}

// A step of a wave: kTiles tiles of 16 keys, ROWS rows. Where the rows are 8 or 4, the 16 columns of a product hold 2 or 4 copies of
// them, and copy c (columns ROWS c on) keeps the scores of tile c alone: the scores of 2 or 4 tiles lie in the registers of one, and the
// softmax and the scales take a half or a quarter of the instructions. In the second product each copy's weights meet its own tile (the
// others' are masked), so that the copies hold sums over different keys, which finish() adds.
template <typename T, int D, int ROWS> struct PagedCore {
  using B = PageBlock<D>;
  static constexpr int kRows = ROWS, kPack = 16 / ROWS, kTiles = kPack == 4 ? 4 : 2, kSets = kTiles / kPack;
  static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1, kG = B::kGroups, kDB = D / 16;
  static constexpr int kWords = D / 32;        // words of K, of V and of either's scales that a lane has of a tile
  bf16x8 q[D / 32][kParts];                    // step 2 g + s (D = 64: s): the dims of group g in piece 2 quad + s
  f32x4 o[kDB];                                // D = 128: dims 64 (db / 4) + 4 r + db % 4, r = 4 quad + i; D = 64: 4 r + db
  float l;

  static __device__ __forceinline__ int quad() { return (threadIdx.x & 63) >> 4; }
  static __device__ __forceinline__ int copy() { return (threadIdx.x & 15) / ROWS; }
  __device__ __forceinline__ void init(const char* qrow) {
    constexpr int E = D / 16;
    const T* x = reinterpret_cast<const T*>(qrow);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int d = (2 * quad() + s) * E;
      float lo[8], hi[8];                      // D = 64: both halves in the first
#pragma unroll
      for (int j = 0; j < E; ++j) {
        lo[j] = (float)x[d + j];
        (D == 128 ? hi[j] : lo[E + j]) = (float)x[D / 2 + d + j];
      }
      set(q[s], lo);
      if constexpr (D == 128) set(q[2 + s], hi);
    }
#pragma unroll
    for (auto& y : o) y = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
  }
  static __device__ __forceinline__ void set(bf16x8 (&to)[kParts], const float (&x)[8]) {
    uint32_t w[kParts][4];
    bf16_parts<kParts>(x, w);
#pragma unroll
    for (int p = 0; p < kParts; ++p) to[p] = __builtin_bit_cast(bf16x8, u32x4{w[p][0], w[p][1], w[p][2], w[p][3]});
  }
  __device__ __forceinline__ void rescale(float a) {
#pragma unroll
    for (auto& y : o) y *= a;
    l *= a;
  }
  // the copies' sums, in all of them
  __device__ __forceinline__ void finish() {
    if constexpr (kPack > 1) {
      const auto add = [](float& x) {
        x += turned<8>(x);
        if constexpr (kPack == 4) x += turned<4>(x);
      };
#pragma unroll
      for (auto& y : o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = y[i];
          add(x);
          y[i] = x;
        }
      add(l);
    }
  }
  __device__ __forceinline__ float row_sum() const {
    const float x = l + __shfl_xor(l, 16);
    return x + __shfl_xor(x, 32);
  }
  static __device__ __forceinline__ float row_max(float x) {
    if constexpr (kPack > 1) x = fmaxf(x, turned<8>(x));
    if constexpr (kPack == 4) x = fmaxf(x, turned<4>(x));
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
  }
  template <typename F> __device__ __forceinline__ void each4(F&& f) const {
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) f(64 * g + 16 * quad() + 4 * i, f32x4{o[4 * g][i], o[4 * g + 1][i], o[4 * g + 2][i], o[4 * g + 3][i]});
  }

  // A lane's words out of a place of the ring (below): codes of a tile's K, of its V, the scales of the quad's four tokens.
  using Words = uint32_t[kWords];
  static __device__ __forceinline__ void load(Words& w, const char* p) {
    if constexpr (kWords == 4) *reinterpret_cast<u32x4*>(w) = *reinterpret_cast<const u32x4*>(p);
    else *reinterpret_cast<u32x2*>(w) = *reinterpret_cast<const u32x2*>(p);
  }
  static __device__ __forceinline__ void load_k(Words& w, const char* place) {
    const int lane = threadIdx.x & 63;
    load(w, place + (D == 128 ? lane * 16 : (quad() >> 1) * 256 + (lane & 15) * 16 + (quad() & 1) * 8));
  }
  static __device__ __forceinline__ void load_v(Words& w, const char* place) { load(w, place + B::kCodes + (threadIdx.x & 63) * kWords * 4); }
  template <bool V> static __device__ __forceinline__ void load_scales(Words& w, const char* place) {
    load(w, place + 2 * B::kCodes + (V ? B::kScales : 0) + quad() * kWords * 4);
  }
  // of token i of the quad, group g
  static __device__ __forceinline__ float scale(const Words& w, int i, int g) {
    const int at = i * kG + g;
    return at & 1 ? bf16_hi(w[at >> 1]) : bf16_lo(w[at >> 1]);
  }

  // The scores of a step whose first place is `mem`: s[set][i] is key 16 (kPack set + copy) + 4 quad + i.
  __device__ __forceinline__ void scores(const char* mem, int place, f32x4 (&s)[kSets]) const {
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      f32x4 sum[kG];
#pragma unroll
      for (int c = 0; c < kPack; ++c) {
        Words k;
        load_k(k, mem + (set * kPack + c) * place);
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const bf16x8 x = numbers8(k[kG * st + g]);
#pragma unroll
            for (int p = kParts - 1; p >= 0; --p) acc = product(x, q[2 * g + st][p], acc);
          }
          if (c == 0) sum[g] = acc;
          else
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[g][i] = copy() == c ? acc[i] : sum[g][i];
        }
      }
      Words sc;
      load_scales<false>(sc, mem + (set * kPack + copy()) * place);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[set][i] = scale(sc, i, 0) * sum[0][i];
        if constexpr (kG == 2) s[set][i] = __builtin_fmaf(scale(sc, i, 1), sum[1][i], s[set][i]);
      }
    }
  }

  // bytes whose low nibble is a code of a and whose high one is b's of the same dim: the even dims, the odd ones
  static __device__ __forceinline__ uint32_t even_pairs(uint32_t a, uint32_t b) { return (a & 0x0f0f0f0fu) | (b << 4 & 0xf0f0f0f0u); }
  static __device__ __forceinline__ uint32_t odd_pairs(uint32_t a, uint32_t b) { return (a >> 4 & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u); }

  // o += V^T P^T of the step, weights w (V's scales come in here); `seen`: a bit for each key of the lane that the row sees, where EDGE.
  // `read` runs once the step's places are read.
  template <bool EDGE, typename F>
  __device__ __forceinline__ void values(const char* mem, int place, const f32x4 (&w)[kSets], uint32_t seen, F&& read) {
    Words sc[kSets], v[kTiles];
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      load_scales<true>(sc[set], mem + (set * kPack + copy()) * place);
      l += (w[set][0] + w[set][1]) + (w[set][2] + w[set][3]);
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) load_v(v[t], mem + t * place);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    read();
    uint32_t p[kSets][kG][kParts][2];          // weights times scales, bf16
#pragma unroll
    for (int set = 0; set < kSets; ++set)
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = w[set][i] * scale(sc[set], i, g);
          if (EDGE) x[i] = (seen >> (4 * set + i)) & 1 ? x[i] : 0.f;   // an unseen key's scale may be anything
        }
        bf16_parts<kParts>(x, p[set][g]);
      }
#pragma unroll
    for (int pair = 0; pair < kTiles / 2; ++pair) {
      uint32_t even[2][2], odd[2][2];          // [tile][tokens (0, 1), (2, 3)]
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // (D = 64: two tokens a word, the second's codes 16 bits on)
          const uint32_t x = D == 128 ? v[2 * pair + b][(2 * h) % kWords] : v[2 * pair + b][h];
          const uint32_t y = D == 128 ? v[2 * pair + b][(2 * h + 1) % kWords] : v[2 * pair + b][h] >> 16;
          even[b][h] = even_pairs(x, y);
          odd[b][h] = odd_pairs(x, y);
        }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        bf16x8 pw[kParts];
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
          u32x4 x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tile = 2 * pair + j / 2;
            x[j] = p[tile / kPack][g][n][j & 1] & (kPack == 1 || copy() == tile % kPack ? ~0u : 0u);
          }
          pw[n] = __builtin_bit_cast(bf16x8, x);
        }
        const auto add = [&](int db, uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
          const bf16x8 x = __builtin_bit_cast(bf16x8, u32x4{a0, a1, b0, b1});
#pragma unroll
          for (int n = kParts - 1; n >= 0; --n) o[db] = product(x, pw[n], o[db]);
        };
        if (g == 0) {                          // bytes 0 and 1: dims 4 r + (0, 1), (2, 3) of the first group
          add(0, numbers<0>(even[0][0]), numbers<0>(even[0][1]), numbers<0>(even[1][0]), numbers<0>(even[1][1]));
          add(1, numbers<0>(odd[0][0]), numbers<0>(odd[0][1]), numbers<0>(odd[1][0]), numbers<0>(odd[1][1]));
          add(2, numbers<1>(even[0][0]), numbers<1>(even[0][1]), numbers<1>(even[1][0]), numbers<1>(even[1][1]));
          add(3, numbers<1>(odd[0][0]), numbers<1>(odd[0][1]), numbers<1>(odd[1][0]), numbers<1>(odd[1][1]));
        } else {
          add(kDB - 4, numbers<2>(even[0][0]), numbers<2>(even[0][1]), numbers<2>(even[1][0]), numbers<2>(even[1][1]));
          add(kDB - 3, numbers<2>(odd[0][0]), numbers<2>(odd[0][1]), numbers<2>(odd[1][0]), numbers<2>(odd[1][1]));
          add(kDB - 2, numbers<3>(even[0][0]), numbers<3>(even[0][1]), numbers<3>(even[1][0]), numbers<3>(even[1][1]));
          add(kDB - 1, numbers<3>(odd[0][0]), numbers<3>(odd[0][1]), numbers<3>(odd[1][0]), numbers<3>(odd[1][1]));
        }
      }
    }
  }
};

// One wave: its rows over steps of keys.
template <typename T, int D, int ROWS> struct PagedWave : RowState<PagedCore<T, D, ROWS>> {
  using C = PagedCore<T, D, ROWS>;
  using RowState<C>::core;
  using RowState<C>::lim;
  using RowState<C>::lim_lo;

  // The step of key kb on, in places from mem on; bad: which of its tiles lie in a page outside the cache (their keys' scores are NaN).
  template <bool EDGE, typename F> __device__ __forceinline__ void step(const char* mem, int place, int kb, float scale, uint32_t bad, F&& read) {
    f32x4 s[C::kSets];
    uint32_t seen = 0;
    core.scores(mem, place, s);
    float mx = -INFINITY;
#pragma unroll
    for (int set = 0; set < C::kSets; ++set) {
      const int tile = set * C::kPack + C::copy();
      if (bad != 0 && (bad >> tile & 1)) s[set] = f32x4{NAN, NAN, NAN, NAN};
      if (EDGE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = kb + 16 * tile + 4 * C::quad() + i < lim;
          seen |= (in ? 1u : 0u) << (4 * set + i);
          s[set][i] = in ? s[set][i] : -INFINITY;
        }
      }
      mx = fmaxf(fmaxf(mx, s[set][0]), s[set][1]);
      mx = fmaxf(fmaxf(mx, s[set][2]), s[set][3]);
    }
    this->cover(C::row_max(mx) * scale);
    const float shift = this->shift();
    f32x4 w[C::kSets];
#pragma unroll
    for (int set = 0; set < C::kSets; ++set)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[set][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[set][i], scale, shift));
    core.template values<EDGE>(mem, place, w, seen, read);
  }
};

// Where a wave's tiles lie: of its next steps' 64 tiles, one a lane.
template <int D, int TILES> struct PageWalk {
  static constexpr int kSteps = 64 / TILES;
  const Pages& pages;
  int64_t seq;
  int kvh, last;                               // the last tile that holds a key
  const char* at;                              // the lane's tile; NULL: its page is none
  __device__ __forceinline__ void look(int t) {   // steps t, t + 4, ...
    const int lane = threadIdx.x & 63;
    const int b = (int)min((int64_t)TILES * (t + 4 * (lane / TILES)) + lane % TILES, (int64_t)last);
    const int page = pages.page(seq, b >> (pages.shift - 4));
    at = page < 0 ? nullptr : pages.block<D>(page, kvh, b << 4);
  }
  __device__ __forceinline__ const char* block(int i) const {
    const uint64_t p = (uint64_t)at;
    return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)p, i));
  }
};

// 4 bytes per lane, global -> LDS, as dma16.
__device__ __forceinline__ void dma4(u32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" :: "v"(voff), "s"(rsrc), "s"(lds) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

// A wave's own ring of steps in LDS, filled by DMA kDepth steps ahead, so that a step's loads take no registers (with a step's loads one
// step ahead in registers the loop's copies of them waited for them). Steps of 64 keys go one ahead: 70 KB of a CU are under way, and
// with twice that memory gives less (a plain read of 415 MB: 6.5 TB/s with 32 KB of a CU under way, 5.2 with 128; 12 sequences of 32000
// keys 87 us, not 92). A place is a block as it lies in memory, but for K, whose 16-byte pieces go where their lane reads them, 256
// bytes a quad: 64 lanes then meet in no bank.
template <int D, int TILES> struct Ring {
  using B = PageBlock<D>;
  static constexpr int kDepth = TILES == 4 ? 1 : 2, kPlace = 2 * B::kCodes + 256, kStep = TILES * kPlace, kWave = kDepth * kStep;
  static constexpr int kLoads = TILES * (D == 128 ? 3 : 2);    // a step's
  uint32_t lds;
  const char* mem;
  __device__ __forceinline__ explicit Ring(char* smem) {
    mem = smem + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kWave;
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr_of(mem));
  }
  // tile b of the step that takes place `at`
  __device__ __forceinline__ void fill(int at, int b, const char* block) const {
    const uint32_t lane = threadIdx.x & 63, to = lds + at * kStep + b * kPlace;
    // (no page: a range of nothing, which reads nothing)
    const u32x4 rsrc = rsrc_words(block, block ? B::kBytes : 0);
    if constexpr (D == 128) {
      dma16(rsrc, (lane & 15) * 64 + (lane >> 4) * 16, 0, to);
      dma16(rsrc, B::kCodes + lane * 16, 0, to + B::kCodes);
    } else {
      dma16(rsrc, lane < 32 ? (lane & 15) * 32 + (lane >> 4) * 16 : lane * 16, 0, to);
    }
    dma4(rsrc, 2 * B::kCodes + lane * 4, to + 2 * B::kCodes);   // the scales; the lanes behind them read nothing
  }
};

// A workgroup's four waves over steps [t0, t1), every fourth to a wave. The first steps are under way before the rows are read.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void paged_run(const AttnParams& P, const Pages& pages, int seq, const Unit& u, PagedWave<T, D, ROWS>& w, char* smem, int t0, int t1) {
  constexpr int kTiles = PagedCore<T, D, ROWS>::kTiles;
  using R = Ring<D, kTiles>;
  using Walk = PageWalk<D, kTiles>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int t = t0 + wave, n = 0;
  const bool any = t < t1;
  const R ring(smem);
  Walk walk{pages, seq, u.kvh, (u.len - 1) >> 4, nullptr};
  uint32_t bad = 0;                            // kTiles bits for each step under way
  const auto fetch = [&] {                     // step n of the wave (behind the last one, the last again)
    if (n % Walk::kSteps == 0) walk.look(t0 + wave + 4 * n);
    bad >>= kTiles;
#pragma unroll
    for (int b = 0; b < kTiles; ++b) {
      const char* block = walk.block(kTiles * (n % Walk::kSteps) + b);
      ring.fill(n % R::kDepth, b, block);
      if (!block) bad |= 1u << (kTiles * (R::kDepth - 1) + b);
    }
    ++n;
  };
  if (any) {
#pragma unroll
    for (int i = 0; i < R::kDepth; ++i) fetch();
  }
  w.init(P, u, u.row0);
  if (any) {
    for (int at = 0; t < t1; t += 4, at = at + 1 == R::kDepth ? 0 : at + 1) {
      wait_loads<R::kLoads * (R::kDepth - 1)>();
      const char* mem = ring.mem + at * R::kStep;
      const int kb = t * 16 * kTiles;
      const uint32_t now = bad & ((1u << kTiles) - 1);
      if (kb + 16 * kTiles > w.lim_lo) w.template step<true>(mem, R::kPlace, kb, P.scale, now, fetch);
      else w.template step<false>(mem, R::kPlace, kb, P.scale, now, fetch);
    }
    wait_loads<0>();                           // the join takes the ring's memory
  }
  w.core.finish();
}

template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256, 2) void paged_stream_kernel(AttnParams P, DecodeState S, Pages pages) {
  using W = PagedWave<T, D, ROWS>;
  constexpr int kLds = std::max({kJoinBytes<T, D, ROWS>, 4 * Ring<D, W::C::kTiles>::kWave, (int)sizeof(Line)});
  __shared__ __attribute__((aligned(16))) char smem[kLds];
  Line& L = *reinterpret_cast<Line*>(smem);    // (before the ring is)
  const int run = blockIdx.x / P.hkv, kvh = blockIdx.x % P.hkv;
  int64_t total, pos, end, base = 0;
  int n, seq = 0;
  Sequence q;
  find_run(P, S, L, run, gridDim.x / P.hkv, total, n, pos, end, seq, base, q);
  lds_barrier();
  SplitJob joined{};
  while (pos < end) {
    const int cost = q.blocks;                 // of a job: S.pad and its blocks
    const int64_t own = (int64_t)q.jobs * cost;
    if (pos >= base + own) {           // the next sequence (jobs == 0: it has no rows)
      base += own;
      q = uniform(sequence_of(P, S, ++seq));
      continue;
    }
    const int64_t into = pos - base;
    const int job = (int)(into / cost), c0 = (int)(into % cost), c1 = (int)min((int64_t)cost, c0 + (end - pos));
    const int b0 = max(c0 - S.pad, 0), b1 = c1 - S.pad;
    const Unit u{nullptr, nullptr, q.len, q.len - q.tokens + 1, q.token0, q.tokens * P.group, job * W::kRows, kvh};
    const int n_rows = min(W::kRows, u.rows - u.row0);
    const bool whole = c0 == 0 && c1 == cost;
    if (bad_keys(P, 0, u.len)) {
      for (int i = threadIdx.x; i < n_rows * (D / 4); i += 256)
        store4<T>(out_row<T, D>(P, u, u.row0 + i / (D / 4)), i % (D / 4) * 4, f32x4{NAN, NAN, NAN, NAN});
    } else {
      W w;
      paged_run<T, D, ROWS>(P, pages, seq, u, w, smem, b0, min(b1, (int)((u.len + (1ll << S.shift) - 1) >> S.shift)));
      const int64_t slot = ((int64_t)(2 * run + (c0 == 0)) * P.hkv + kvh) * S.slot_rows;
      join_waves<T, D>(P, u, w, smem, u.row0, b0 << S.shift, !whole, [&](int r) { return slot + r; });
    }
    if (c0 > 0 && c1 == cost) {
      // the run that holds the job's first block: the last whose share begins there, in its padding or before
      const int64_t first = pos - c0 + S.pad;
      int w0 = (int)min((int64_t)((float)first / (float)total * n), (int64_t)run);
      while (w0 > 0 && share(total, w0, n) > first) --w0;
      while (w0 < run && share(total, w0 + 1, n) <= first) ++w0;
      joined = SplitJob{u.token0, u.rows, u.row0, w0, run - w0 + 1};
    }
    pos += c1 - c0;
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
  int runs, slot_rows, tile, join_rows;   // join_rows: workgroups that share a job's rows in the join
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
  const int64_t own_rows = (rows + std::max<int64_t>(n_seqs, 1) - 1) / std::max<int64_t>(n_seqs, 1);   // a sequence's, in the mean
  D.tile = own_rows <= 4 ? 4 : own_rows <= 8 ? 8 : 16;
  const int64_t tiles = std::max<int64_t>((own_rows + D.tile - 1) / D.tile, 1), keys = D.tile == 4 ? 64 : 32;
  const int64_t jobs = n_seqs * tiles, blocks = jobs * ((max_len + keys - 1) / keys);
  D.runs = (int)std::max<int64_t>(std::min(slots / num_kv_heads, std::max((blocks + 3) / 4, jobs)), 1);
  D.slot_rows = (int)std::min<int64_t>(D.tile, std::max<int64_t>(rows, 1));
  // up to 8 parts a workgroup joins 8 rows at once; with more a row each, so that its parts come in one trip to memory
  D.join_rows = D.runs <= 8 * jobs ? (D.slot_rows + 7) / 8 : D.slot_rows;
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
  S.tile = plan.tile;
  S.shift = plan.tile == 4 ? 6 : 5;
  // what a job costs beside its keys (rows, first loads, join), and jobs that are not worth a part, in blocks: 96 sequences of up to 7900 keys
  // 93 us, not 122 without either. Found there alone, with bf16, heads of 128 and blocks of 64 keys; with blocks of 32, heads of 64 or fp32's
  // three products a block is another share of a job's cost, and the same counts stand unmeasured.
  S.pad = 12;
  S.keep = 24;
  const dim3 grid((unsigned)(plan.runs * num_kv_heads));
#define QVL_PAGED(T, D)                                                                                                              \
  do {                                                                                                                               \
    if (plan.tile == 4) hipLaunchKernelGGL((paged_stream_kernel<T, D, 4>), grid, dim3(256), 0, (hipStream_t)stream, P, S, pages);    \
    else if (plan.tile == 8) hipLaunchKernelGGL((paged_stream_kernel<T, D, 8>), grid, dim3(256), 0, (hipStream_t)stream, P, S, pages); \
    else hipLaunchKernelGGL((paged_stream_kernel<T, D, 16>), grid, dim3(256), 0, (hipStream_t)stream, P, S, pages);                  \
  } while (0)
  if (dtype == QVL_DTYPE_BF16) {
    if (head_dim == 128) QVL_PAGED(bf16, 128);
    else QVL_PAGED(bf16, 64);
  } else {
    if (head_dim == 128) QVL_PAGED(float, 128);
    else QVL_PAGED(float, 64);
  }
#undef QVL_PAGED
  QVL_TRY_RC(check_launch("paged_stream"));
  if (plan.runs == 1) return QVL_OK;
  QVL_ATTN_LAUNCH(paged_join_kernel, dim3((unsigned)plan.runs, (unsigned)num_kv_heads, (unsigned)plan.join_rows), P, S);
  return check_launch("paged_join");
}

}  // extern "C"
