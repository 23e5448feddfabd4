// Attention of drafted tokens over a paged key/value cache, for gfx950 (include/cugo_hip.h,
// cugo_tree_attention):
//
//   out[i, h, :] = sum_t softmax_t(q[i, h, :] . K[t] scale) V[t]
//
// over the positions t of the query's row that lie before its sequence's prefix or whose bit is
// set in its mask.  A sequence's queries and the heads that share a key head make the M = queries x
// group rows of one product with that head's keys, 16 MT of them (MT = 1, 2) a wavefront, so
// each key and value is read once for all of them.  A wavefront goes through tiles of 32 tokens (16
// in float32) with one running maximum and sum; nothing but the partial results of split rows leaves
// it.
//
// Scores are formed as S^T = K Q^T (16 x 16 matrix instructions, K the A operand), so that a lane
// has one query's scores (lane & 15) of tokens 4 g ... 4 g + 3 of each 16 (g = lane >> 4).  A lane's
// weights are the B operand of O^T += V^T P^T as they are, with those tokens in the product's inner
// places 8 g ... 8 g + 7, which V^T's A operand only has to follow: weights never move between lanes.
// That operand takes, for one element of the head, a lane's 8 tokens: a lane loads W consecutive
// elements of each (16 lanes cover a token's row) and turns the 8 x W block by v_perm_b32, so keys
// and values both come from memory into registers in whole rows.
//
// The running maximum moves only when a score exceeds it by more than 2^8 in the weight (kSlack):
// until then weights are at most 2^8, which neither type nor the sums mind, and a tile needs no
// exchange between lanes.  16-bit weights meet V as the sum of two numbers of the type, which costs
// nothing beside the memory (4,096 trees over 320 tokens: the same time) and leaves little but the
// output's rounding (2^-16 of a weight in bfloat16; 2^-22 in float16, or 2^-32 of the largest weight,
// half its smallest step, where that is more); where many rows make the products the bound
// (chunk_kernel), rounded once, half a step each, as much again as the output's rounding.  Their sum
// is taken from what meets V (a matrix instruction with ones), so they add up to one.
//
// Bound (us a call among others, joining included): memory where a key head has few rows (4,096 trees of
// 16 tokens over rows of up to 320, dh 32 bf16: 183 us, 4.7 TB/s; 24 trees over rows of up to 32,768,
// dh 128 float16: 377 us, 4.8 TB/s), the matrix and vector pipes in turn where it has many (4 x 512
// queries over 14,336 tokens, dh 128 bf16: 142 to 155 us, 690 to 751 TFLOP/s), latency in the smallest
// calls (one query: 9.3 us, its kernel 4.9).
//
// Tiles in which some query may not see some token (the drafts, a row's end) take their scores
// from the masks.  Values that are infinite or NaN go through products of their own (indicators of
// +inf and -inf), since 0 x inf would show in queries that do not attend them, and be NaN in those
// whose weight, or its second number, is 0: found among a tile's values (4,096 trees: the same time; where
// products are the bound, 2,048 queries of dh 32 131 -> 139 us, of float32 1,125 -> 1,154), or by
// chunk_kernel, whose full tiles do not pass through registers first, in its outputs.
#include <type_traits>

#include "tree_share.h"

namespace cugo_amd {
namespace paged {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// kLift: weights are 2^kLift times what they are against the running maximum (with kSlack at most 2^15,
// which float16 holds; its smallest step is then 2^-31 of the largest weight, not 2^-24).  Sums and
// outputs carry the factor alike.  The other types' steps are far below any that matters.
struct BF16 {
  static constexpr float kLift = 0.f;
  using storage = __bf16;
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7f80u;
  // x, or NaN where one of the word's numbers is infinite or NaN.
  __device__ __forceinline__ static float unless_odd(uint32_t w, float x) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, w), __builtin_bit_cast(pair, 0), x, false);
  }
  __device__ __forceinline__ static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a),
                                                   __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct F16 {
  static constexpr float kLift = 7.f;
  using storage = _Float16;
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7c00u;
  __device__ __forceinline__ static float unless_odd(uint32_t w, float x) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, w), __builtin_bit_cast(pair, 0), x, false);
  }
  __device__ __forceinline__ static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a),
                                                  __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct F32 {
  static constexpr float kLift = 0.f;
  using storage = float;
  __device__ __forceinline__ static float unless_odd(uint32_t w, float x) {
    return __builtin_fmaf(__uint_as_float(w), 0.f, x);
  }
};

constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.f;
constexpr int kWaves = 4;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// x times a weight, of which infinities and NaN are left where it is so small that it is 0.
__device__ __forceinline__ float scaled(float x, float weight) {
  return weight == 0.f && x - x != 0.f ? x : x * weight;
}

// The largest over the four lanes that hold one query (lane & 15).
__device__ __forceinline__ float query_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// W bytes / 4 words at p.
template <int N>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    static_assert(N == 4, "runs are of 4, 8 or 16 bytes");
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  }
}

// How a head's elements and a tile's tokens lie in a wavefront.
template <class T, int DH>
struct Shape {
  using S = typename T::storage;
  static constexpr int E = sizeof(S);
  static constexpr bool kWide = E == 4;
  static constexpr int KT = kWide ? 16 : 32;       // tokens a tile
  static constexpr int N = KT / 4;                 // of them a lane has scores and values
  static constexpr int KC = DH * E / 64;           // 16-byte parts of a key a lane holds
  static constexpr int KL = kWide ? 1 : 2;         // keys a lane holds parts of
  static constexpr int W = DH / 16 < 16 / E ? DH / 16 : 16 / E;  // a value's run of a lane
  static constexpr int H = DH / (16 * W);          // runs a value
  static constexpr int RW = W * E / 4;             // words a run
  static constexpr int NJ = DH / 16;               // 16 x 16 tiles of O^T
  // The place of a lane's token e in the tile, after 4 g.
  __device__ __forceinline__ static constexpr int place(int e) { return e + (e >= 4 ? 12 : 0); }
  // The element that row 4 g + i of tile j of O^T is.
  __device__ __forceinline__ static int element(int j, int row) { return j / W * 16 * W + W * row + j % W; }
};

// The parts of a tile's keys and values that a lane holds; at0 and at1: its first and second 16 tokens.
template <class T, int DH>
__device__ __forceinline__ void load_keys(const char* at0, const char* at1,
                                 u32x4 (&k)[Shape<T, DH>::KL][Shape<T, DH>::KC]) {
  using Sh = Shape<T, DH>;
  const unsigned lane = threadIdx.x & 63, mine = (lane & 15) * (DH * Sh::E) + (lane >> 4) * 16;
#pragma unroll
  for (int a = 0; a < Sh::KL; ++a)
#pragma unroll
    for (int p = 0; p < Sh::KC; ++p)
      k[a][p] = *reinterpret_cast<const u32x4*>((a ? at1 : at0) + mine + p * 64);
}
template <class T, int DH>
__device__ __forceinline__ void load_values(const char* at0, const char* at1,
                                   uint32_t (&v)[Shape<T, DH>::N][Shape<T, DH>::H][Shape<T, DH>::RW]) {
  using Sh = Shape<T, DH>;
  const unsigned lane = threadIdx.x & 63;
  const unsigned mine = (lane >> 4) * (4 * DH * Sh::E) + (lane & 15) * (Sh::W * Sh::E);
#pragma unroll
  for (int t = 0; t < Sh::N; ++t)
#pragma unroll
    for (int h = 0; h < Sh::H; ++h)
      load_words<Sh::RW>((t < 4 ? at0 : at1) + mine + (t & 3) * DH * Sh::E + h * 16 * Sh::W * Sh::E,
                         v[t][h]);
}

// What a wavefront holds of 16 MT queries, and its work on a tile of tokens.
template <class T, int DH, int MT>
struct Wave {
  using Sh = Shape<T, DH>;
  static constexpr int KT = Sh::KT, N = Sh::N, KC = Sh::KC, KL = Sh::KL, NJ = Sh::NJ;
  u32x4 q[MT][KC];
  f32x4 acc[MT][NJ];
  f32x4 sum[MT];
  float top[MT];

  struct Keys {
    u32x4 k[KL][KC];
  };
  // A product operand of N numbers, rounded to the type.
  struct Weights {
    uint32_t w[4];
  };
  // A tile's values in registers.
  struct Values {
    static constexpr bool kInPlace = true;
    uint32_t v[N][Sh::H][Sh::RW];
    // Elements j of the lane's N tokens.
    __device__ __forceinline__ Weights column(int, int j) const {
      Weights y;
      const int h = j / Sh::W, e = j % Sh::W;
      if constexpr (Sh::kWide) {
#pragma unroll
        for (int t = 0; t < 4; ++t) y.w[t] = v[t][h][e];
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          y.w[t] = __builtin_amdgcn_perm(v[2 * t + 1][h][e / 2], v[2 * t][h][e / 2],
                                         e & 1 ? 0x07060302u : 0x05040100u);
      }
      return y;
    }
    // Whether an infinity or NaN is among them.
    __device__ __forceinline__ bool odd() const {
      float x = 0.f;  // one instruction a word
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int h = 0; h < Sh::H; ++h)
#pragma unroll
          for (int e = 0; e < Sh::RW; ++e) x = T::unless_odd(v[t][h][e], x);
      return x != x;
    }
    // Zeros for the tokens from `until` on after the lane's first; whether an infinity or NaN is left.
    __device__ __forceinline__ bool clear(int until) {
      uint32_t odd = 0;
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int h = 0; h < Sh::H; ++h)
#pragma unroll
          for (int e = 0; e < Sh::RW; ++e) {
            v[t][h][e] = Sh::place(t) < until ? v[t][h][e] : 0u;
            odd |= odd_bits(v[t][h][e]);
          }
      return odd & kSigns;
    }
    __device__ __forceinline__ Weights cleared(int j) const { return column(0, j); }
    __device__ __forceinline__ void only_finite() {
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int h = 0; h < Sh::H; ++h)
#pragma unroll
          for (int e = 0; e < Sh::RW; ++e) v[t][h][e] = finite(v[t][h][e]);
    }
  };

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = kNegInf;
      sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // d[e]: the product of query lane & 15 with the lane's token e.
  __device__ __forceinline__ static void scores(const Keys& x, const u32x4 (&qm)[KC], float (&d)[N]) {
#pragma unroll
    for (int a = 0; a < KL; ++a) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < KC; ++p) {
        if constexpr (Sh::kWide) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[a][p][e]),
                                                     __uint_as_float(qm[p][e]), s, 0, 0, 0);
        } else {
          s = T::mfma(x.k[a][p], qm[p], s);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) d[4 * a + e] = s[e];
    }
  }

  __device__ __forceinline__ static Weights pack(const float (&p)[N]) {
    Weights x;
    if constexpr (Sh::kWide) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x.w[e] = __float_as_uint(p[e]);
    } else {
      typename T::vec y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (typename T::storage)p[e];
      const u32x4 z = __builtin_bit_cast(u32x4, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.w[e] = z[e];
    }
    return x;
  }
  // c += A P^T for the A operand `a` of N tokens.
  __device__ __forceinline__ static f32x4 product(const Weights& a, const Weights& p, f32x4 c) {
    if constexpr (Sh::kWide) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[e]), __uint_as_float(p.w[e]),
                                                 c, 0, 0, 0);
      return c;
    } else {
      return T::mfma(u32x4{a.w[0], a.w[1], a.w[2], a.w[3]}, u32x4{p.w[0], p.w[1], p.w[2], p.w[3]}, c);
    }
  }
  // What rounding to the type left of N numbers, rounded to it too.
  __device__ __forceinline__ static Weights rest(const float (&p)[N], const Weights& x) {
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
      y[e] = p[e] - (float)__builtin_bit_cast(typename T::storage, (uint16_t)(x.w[e / 2] >> 16 * (e % 2)));
    return pack(y);
  }

  // SUB tiles' share of every query.  kTwice: 16-bit weights as the sum of two numbers.  kAll: every query
  // attends every token, and each has a page.  keys(s): the lane's parts of tile s's keys; values.column(s, j):
  // its operand for elements j of the values.  Otherwise window(m) has a bit for each position of
  // the tile (one then) that query m attends, positions from `inside` on are past the row's end, and
  // bit h of `bad` says that the tile's half h has no page.
  template <int SUB, bool kAll, bool kTwice, class KeysOf, class V, class Window>
  __device__ __forceinline__ void fold(float scale, KeysOf keys, V& values, Window window, int inside,
                                       unsigned bad) {
    static_assert(kAll || SUB == 1, "tiles with masks come alone");
    const int g = threadIdx.x >> 4 & 3;
    uint32_t seen[MT];
    float d[SUB][MT][N], most[MT];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const Keys& x = keys(s);
#pragma unroll
      for (int m = 0; m < MT; ++m) scores(x, q[m], d[s][m]);
      if constexpr (SUB > 1) __builtin_amdgcn_sched_barrier(0);  // one tile's keys in registers
    }
    if constexpr (!kAll) {
      // The scores read here, in the products' block: where the masks' branches came between, ROCm 7.2's
      // compiler left two wait states of the eight (float32: ten) that a matrix instruction's result
      // needs, and the last score read was an older one.
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < N; ++e) asm volatile("" : "+v"(d[0][m][e]));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t w = (uint32_t)window(m) >> 4 * g;
        seen[m] = (w & 0xfu) | (N == 8 ? w >> 12 & 0xf0u : 0u);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = bad >> e / 4 & 1 ? __builtin_nanf("") : d[0][m][e];
          d[0][m][e] = seen[m] >> e & 1 ? x : kNegInf;
        }
      }
    }
    bool more = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      most[m] = kNegInf;
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int e = 0; e < N; ++e) most[m] = fmaxf(most[m], d[s][m][e]);
      most[m] *= scale;
      more = more || most[m] - kSlack > top[m];
    }
    if (__ballot(more)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float now = fmaxf(top[m], query_max(most[m]));
        const float less = now == kNegInf ? 1.f : exp2_fast(top[m] - now);
        top[m] = now;
        sum[m] *= less;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if constexpr (kAll && !V::kInPlace) {
            acc[m][j] *= less;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][j][e] = scaled(acc[m][j][e], less);
          }
        }
      }
    }
    float one[N];
#pragma unroll
    for (int e = 0; e < N; ++e) one[e] = 1.f;
    const Weights ones = pack(one);
    Weights w[SUB][MT], low[kTwice ? MT : 1];
    static_assert(!kTwice || SUB == 1, "two weights for one tile");
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float base = top[m] == kNegInf ? 0.f : top[m] - T::kLift;
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int e = 0; e < N; ++e) d[s][m][e] = exp2_fast(__builtin_fmaf(d[s][m][e], scale, -base));
        w[s][m] = pack(d[s][m]);
        sum[m] = product(ones, w[s][m], sum[m]);
        if constexpr (kTwice) {
          low[m] = rest(d[s][m], w[s][m]);
          sum[m] = product(ones, low[m], sum[m]);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      if constexpr (!kAll) {
        // tokens past the row's end hold anything; among the others infinities and NaN are rare
        if (__ballot(values.clear(inside - 4 * g))) {
          fold_odd(values, seen);
          values.only_finite();
        }
        if constexpr (!V::kInPlace) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            const Weights x = values.cleared(j);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][j] = product(x, w[s][m], acc[m][j]);
          }
          continue;
        }
      } else if constexpr (V::kInPlace) {
        // (an infinity times a weight's second number, or one that is 0, is none)
        if (__ballot(values.odd())) {
#pragma unroll
          for (int m = 0; m < MT; ++m) seen[m] = ~0u;
          fold_odd(values, seen);
          values.only_finite();
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const Weights x = values.column(s, j);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][j] = product(x, w[s][m], acc[m][j]);
        if constexpr (kTwice)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][j] = product(x, low[m], acc[m][j]);
      }
    }
  }

  // Whether an output of the wavefront is infinite or NaN.
  __device__ __forceinline__ bool odd() const {
    float x = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = __builtin_fmaf(acc[m][j][e], 0.f, x);
    return __ballot(x != x) != 0;
  }

  __device__ __forceinline__ static constexpr uint32_t inf_bits() {
    if constexpr (Sh::kWide) return 0x7f800000u;
    else return T::kInf;
  }
  // A sign bit of this is set where the word holds an infinite number or NaN.
  static constexpr uint32_t kSigns = Sh::kWide ? 0x80000000u : 0x80008000u;
  __device__ __forceinline__ static uint32_t odd_bits(uint32_t w) {
    constexpr uint32_t both = Sh::kWide ? 1u : 0x10001u, exponent = inf_bits() * both;
    return (w & exponent) + (0x8000u * (Sh::kWide ? 0x10000u : both) - exponent);
  }
  // The word with its infinite numbers and NaN as zeros.
  __device__ __forceinline__ static uint32_t finite(uint32_t w) {
    if constexpr (Sh::kWide) return (w & inf_bits()) == inf_bits() ? 0u : w;
    if ((w & inf_bits()) == inf_bits()) w &= 0xffff0000u;
    if ((w >> 16 & inf_bits()) == inf_bits()) w &= 0x0000ffffu;
    return w;
  }
  // 1 where a value is an infinity of the sign `negative`, or NaN (which is both), else 0.
  __device__ __forceinline__ static Weights infinite(const Weights& a, bool negative) {
    float y[N];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (Sh::kWide) {
        const float v = __uint_as_float(a.w[t]);
        y[t] = v != v || v == (negative ? kNegInf : -kNegInf) ? 1.f : 0.f;
      } else {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t v = a.w[t] >> 16 * b & 0xffffu;
          const bool nan = (v & 0x7fffu) > inf_bits();
          y[2 * t + b] = nan || v == (inf_bits() | (negative ? 0x8000u : 0u)) ? 1.f : 0.f;
        }
      }
    }
    return pack(y);
  }
  // What infinite values and NaN bring to the queries that attend them.
  template <class V>
  __device__ __forceinline__ void fold_odd(V& values, const uint32_t (&seen)[MT]) {
    Weights who[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float yes[N];
#pragma unroll
      for (int e = 0; e < N; ++e) yes[e] = seen[m] >> e & 1 ? 1.f : 0.f;
      who[m] = pack(yes);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      // one after another: interleaved, this rare path would decide the kernel's registers
      __builtin_amdgcn_sched_barrier(0);
      const Weights a = values.cleared(j), positive = infinite(a, false), negative = infinite(a, true);
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const f32x4 up = product(positive, who[m], zero), down = product(negative, who[m], zero);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (up[e] > 0.f) acc[m][j][e] += -kNegInf;
          if (down[e] > 0.f) acc[m][j][e] += kNegInf;
        }
      }
    }
  }
};

// The low `n` bits set (n <= 0: none, n >= 64: all).
__device__ __forceinline__ u64 low_bits(int n) {
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}

// Which of the 64 positions from `at` on a query may attend: those before `limit`, with a mask those
// before its prefix or set in it.  (`at`, `limit` and `prefix` are the same for a tile, or nearly.)
__device__ __forceinline__ u64 window_of(int at, int limit, int prefix, const u64* mask, int words) {
  u64 bits = low_bits(limit - at);
  if (mask != nullptr) {
    const int b = at - prefix;
    if (b >= 0) {
      const int word = b >> 6, shift = b & 63;
      u64 x = word < words ? mask[word] >> shift : 0;
      if (shift != 0 && word + 1 < words) x |= mask[word + 1] << (64 - shift);
      bits &= x;
    } else if (b > -64) {
      bits &= (words > 0 ? mask[0] << -b : 0) | low_bits(-b);
    }
  }
  return bits;
}

// The sequence of tile x and the tile's place in it.
__device__ __forceinline__ int find_tile(const Call& a, int x, int rows, int& tile) {
  if (a.offsets == nullptr) {
    const int each = tiles_before(a, 1, rows, 0);
    const int i = (unsigned)x / (unsigned)each;
    tile = x - i * each;
    return i;
  }
  const int lane = threadIdx.x & 63;
  const i64 origin = origin_of(a);
  // 64 probes a turn; the last that starts at or before x
  int low = 0, span = a.n;
  while (span > 1) {
    const int step = (span + 63) >> 6;
    const bool before = lane * step < span && tiles_before(a, low + lane * step, rows, origin) <= x;
    const int last = 63 - __clzll((long long)(__ballot(before) | 1));
    span = min(step, span - last * step);
    low += last * step;
  }
  low = same(low);
  tile = same(x - tiles_before(a, low, rows, origin));
  return low;
}

// before[i]: the work of the sequences before i; before[n]: all of it.  `scratch`: kWaves numbers.
__device__ __forceinline__ void sum_work(const Call& a, int rows, int tokens, unsigned* before,
                                         unsigned* scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned carry = 0;
  for (int base = 0; base < a.n; base += 64 * kWaves) {
    const int i = base + threadIdx.x;
    unsigned x = i < a.n ? work_of(a, i, rows, tokens) : 0;
    const unsigned mine = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned y = __shfl_up(x, off);
      if (lane >= off) x = plus(x, y);
    }
    if (lane == 63) scratch[wave] = x;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) x = plus(x, scratch[w]);
      total = plus(total, scratch[w]);
    }
    if (i < a.n) before[i] = plus(carry, x) - mine;
    carry = plus(carry, total);
    __syncthreads();
  }
  if (threadIdx.x == 0) before[a.n] = carry;
  __syncthreads();
}

// Workgroups in an order that gives consecutive ones to one XCD (they go round the 8 of them): tiles
// of one sequence read the same keys.
__device__ __forceinline__ unsigned in_order() {
  const unsigned groups = gridDim.x, whole = groups & ~7u;
  return blockIdx.x < whole ? (blockIdx.x & 7) * (whole >> 3) + (blockIdx.x >> 3) : blockIdx.x;
}

// Stores W consecutive elements.
template <class S, int W>
__device__ __forceinline__ void store_run(S* p, const float (&x)[W]) {
  struct alignas(sizeof(S) * W) Run {
    S v[W];
  } y;
#pragma unroll
  for (int e = 0; e < W; ++e) y.v[e] = (S)x[e];
  *reinterpret_cast<Run*>(p) = y;
}
template <int W>
__device__ __forceinline__ void store_floats(float* p, const float (&x)[W]) {
#pragma unroll
  for (int e = 0; e < W; e += W < 4 ? 2 : 4) {
    if constexpr (W < 4) *reinterpret_cast<float2*>(p + e) = make_float2(x[e], x[e + 1]);
    else *reinterpret_cast<float4*>(p + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
  }
}

// The 16 MT queries of a wavefront: query lane & 15 of each 16 is the lane's.
template <int MT>
struct Queries {
  bool real[MT];
  int index[MT];  // in the sequence
  int token[MT], head[MT];
  __device__ __forceinline__ void find(const Call& a, const Sequence& s, int key_head, int row0, int M) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = row0 + 16 * m + (threadIdx.x & 15), held = min(row, M - 1);
      real[m] = row < M;
      index[m] = (unsigned)held / (unsigned)a.group;
      token[m] = s.first + index[m];
      head[m] = key_head * a.group + (held - index[m] * a.group);
    }
  }
  template <class Wv>
  __device__ __forceinline__ void load(const Call& a, Wv& w) const {
    using Sh = typename Wv::Sh;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const char* at = a.q + token[m] * a.q_stride + head[m] * (Sh::KC * 64) + (threadIdx.x >> 4 & 3) * 16;
#pragma unroll
      for (int k = 0; k < Sh::KC; ++k) {
        u32x4 y = *reinterpret_cast<const u32x4*>(at + k * 64);
        y ^= a.flip;
        w.q[m][k] = real[m] ? y : u32x4{0, 0, 0, 0};
      }
    }
  }
  // Of the 64 positions from `at` on, those that the lane's query m attends.
  __device__ __forceinline__ u64 window(const Call& a, const Sequence& s, int m, int at) const {
    const u64* mask = a.mask ? a.mask + (a.mask_rows == a.tokens ? token[m] : index[m]) * (i64)a.words : nullptr;
    const int limit = a.mask ? s.end : end_of(s, index[m]);
    return window_of(at, limit, s.prefix, mask, a.words);
  }
};

// The lane's row 4 g + i of O^T (element(j, 4 g + i) of query m) to its place: out, or a part.
// `part_row`: the query's row in the part's slot, or -1.
template <class T, int DH, int MT>
__device__ __forceinline__ void finish(const Call& a, const Queries<MT>& q, int m, int i, i64 part_row,
                              bool exists, const f32x4 (&o)[DH / 16], int from, float total, float top) {
  using Sh = Shape<T, DH>;
  using S = typename T::storage;
  if (!q.real[m]) return;
  const int g = threadIdx.x >> 4 & 3;
  if (part_row >= 0) {
#pragma unroll
    for (int h = 0; h < Sh::H; ++h) {
      float y[Sh::W];
#pragma unroll
      for (int e = 0; e < Sh::W; ++e) y[e] = o[h * Sh::W + e][from];
      store_floats<Sh::W>(a.part_o + part_row * DH + Sh::element(h * Sh::W, 4 * g + i), y);
    }
    if (i == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + part_row * 2) = make_float2(top, total);
    return;
  }
  const float scale = !exists ? __builtin_nanf("") : total == 0.f ? 0.f : 1.f / total;
  S* out = reinterpret_cast<S*>(a.out) + ((i64)q.token[m] * a.heads + q.head[m]) * DH;
#pragma unroll
  for (int h = 0; h < Sh::H; ++h) {
    float y[Sh::W];
#pragma unroll
    for (int e = 0; e < Sh::W; ++e) y[e] = o[h * Sh::W + e][from] * scale;
    store_run<S, Sh::W>(out + Sh::element(h * Sh::W, 4 * g + i), y);
  }
}

// Who does an item.
enum Mode {
  kEach,    // a wavefront
  kGroup,   // a workgroup, whose wavefronts take every fourth tile of tokens and merge through LDS
  kShared,  // workgroups that share out all items' tokens
};

template <class T, int DH, int MT>
constexpr size_t merge_bytes() {
  return (size_t)kWaves * MT * 64 * (DH / 4 + 2) * sizeof(float);
}
constexpr size_t kShareBytes = (kMostShared + 1 + kWaves) * sizeof(unsigned);

template <class T, int DH, int MT, int MODE>
__global__ __launch_bounds__(64 * kWaves) void tree_kernel(Call a) {
  using Sh = Shape<T, DH>;
  using Wv = Wave<T, DH, MT>;
  constexpr int KT = Sh::KT, N = Sh::N, NJ = Sh::NJ;
  constexpr int kRows = 16 * MT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned group = in_order();
  Job job;
  Share share;
  if constexpr (MODE == kShared) {
    unsigned* before = reinterpret_cast<unsigned*>(lds + merge_bytes<T, DH, MT>());
    if (threadIdx.x == 0) note_none(a, group);
    sum_work(a, kRows, KT, before, before + kMostShared + 1);
    share = share_of(a, before, group, gridDim.x, kWaves);  // a tile of tokens each wavefront
  } else {
    const unsigned item = MODE == kEach ? group * kWaves + wave : group;
    if (item >= (unsigned)a.items) return;
    const int x = item / (unsigned)c.kv_heads;
    job.head = item - x * (unsigned)c.kv_heads;
    job.s = same(sequence_at(a, find_tile(a, x, kRows, job.tile)));
    job.from = 0, job.to = 1 << 30, job.slot = -1;
    if ((i64)job.tile * kRows >= (i64)job.s.queries * a.group) return;
  }
  while (true) {
    if constexpr (MODE == kShared) {
      if (!share.next(a, kRows, KT, job)) return;
    }
    const Sequence& s = job.s;
    const int M = s.queries * a.group, row0 = job.tile * kRows;
    Queries<MT> q;
    q.find(a, s, job.head, row0, M);
    Wv w;
    w.clear();
    if (s.exists) {
      // positions that some query of the tile attends end at `end`, those that all do at `full`
      const int q_first = (unsigned)row0 / (unsigned)a.group;
      const int q_last = (unsigned)min(row0 + kRows - 1, M - 1) / (unsigned)a.group;
      const int end = a.mask ? s.end : end_of(s, q_last);
      const int full_tiles = (a.mask ? s.prefix : end_of(s, q_first)) / KT;
      const int to = min(job.to, (end + KT - 1) / KT);
      const int step = MODE == kEach ? 1 : kWaves;
      const int begin = job.from + (MODE == kEach ? 0 : wave);
      q.load(a, w);
      const i64 head_offset = a.layer_offset + slot_offset(c, 0, job.head, 0);
      const char* k_head = c.k + head_offset;
      const char* v_head = c.v + head_offset;
      const int32_t* table = c.table + s.row * c.width;
      // the pages of the next 64 tiles, one a lane; -1 for none (past the last: the last's).  Without a branch
      // by lanes: at its end, in the largest of these kernels, the compiler (ROCm 7.2) saved a register that
      // all lanes need while only those of the branch were on
      int ids0 = -1, ids1 = -1;
      const auto pages_from = [&](int tile) {
        const int first = min(tile + lane * step, to - 1) * KT, last = min(first + KT, end) - 1;
        ids0 = page_of(c, table[first >> c.page_shift]);
        ids1 = page_of(c, table[last >> c.page_shift]);
      };
      typename Wv::Keys now, next;
      typename Wv::Values values;
      int at = 0;  // the current tile among the 64
      int id0 = 0, id1 = 0, next0 = 0, next1 = 0;
      const int in_page = (1 << c.page_shift) - 1;
      const auto offset = [&](int id, int position) {  // of 16 tokens from a position on
        return (i64)max(id, 0) * c.page_bytes + (position & in_page) * (DH * Sh::E);
      };
      if (begin < to) {
        pages_from(begin);
        id0 = __builtin_amdgcn_readlane(ids0, 0), id1 = __builtin_amdgcn_readlane(ids1, 0);
        load_keys<T, DH>(k_head + offset(id0, begin * KT), k_head + offset(id1, begin * KT + 16), now.k);
      }
      int tile = begin;
      // first the tiles that all of it attends, in a loop without what the others need
      const auto run = [&](auto all) __attribute__((always_inline)) {
        for (; tile < to && (!all || (tile < full_tiles && min(id0, id1) >= 0)); tile += step) {
          load_values<T, DH>(v_head + offset(id0, tile * KT), v_head + offset(id1, tile * KT + 16), values.v);
          if (++at == 64) {
            at = 0;
            pages_from(tile + step);
          }
          if (tile + step < to) {
            next0 = __builtin_amdgcn_readlane(ids0, at), next1 = __builtin_amdgcn_readlane(ids1, at);
            load_keys<T, DH>(k_head + offset(next0, (tile + step) * KT),
                             k_head + offset(next1, (tile + step) * KT + 16), next.k);
          }
          w.template fold<1, decltype(all)::value, !Sh::kWide>(
              a.scale_log2, [&](int) -> const typename Wv::Keys& { return now; }, values,
              [&](int m) { return q.window(a, s, m, tile * KT); }, end - tile * KT,
              (unsigned)(id0 < 0) | (unsigned)(id1 < 0) << 1);
          now = next;
          id0 = next0, id1 = next1;
        }
      };
      run(std::true_type());
      run(std::false_type());
    }
    const i64 slot = MODE == kShared && job.slot >= 0 ? ((i64)group * 2 + job.slot) * kRows : -1;
    if constexpr (MODE == kEach) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          finish<T, DH, MT>(a, q, m, i, -1, s.exists, w.acc[m], i, w.sum[m][0], w.top[m]);
      return;
    } else {
      // merge: [wave][m][j][i][lane] sums, then [wave][m][2][lane] maxima and totals
      float* merged = reinterpret_cast<float*>(lds);
      constexpr int kPart = MT * NJ * 4 * 64;
      float* tops = merged + kWaves * kPart;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            merged[wave * kPart + ((m * NJ + j) * 4 + i) * 64 + lane] = w.acc[m][j][i];
        tops[((wave * MT + m) * 2 + 0) * 64 + lane] = w.top[m];
        tops[((wave * MT + m) * 2 + 1) * 64 + lane] = w.sum[m][0];
      }
      __syncthreads();
      const int i = wave;  // each wavefront finishes every fourth row
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float top = kNegInf, total = 0.f, less[kWaves];
#pragma unroll
        for (int v = 0; v < kWaves; ++v) top = fmaxf(top, tops[((v * MT + m) * 2) * 64 + lane]);
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
          const float t = tops[((v * MT + m) * 2) * 64 + lane];
          less[v] = t == kNegInf ? 0.f : exp2_fast(t - top);
          total += tops[((v * MT + m) * 2 + 1) * 64 + lane] * less[v];
        }
        f32x4 o[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          o[j][0] = 0.f;
#pragma unroll
          for (int v = 0; v < kWaves; ++v)
            o[j][0] += scaled(merged[v * kPart + ((m * NJ + j) * 4 + i) * 64 + lane], less[v]);
        }
        finish<T, DH, MT>(a, q, m, i, slot < 0 ? -1 : slot + 16 * m + r, s.exists, o, 0, total, top);
      }
    }
    if constexpr (MODE != kShared) return;
    if (threadIdx.x == 0) note(a, group, job, kRows);
    __syncthreads();  // the merge's last readers
  }
}

// Many rows: a workgroup's 4 wavefronts have 32 rows each and share tiles of 64 tokens (32 at dh 256)
// in LDS, in two buffers (32 KiB at dh 64, else 64), which global_load_lds_dwordx4 fills without going
// through registers (1,024 consecutive bytes of LDS an instruction; a wavefront brings a quarter of a
// tile).  A token's 16-byte parts are exchanged there, so that what is read at once comes from
// different banks: the same part of 16 keys, or 32 bytes of four values, which ds_read_b64_tr_b16 turns
// as it reads (four lanes a token's 16 elements in, one element's four tokens a lane out; no
// v_perm_b32).  Elements j of the values are 16 j ... 16 j + 15 here.
template <class T, int DH>
struct Chunk {
  static constexpr int kTokens = DH == 256 ? 32 : 64;
  static constexpr int MT = 2, kRows = 16 * MT * kWaves;
  static constexpr int kToken = DH * 2;             // bytes
  static constexpr int kTile = kTokens * kToken;    // of keys, and of values
  static constexpr int kBuffers = 2, kLds = kBuffers * 2 * kTile;
  static_assert(kLds <= 65536, "the loads' place in LDS has 16 bits");
  static constexpr int kResident = DH == 64 ? 3 : DH == 128 ? 2 : 1;  // workgroups a compute unit
  static constexpr int kBlocks = kTokens / 16;      // of 16 tokens, which share a page
  static constexpr int kSub = kTokens / 32;
  static constexpr int kParts = DH / 8;             // 16-byte parts a token
  static constexpr int kBring = kTokens / kWaves;   // tokens a wavefront brings
  static constexpr int kLoads = kBring * kToken / 1024;  // of keys, and as many of values
  // Where part `part` of a key or value lies among its token's.
  __device__ __forceinline__ static int key_part(int token, int part) {
    return part ^ (kParts >= 16 ? token & 15 : token >> 1 & 7);
  }
  __device__ __forceinline__ static int value_part(int token, int part) {
    return part ^ (kParts >= 16 ? token & 3 : token >> 1 & 1) * 2;
  }
  static constexpr int kTurns = kParts >= 16 ? 4 : 2;  // places of elements j that differ by more than j
  static constexpr int kKeyTurns = kParts >= 16 ? 4 : 2;  // and of a key's parts 4 p + g
};

// 16 bytes a lane from base + offset to LDS at `to` + 16 lane; waited for by wait_loads().  In
// assembly, since the compiler takes every later read of LDS for one of what such a load brings and
// waits for it first; here a barrier stands between them.  A load to LDS must not come directly behind
// the scalar instruction that writes m0 (one wait state), which the compiler does not see to in here.
__device__ __forceinline__ void load_to_lds(const char* base, unsigned offset, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base)
               : "memory", "m0");
}
// Until at most kLeft of them are on their way.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}

// Four 16-bit numbers a lane: of each 16 lanes, number l of those that lanes 4 k ... 4 k + 3 name
// together, k = 0 ... 3.
__device__ __forceinline__ uint2 read_turned(const char* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 Lds;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)p));
}

// The lane's elements 16 j + 4 g ... + 3 of query m to their place: out, or a part (finish).
template <class T, int DH, int MT>
__device__ __forceinline__ void finish_turned(const Call& a, const Queries<MT>& q, int m, i64 part_row,
                                     bool exists, const f32x4 (&o)[DH / 16], float total, float top) {
  using S = typename T::storage;
  if (!q.real[m]) return;
  const int g = threadIdx.x >> 4 & 3;
  if (part_row >= 0) {
#pragma unroll
    for (int j = 0; j < DH / 16; ++j)
      *reinterpret_cast<f32x4*>(a.part_o + part_row * DH + 16 * j + 4 * g) = o[j];
    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + part_row * 2) = make_float2(top, total);
    return;
  }
  const float scale = !exists ? __builtin_nanf("") : total == 0.f ? 0.f : 1.f / total;
  S* out = reinterpret_cast<S*>(a.out) + ((i64)q.token[m] * a.heads + q.head[m]) * DH;
#pragma unroll
  for (int j = 0; j < DH / 16; ++j) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = o[j][e] * scale;
    store_run<S, 4>(out + 16 * j + 4 * g, y);
  }
}

// A tile's values in LDS; `at`: where the lane reads its elements j, j below kTurns, of the first.
template <class T, int DH>
struct TurnedValues {
  using Wv = Wave<T, DH, Chunk<T, DH>::MT>;
  using Weights = typename Wv::Weights;
  static constexpr bool kInPlace = false;
  static constexpr int kToken = Chunk<T, DH>::kToken, kTurns = Chunk<T, DH>::kTurns;
  const char* at[kTurns];
  uint32_t held[4];
  bool all_finite;
  __device__ __forceinline__ Weights column(int s, int j) const {
    const char* x = at[j % kTurns] + 32 * s * kToken + j / kTurns * kTurns * 32;
    const uint2 low = read_turned(x), high = read_turned(x + 16 * kToken);
    return Weights{{low.x, low.y, high.x, high.y}};
  }
  __device__ __forceinline__ Weights cleared(int j) const {
    Weights x = column(0, j);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x.w[t] &= held[t];
      if (all_finite) x.w[t] = Wv::finite(x.w[t]);
    }
    return x;
  }
  __device__ __forceinline__ bool clear(int until) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      held[t] = (Wv::Sh::place(2 * t) < until ? 0xffffu : 0u) |
                (Wv::Sh::place(2 * t + 1) < until ? 0xffff0000u : 0u);
    all_finite = false;
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < Wv::NJ; ++j) {
      const Weights x = cleared(j);
#pragma unroll
      for (int t = 0; t < 4; ++t) odd |= Wv::odd_bits(x.w[t]);
    }
    asm volatile("" ::: "memory");  // read again afterwards, not kept
    return odd & Wv::kSigns;
  }
  __device__ __forceinline__ void only_finite() {
    all_finite = true;
    asm volatile("" ::: "memory");
  }
};

template <class T, int DH, int MODE>
__global__ __launch_bounds__(64 * kWaves, (Chunk<T, DH>::kResident)) void chunk_kernel(Call a) {
  using Ch = Chunk<T, DH>;
  constexpr int MT = Ch::MT;
  using Sh = Shape<T, DH>;
  using Wv = Wave<T, DH, MT>;
  constexpr int N = Sh::N, NJ = Sh::NJ;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned group = in_order();
  Job job;
  Share share;
  if constexpr (MODE == kShared) {
    unsigned* before = reinterpret_cast<unsigned*>(lds + Ch::kLds);
    if (threadIdx.x == 0) note_none(a, group);
    sum_work(a, Ch::kRows, Ch::kTokens, before, before + kMostShared + 1);
    share = share_of(a, before, group, gridDim.x, 4);
  } else {
    if (group >= (unsigned)a.items) return;
    const int x = group / (unsigned)c.kv_heads;
    job.head = group - x * (unsigned)c.kv_heads;
    job.s = same(sequence_at(a, find_tile(a, x, Ch::kRows, job.tile)));
    job.from = 0, job.to = 1 << 30, job.slot = -1;
    if ((i64)job.tile * Ch::kRows >= (i64)job.s.queries * a.group) return;
  }
  const unsigned lds_at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // the parts that the lane brings of its wavefront's 16 tokens
  unsigned bring_k[Ch::kLoads], bring_v[Ch::kLoads];
#pragma unroll
  for (int i = 0; i < Ch::kLoads; ++i) {
    const int token = wave * Ch::kBring % 16 + (i * 64 + lane) / Ch::kParts, part = lane % Ch::kParts;
    bring_k[i] = token * Ch::kToken + Ch::key_part(token, part) * 16;
    bring_v[i] = token * Ch::kToken + Ch::value_part(token, part) * 16;
  }
  // what it reads: key r's parts 4 p + g, and elements j of value 4 g + r / 4
  unsigned key_at[Ch::kKeyTurns], value_at[Ch::kTurns];
#pragma unroll
  for (int p = 0; p < Ch::kKeyTurns; ++p) key_at[p] = r * Ch::kToken + Ch::key_part(r, 4 * p + g) * 16;
#pragma unroll
  for (int j = 0; j < Ch::kTurns; ++j) {
    const int token = 4 * g + (r >> 2), part = 2 * j + (r >> 1 & 1);
    value_at[j] = token * Ch::kToken + Ch::value_part(token, part) * 16 + (r & 1) * 8;
  }
  while (true) {
    if constexpr (MODE == kShared) {
      if (!share.next(a, Ch::kRows, Ch::kTokens, job)) return;
    }
    const Sequence& s = job.s;
    const int M = s.queries * a.group, row0 = job.tile * Ch::kRows, mine0 = row0 + wave * 16 * MT;
    Queries<MT> q;
    q.find(a, s, job.head, mine0, M);
    Wv w;
    w.clear();
    if (s.exists) {
      // positions that some query of the workgroup attends end at `end`, those that all do at `full`
      const int q_first = (unsigned)row0 / (unsigned)a.group;
      const int q_last = (unsigned)min(row0 + Ch::kRows - 1, M - 1) / (unsigned)a.group;
      const int end = a.mask ? s.end : end_of(s, q_last);
      const int full = a.mask ? s.prefix : end_of(s, q_first);
      const int to = min(job.to, (end + Ch::kTokens - 1) / Ch::kTokens);
      q.load(a, w);
      const i64 head_offset = a.layer_offset + slot_offset(c, 0, job.head, 0);
      const char* k_head = c.k + head_offset;
      const char* v_head = c.v + head_offset;
      const int32_t* table = c.table + s.row * c.width;
      // the pages of the next 64 blocks of 16 tokens, one a lane; -1 for none (past the end: the last)
      int ids = -1;
      const auto pages_from = [&](int tile) {
        const int first = min(tile * Ch::kTokens + lane * 16, end - 1);
        ids = page_of(c, table[first >> c.page_shift]);
      };
      // Brings a tile to a buffer; kBlocks bits of `bad` a buffer: blocks without a page.
      unsigned bad = 0;
      int block;  // the next tile's first among the lanes' 64
      const auto fetch = [&](int tile, int buffer) {
        if (block == 64) {
          block = 0;
          pages_from(tile);
        }
        unsigned none = 0;
#pragma unroll
        for (int b = 0; b < Ch::kBlocks; ++b)
          none |= (unsigned)(__builtin_amdgcn_readlane(ids, block + b) < 0) << b;
        const int shift = buffer * Ch::kBlocks;
        bad = (bad & ~(((1u << Ch::kBlocks) - 1) << shift)) | none << shift;
        const int page = max(__builtin_amdgcn_readlane(ids, block + wave * Ch::kBring / 16), 0);
        block += Ch::kBlocks;
        const int first = tile * Ch::kTokens + wave * Ch::kBring / 16 * 16;
        const i64 from = (i64)page * c.page_bytes + (first & ((1 << c.page_shift) - 1)) * Ch::kToken;
        const unsigned here = lds_at + buffer * 2 * Ch::kTile + wave * Ch::kLoads * 1024;
#pragma unroll
        for (int i = 0; i < Ch::kLoads; ++i) {
          load_to_lds(k_head + from, bring_k[i], here + i * 1024);
          load_to_lds(v_head + from, bring_v[i], here + Ch::kTile + i * 1024);
        }
      };
      constexpr int kAhead = Ch::kBuffers - 1;  // tiles on their way while one is worked on
      int buffer, tile;
      const auto start = [&]() __attribute__((always_inline)) {
        buffer = block = 0, tile = job.from;
        if (tile < to) {
          pages_from(tile);
#pragma unroll
          for (int t = 0; t < kAhead; ++t)
            if (tile + t < to) fetch(tile + t, t);
          if (tile + kAhead <= to) wait_loads<(kAhead - 1) * 2 * Ch::kLoads>();
          else wait_loads<0>();
          __syncthreads();
        }
      };
      // first the tiles that all of it attends, in a loop without what the others need
      const auto run = [&](auto all) __attribute__((always_inline)) {
        for (; tile < to; ++tile) {
          const unsigned now = bad >> buffer * Ch::kBlocks & ((1u << Ch::kBlocks) - 1);
          if (all && ((tile + 1) * Ch::kTokens > full || now)) break;
          const bool more = tile + kAhead < to;
          if (more) fetch(tile + kAhead, buffer == 0 ? kAhead : buffer - 1);
          const char* keys = lds + buffer * 2 * Ch::kTile;
          TurnedValues<T, DH> values;
#pragma unroll
          for (int j = 0; j < Ch::kTurns; ++j) values.at[j] = keys + Ch::kTile + value_at[j];
          const auto part = [&](int t) {
            typename Wv::Keys x;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int p = 0; p < Sh::KC; ++p)
                x.k[h][p] = *reinterpret_cast<const u32x4*>(keys + key_at[p % Ch::kKeyTurns] +
                                                            p / Ch::kKeyTurns * Ch::kKeyTurns * 64 +
                                                            (32 * t + 16 * h) * Ch::kToken);
            return x;
          };
          if (mine0 >= M) {
          } else if constexpr (decltype(all)::value) {
            w.template fold<Ch::kSub, true, false>(a.scale_log2, part, values, [](int) { return u64(0); }, 0, 0u);
          } else {
            u64 seen[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) seen[m] = q.window(a, s, m, tile * Ch::kTokens);
#pragma unroll 1
            for (int t = 0; t < Ch::kSub; ++t) {
              w.template fold<1, false, false>(
                  a.scale_log2, [&](int) { return part(t); }, values, [&](int m) { return seen[m] >> 32 * t; },
                  end - tile * Ch::kTokens - 32 * t, now >> 2 * t);
#pragma unroll
              for (int j = 0; j < Ch::kTurns; ++j) values.at[j] += 32 * Ch::kToken;
            }
          }
          buffer = buffer == kAhead ? 0 : buffer + 1;
          // the next tile is there; nobody reads this one any more
          if (more) wait_loads<(kAhead - 1) * 2 * Ch::kLoads>();
          else wait_loads<0>();
          __syncthreads();
        }
      };
      // Outputs that are not finite: everything once more, by all wavefronts, as tiles with masks, which
      // take infinite values apart (an infinity times a weight that is 0 is NaN).
      start();
      run(std::true_type());
      run(std::false_type());
      int* again = reinterpret_cast<int*>(lds);  // nobody reads or brings a tile now
      if (threadIdx.x == 0) *again = 0;
      __syncthreads();
      if (w.odd() && lane == 0) *again = 1;
      __syncthreads();
      const int odd = same(*again);
      __syncthreads();  // its readers
      if (odd) {
        w.clear();
        start();
        run(std::false_type());
      }
    }
    const i64 slot = MODE == kShared && job.slot >= 0 ? ((i64)group * 2 + job.slot) * Ch::kRows : -1;
#pragma unroll
    for (int m = 0; m < MT; ++m)
      finish_turned<T, DH, MT>(a, q, m, slot < 0 ? -1 : slot + (wave * MT + m) * 16 + r, s.exists, w.acc[m],
                               w.sum[m][0], w.top[m]);
    if constexpr (MODE != kShared) return;
    if (threadIdx.x == 0) note(a, group, job, Ch::kRows);
  }
}

// Joins the parts of items: a row a wavefront (or workgroup), whose lanes have a part's maximum and sum
// each, then four elements of every 64 / (DH / 4)-th part.
template <class T, int DH>
__global__ __launch_bounds__(64 * kWaves) void join_kernel(Call a, int rows, int groups) {
  using S = typename T::storage;
  constexpr int kLanes = DH / 4, kSides = 64 / kLanes;
  const int lane = threadIdx.x & 63;
  const int x = blockIdx.x / (unsigned)a.c.kv_heads, key_head = blockIdx.x - x * a.c.kv_heads;
  int tile;
  const int sequence = find_tile(a, x, rows, tile);
  const Sequence s = sequence_at(a, sequence);
  const int M = s.queries * a.group, row0 = tile * rows;
  if (row0 >= M) return;
  const int group = begun_by(a, blockIdx.x, groups);
  if (group < 0) return;
  const bool did = did_begin(a, group, blockIdx.x, sequence);
  int parts = 1;
  for (int base = group + 1; base < groups; base += 64) {
    const u64 ends = __ballot(base + lane < groups && a.ended[min(base + lane, groups - 1)]);
    if (ends) {
      parts = base - group + __builtin_ctzll(ends) + 1;
      break;
    }
  }
  if (!did) return;
  // many parts of a row: the workgroup's wavefronts take 64 of them in turn and merge through LDS
  __shared__ float merged[kWaves][64][6];
  const int wave = threadIdx.x >> 6;
  const bool together = parts > 32;
  const int first = together ? wave * 64 : 0, step = together ? kWaves * 64 : 64;
  const auto slot = [&](int k, int row) { return ((i64)(group + k) * 2 + (k == 0)) * rows + row; };
  for (int base_row = blockIdx.y * (together ? 1 : kWaves); base_row < rows && row0 + base_row < M;
       base_row += gridDim.y * (together ? 1 : kWaves)) {
    const int row = base_row + (together ? 0 : wave);
    if (row >= rows || row0 + row >= M) continue;  // (of those that merge, none)
    float top = kNegInf;
    for (int k = first + lane; k < parts; k += step) top = fmaxf(top, a.part_ml[slot(k, row) * 2]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
    float total;
    f32x4 o;
    const int side = lane / kLanes, at = lane % kLanes * 4;
    const auto sum_up = [&](auto small) __attribute__((always_inline)) {
      total = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int base = first; base < parts; base += step) {
        float less = 0.f;
        if (base + lane < parts) {
          const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + slot(base + lane, row) * 2);
          less = ml.x == kNegInf ? 0.f : exp2_fast(ml.x - top);
          total += ml.y * less;
        }
        const int here = min(64, parts - base);
#pragma unroll 16
        for (int k = 0; k < here; k += kSides) {
          const int mine = k + side;
          const float weight = __shfl(less, mine & 63);
          if (mine < here) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(a.part_o + slot(base + mine, row) * DH + at);
            if constexpr (decltype(small)::value) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] += scaled(y[e], weight);
            } else {
              o += y * weight;
            }
          }
        }
      }
    };
    sum_up(std::false_type());
    const float sum = o[0] + o[1] + o[2] + o[3];
    if (__ballot(sum - sum != 0.f)) sum_up(std::true_type());  // infinities of parts whose weight is 0
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) total += __shfl_xor(total, off);
#pragma unroll
    for (int off = kLanes; off < 64; off <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off);
    if (together) {
      float* mine = merged[wave][lane];
      mine[0] = top, mine[1] = total;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[2 + e] = o[e];
      __syncthreads();
      float least = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) least = fmaxf(least, merged[w][lane][0]);
      total = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float* x = merged[w][lane];
        const float less = x[0] == kNegInf ? 0.f : exp2_fast(x[0] - least);
        total += x[1] * less;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += scaled(x[2 + e], less);
      }
      __syncthreads();  // its readers
      if (wave != 0) continue;
    }
    if (side != 0) continue;
    const float scale = total == 0.f ? 0.f : 1.f / total;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = o[e] * scale;
    const int query = (unsigned)(row0 + row) / (unsigned)a.group;
    const int head = key_head * a.group + (row0 + row - query * a.group);
    store_run<S, 4>(reinterpret_cast<S*>(a.out) + ((i64)(s.first + query) * a.heads + head) * DH + at, y);
  }
}

// ------------------------------------------------------------------------------ the host's part

inline int current_units() {
  thread_local int device = -1, count = 256;
  int now = 0;
  if (hipGetDevice(&now) != hipSuccess) return 256;
  if (now != device) {
    int units = 0;
    count = hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, now) == hipSuccess &&
                    units > 0 ? units : 256;
    device = now;
  }
  return count;
}

// What a call's launch is.
struct Plan {
  int rows;    // a tile's: 16 MT of tree_kernel, 128 of chunk_kernel
  Mode mode;
  i64 groups;  // workgroups
};

// Rows a tile by the rows a sequence has on the mean; an item a wavefront where that fills the
// device, else a workgroup, and where rows may be long (by the table's width: lengths are on the
// device) their tokens shared out.  Sharing out costs a second launch and 5 us: at 64 queries x 4
// heads of one row (dh 64), us of a workgroup an item / shared, 540 tokens 17 / 22, 1,100 tokens 25 /
// 23, 2,200 tokens 42 / 27; at 4 queries 1,100 tokens 10.3 / 14.4, 2,200 tokens 15.8 / 17.
inline int plan(Call* a, int dh, int size, Plan* p) {
  const i64 rows = ((i64)a->tokens * a->group + a->n - 1) / a->n;
  const int cus = current_units();
  // chunk_kernel for many rows: more than 64, or than 32 where few items leave the memory to be kept
  // busy (24 rows of up to 32,768 tokens, dh 128: 42 rows 327 us against 484, 16 rows 316 against 312;
  // 4,096 rows of up to 320 tokens, 6 rows 832 against 610)
  const bool many = ((i64)a->tokens * a->group / 32 + a->n) * a->c.kv_heads >= 8 * cus;
  const bool chunks = size == 2 && dh >= 64 && rows > (many ? 64 : 32);
  p->rows = chunks ? 128 : rows <= 16 || dh == 256 ? 16 : 32;
  const i64 tiles = a->offsets ? (i64)a->tokens * a->group / p->rows + a->n
                               : a->n * (((i64)a->each * a->group + p->rows - 1) / p->rows);
  const i64 items = tiles * a->c.kv_heads;
  if (items >= (i64)1 << 26) return -1;
  const i64 longest = (i64)a->c.width << a->c.page_shift;
  a->items = (int)items;
  p->groups = items;
  const i64 most = items * ((longest + 15) / 16);  // tiles of tokens, which are counted in 32 bits
  if (items < 8 * cus && a->n <= kMostShared && longest > (chunks ? 1024 : 4096) &&
      most < (i64)1 << 31) {
    p->mode = kShared;
    p->groups = (!chunks ? 4 : dh == 64 ? 3 : dh == 128 ? 2 : 1) * cus;
    if (p->groups > most) p->groups = most;
  } else if (chunks || items < 8 * cus) {
    p->mode = kGroup;
  } else {
    p->mode = kEach;
    p->groups = (items + kWaves - 1) / kWaves;
  }
  return p->groups < (i64)1 << 24 ? 0 : -1;  // a launch has fewer than 2^32 threads in x
}

inline i64 part_floats(const Plan& p, int dh) { return p.groups * 2 * p.rows * dh; }
inline i64 part_bytes(const Plan& p, int dh, i64 items) {
  return p.mode != kShared ? 0
                           : (part_floats(p, dh) + p.groups * 2 * p.rows * 2) * (i64)sizeof(float) +
                                 p.groups * (i64)sizeof(int2) + (items + p.groups) * (i64)sizeof(int);
}

// A launch with more than 64 KiB of LDS has to say so once a device and kernel.
template <class K>
int allow_lds(K* kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <class K>
int launch(K* kernel, const Call& a, i64 groups, size_t lds, hipStream_t stream) {
  if (const int bad = allow_lds(kernel, lds)) return bad;
  hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(64 * kWaves), lds, stream, a);
  return (int)hipGetLastError();
}

template <class T, int DH, int MT>
int by_mode(const Call& a, const Plan& p, hipStream_t stream) {
  constexpr size_t kMerge = merge_bytes<T, DH, MT>();
  if (p.mode == kEach) return launch(tree_kernel<T, DH, MT, kEach>, a, p.groups, 0, stream);
  if (p.mode == kGroup) return launch(tree_kernel<T, DH, MT, kGroup>, a, p.groups, kMerge, stream);
  return launch(tree_kernel<T, DH, MT, kShared>, a, p.groups, kMerge + kShareBytes, stream);
}

template <class T, int DH>
int by_rows(const Call& a, const Plan& p, hipStream_t stream) {
  constexpr int kSize = sizeof(typename T::storage);
  int rc = -1;
  if (p.rows == 16) rc = by_mode<T, DH, 1>(a, p, stream);
  if constexpr (DH < 256) {
    if (p.rows == 32) rc = by_mode<T, DH, 2>(a, p, stream);
  }
  if constexpr (kSize == 2 && DH >= 64) {
    constexpr size_t kTiles = Chunk<T, DH>::kLds;
    if (p.rows == 128)
      rc = p.mode == kGroup ? launch(chunk_kernel<T, DH, kGroup>, a, p.groups, kTiles, stream)
                            : launch(chunk_kernel<T, DH, kShared>, a, p.groups, kTiles + kShareBytes, stream);
  }
  if (rc || p.mode != kShared) return rc;
  // about 2,048 workgroups, or one a row (of many parts)
  const int want = 2048 / a.items + 1;
  hipLaunchKernelGGL((join_kernel<T, DH>), dim3((unsigned)a.items, (unsigned)(want < p.rows ? want : p.rows)),
                     dim3(64 * kWaves), 0, stream, a, p.rows, (int)p.groups);
  return (int)hipGetLastError();
}

template <class T>
int by_dh(const Call& a, const Plan& p, int dh, hipStream_t stream) {
  switch (dh) {
    case 32:
      return by_rows<T, 32>(a, p, stream);
    case 64:
      return by_rows<T, 64>(a, p, stream);
    case 128:
      return by_rows<T, 128>(a, p, stream);
    default:
      return by_rows<T, 256>(a, p, stream);
  }
}

// Checks a call as its documentation says and gives the kernels' view of it.
inline int view(const CugoTreeAttention* p, Call* a) {
  if (!p) return -1;
  if (const int bad = view(p->cache, &a->c)) return bad;
  if (p->layer < 0 || p->layer >= p->cache->layers || p->tokens < 0 || p->n < 0) return -1;
  if (p->heads <= 0 || p->heads > 65535 || p->heads % p->cache->kv_heads != 0) return -1;
  if (p->tokens >= (i64)1 << 24 || p->n >= (i64)1 << 24 || p->tokens * p->heads >= (i64)1 << 31)
    return -1;
  if (p->q_stride < p->heads * p->cache->dh || p->words < 0 || p->words > (1 << 16)) return -1;
  if (!(p->scale > 0.f || p->scale < 0.f) || p->scale - p->scale != 0.f) return -1;
  if (p->tokens > 0 && (p->n == 0 || !p->q || !p->prefix || !p->out)) return -1;
  if (!p->offsets && p->n > 0 && p->tokens % p->n != 0) return -1;
  if (p->mask && p->mask_rows != p->tokens &&
      (p->offsets || p->n == 0 || p->mask_rows != p->tokens / p->n))
    return -1;
  const int size = element_size(p->cache->dtype);
  if (!aligned16(p->q) || !aligned16(p->out) || p->q_stride * size % 16 != 0) return -4;
  a->layer_offset = p->layer * a->c.layer_bytes;
  a->q = static_cast<const char*>(p->q);
  a->q_stride = p->q_stride * size;
  a->tokens = (int)p->tokens;
  a->n = (int)p->n;
  a->each = p->n > 0 ? (int)(p->tokens / p->n) : 0;
  a->heads = (int)p->heads;
  a->group = (int)(p->heads / p->cache->kv_heads);
  a->prefix = p->prefix;
  a->rows = p->rows;
  a->offsets = p->offsets;
  a->mask = reinterpret_cast<const u64*>(p->mask);
  a->mask_rows = p->mask_rows;
  a->words = (int)p->words;
  const float scale = p->scale < 0.f ? -p->scale : p->scale;
  a->flip = p->scale < 0.f ? (size == 4 ? 0x80000000u : 0x80008000u) : 0u;
  a->scale_log2 = scale * 1.4426950408889634f;  // softmax in base 2
  if (a->scale_log2 - a->scale_log2 != 0.f) return -1;
  a->out = static_cast<char*>(p->out);
  a->part_o = a->part_ml = nullptr;
  a->left = nullptr;
  a->begun = a->ended = nullptr;
  return 0;
}

}  // namespace paged
}  // namespace cugo_amd

extern "C" {

int64_t cugo_tree_attention_workspace(const CugoTreeAttention* call) {
  using namespace cugo_amd::paged;
  Call a;
  Plan p;
  if (view(call, &a) || a.tokens == 0) return 0;
  const int dh = (int)call->cache->dh;
  return plan(&a, dh, element_size(call->cache->dtype), &p) ? 0 : part_bytes(p, dh, a.items);
}

int cugo_tree_attention(const CugoTreeAttention* call, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream) {
  using namespace cugo_amd::paged;
  Call a;
  Plan p;
  if (const int bad = view(call, &a)) return bad;
  if (a.tokens == 0) return 0;
  const int dh = (int)call->cache->dh;
  if (const int bad = plan(&a, dh, element_size(call->cache->dtype), &p)) return bad;
  if (const int64_t need = part_bytes(p, dh, a.items)) {
    if (!workspace) return -1;
    if (!aligned16(workspace)) return -4;
    if (workspace_bytes < need) return -5;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + part_floats(p, dh);
    a.left = reinterpret_cast<int2*>(a.part_ml + p.groups * 2 * p.rows * 2);
    a.begun = reinterpret_cast<int*>(a.left + p.groups);
    a.ended = a.begun + a.items;
  }
  switch (call->cache->dtype) {
    case CUGO_DTYPE_BF16:
      return by_dh<BF16>(a, p, dh, stream);
    case CUGO_DTYPE_F16:
      return by_dh<F16>(a, p, dh, stream);
    default:
      return by_dh<F32>(a, p, dh, stream);
  }
}

}  // extern "C"
