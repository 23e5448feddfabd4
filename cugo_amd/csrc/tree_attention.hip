// Attention of drafted tokens over a paged key/value cache, for gfx950 (include/cugo_hip.h,
// cugo_tree_attention):
//
//   out[i, h, :] = sum_t softmax_t(q[i, h, :] . K[t] scale) V[t]
//
// over the positions t of the query's row that lie before its sequence's prefix or whose bit is
// set in its mask.  A sequence's queries and the heads that share a key head make the M = queries x
// group rows of one product with that head's keys, 16 MT of them (MT = 1, 2, 4) a wavefront, so
// each key and value is read once for all of them.  A wavefront goes through tiles of 32 tokens (16
// in float32) with one running maximum and sum; nothing but the partial results of split rows leaves
// it.
//
// Scores are formed as S^T = K Q^T (16 x 16 matrix instructions, K the A operand), so that a lane
// has one query's scores (lane & 15) of a few tokens; those are the weights' places in the B operand
// of O^T += V^T P^T too, if a tile's tokens are dealt to the rows of the two K operands as
// 8 (r / 4) + r % 4 (+ 4): weights never move between lanes.  V^T's A operand takes, for one
// element of the head, 8 tokens a lane: a lane loads W consecutive elements of each of its tokens (16
// lanes cover a token's row) and turns the 8 x W block by v_perm_b32, so keys and values both come
// straight from memory into registers in whole rows.
//
// The running maximum moves only when a score exceeds it by more than 2^8 in the weight (kSlack):
// until then weights are at most 2^8, which neither type nor the sums mind, and a tile needs no
// exchange between lanes.  Weights are rounded to the cache's type for the product with V; their sum
// is taken from the rounded ones (a matrix instruction with ones), so they add up to one.
//
// Tiles in which some query may not see some token (the drafts, a row's end) take their scores
// from the masks, and values that are infinite or NaN there go through products of their own
// (indicators of +inf and -inf), since 0 x inf would show in queries that do not attend them.
#include "paged.h"

namespace cugo_amd {
namespace paged {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

struct BF16 {
  using storage = __bf16;
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7f80u;
  __device__ static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a),
                                                   __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct F16 {
  using storage = _Float16;
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kInf = 0x7c00u;
  __device__ static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a),
                                                  __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct F32 {
  using storage = float;
};

struct Call {
  Cache c;
  i64 layer_offset;
  const char* q;
  i64 q_stride;  // bytes
  i64 mask_rows;
  const i64* prefix;
  const i64* rows;
  const i64* offsets;
  const u64* mask;
  char* out;
  float* part_o;     // of split rows: [splits, tokens * heads, dh]
  float* part_ml;    // [splits, tokens * heads, 2]: maximum (base 2) and sum
  int tokens, n, each;  // each: queries a sequence without offsets
  int heads, group, words;
  int tiles;         // of 16 MT rows, over all sequences
  int items;         // (tile, key head, split) in all
  int parts, splits;
  float scale_log2;  // > 0: a negative scale turns q's signs
  uint32_t flip;
};

constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.f;
constexpr int kWaves = 4;

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest over the four lanes that hold one query (lane & 15).
__device__ inline float query_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// W bytes / 4 words at p.
template <int N>
__device__ inline void load_words(const char* p, uint32_t (&w)[N]) {
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
  // The element that row 4 g + i of tile j of O^T is.
  __device__ static int element(int j, int row) { return j / W * 16 * W + W * row + j % W; }
};

template <class T, int DH, int MT>
struct Wave {
  using Sh = Shape<T, DH>;
  static constexpr int KT = Sh::KT, N = Sh::N, KC = Sh::KC, KL = Sh::KL, NJ = Sh::NJ;
  u32x4 q[MT][KC];
  f32x4 acc[MT][NJ];
  f32x4 sum[MT];
  float top[MT];

  struct Tile {
    u32x4 k[KL][KC];
    uint32_t v[N][Sh::H][Sh::RW];
  };

  // Reads tile `tile` whose halves lie in pages id0 and id1 (of the pool).
  __device__ static void load(const Cache& c, const char* k_head, const char* v_head, int tile,
                              int id0, int id1, Tile& x) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int in_page = (1 << c.page_shift) - 1;
    const int from = tile * KT & in_page;
    const int k_token = Sh::kWide ? r : 8 * (r >> 2) + (r & 3);
    const char* kb = k_head + (i64)(!Sh::kWide && k_token >= 16 ? id1 : id0) * c.page_bytes +
                     ((from + k_token) & in_page) * (DH * Sh::E) + g * 16;
    const char* vb = v_head + (i64)(!Sh::kWide && g >= 2 ? id1 : id0) * c.page_bytes +
                     ((from + N * g) & in_page) * (DH * Sh::E) + r * (Sh::W * Sh::E);
#pragma unroll
    for (int a = 0; a < KL; ++a)
#pragma unroll
      for (int p = 0; p < KC; ++p)
        x.k[a][p] = *reinterpret_cast<const u32x4*>(kb + a * 4 * DH * Sh::E + p * 64);
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int h = 0; h < Sh::H; ++h)
        load_words<Sh::RW>(vb + t * DH * Sh::E + h * 16 * Sh::W * Sh::E, x.v[t][h]);
  }

  // d[e]: the product of query lane & 15 with the lane's token e.
  __device__ static void scores(const Tile& x, const u32x4 (&qm)[KC], float (&d)[N]) {
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

  // A product operand of N numbers, rounded to the type.
  struct Weights {
    uint32_t w[4];
  };
  __device__ static Weights pack(const float (&p)[N]) {
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
  __device__ static f32x4 product(const Weights& a, const Weights& p, f32x4 c) {
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
  // Element j of the lane's N tokens.
  __device__ static Weights column(const Tile& x, int j) {
    Weights y;
    const int h = j / Sh::W, e = j % Sh::W;
    if constexpr (Sh::kWide) {
#pragma unroll
      for (int t = 0; t < 4; ++t) y.w[t] = x.v[t][h][e];
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        y.w[t] = __builtin_amdgcn_perm(x.v[2 * t + 1][h][e / 2], x.v[2 * t][h][e / 2],
                                       e & 1 ? 0x07060302u : 0x05040100u);
    }
    return y;
  }

  // The tile's share of every query.  `seen[m]`: bits of the lane's tokens that query m may
  // attend; all: every query attends every token.
  __device__ void fold(Tile& x, float scale, bool all, const uint32_t (&seen)[MT], int inside,
                       bool bad) {
    float d[MT][N];
    float most[MT];
    bool more = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      scores(x, q[m], d[m]);
      if (bad)
#pragma unroll
        for (int e = 0; e < N; ++e) d[m][e] = __builtin_nanf("");
      if (!all)
#pragma unroll
        for (int e = 0; e < N; ++e) d[m][e] = seen[m] >> e & 1 ? d[m][e] : kNegInf;
      most[m] = d[m][0];
#pragma unroll
      for (int e = 1; e < N; ++e) most[m] = fmaxf(most[m], d[m][e]);
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
        for (int j = 0; j < NJ; ++j) acc[m][j] *= less;
      }
    }
    Weights w[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float base = top[m] == kNegInf ? 0.f : top[m];
#pragma unroll
      for (int e = 0; e < N; ++e) d[m][e] = exp2_fast(__builtin_fmaf(d[m][e], scale, -base));
      w[m] = pack(d[m]);
    }
    float one[N];
#pragma unroll
    for (int e = 0; e < N; ++e) one[e] = 1.f;
    const Weights ones = pack(one);
#pragma unroll
    for (int m = 0; m < MT; ++m) sum[m] = product(ones, w[m], sum[m]);
    if (!all) {
      // tokens past the row's end hold anything; among the others infinities and NaN are rare
      bool odd = false;
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int h = 0; h < Sh::H; ++h)
#pragma unroll
          for (int e = 0; e < Sh::RW; ++e) {
            const uint32_t y = t < inside ? x.v[t][h][e] : 0u;
            x.v[t][h][e] = y;
            if constexpr (Sh::kWide) odd = odd || (y & 0x7f800000u) == 0x7f800000u;
            else odd = odd || (y & T_inf()) == T_inf() || (y >> 16 & T_inf()) == T_inf();
          }
      if (__ballot(odd)) {
        fold_odd(x, seen);
        return fold_values<true>(x, w);
      }
    }
    fold_values<false>(x, w);
  }

  __device__ static constexpr uint32_t T_inf() {
    if constexpr (Sh::kWide) return 0x7f800000u;
    else return T::kInf;
  }

  template <bool kFinite>
  __device__ void fold_values(const Tile& x, const Weights (&w)[MT]) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      Weights a = column(x, j);
      if constexpr (kFinite) a = only_finite(a);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][j] = product(a, w[m], acc[m][j]);
    }
  }
  __device__ static Weights only_finite(Weights a) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (Sh::kWide) {
        a.w[t] = (a.w[t] & T_inf()) == T_inf() ? 0u : a.w[t];
      } else {
        if ((a.w[t] & T_inf()) == T_inf()) a.w[t] &= 0xffff0000u;
        if ((a.w[t] >> 16 & T_inf()) == T_inf()) a.w[t] &= 0x0000ffffu;
      }
    }
    return a;
  }
  // 1 where a value is an infinity of the sign `negative`, or NaN (which is both), else 0.
  __device__ static Weights infinite(const Weights& a, bool negative) {
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
          const bool nan = (v & 0x7fffu) > T_inf();
          y[2 * t + b] = nan || v == (T_inf() | (negative ? 0x8000u : 0u)) ? 1.f : 0.f;
        }
      }
    }
    return pack(y);
  }
  // What infinite values and NaN bring to the queries that attend them.
  __device__ void fold_odd(const Tile& x, const uint32_t (&seen)[MT]) {
#pragma unroll 1
    for (int m = 0; m < MT; ++m) {
      float yes[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        uint32_t s = seen[0];
#pragma unroll
        for (int i = 1; i < MT; ++i) s = m == i ? seen[i] : s;
        yes[e] = s >> e & 1 ? 1.f : 0.f;
      }
      const Weights who = pack(yes);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const Weights a = column(x, j);
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 up = product(infinite(a, false), who, zero);
        const f32x4 down = product(infinite(a, true), who, zero);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          if (m == i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (up[e] > 0.f) acc[i][j][e] += -kNegInf;
              if (down[e] > 0.f) acc[i][j][e] += kNegInf;
            }
      }
    }
  }
};

// Bits of the N positions from `at` on that a query may attend: before `limit` and (with a mask)
// before its prefix or set in its mask.
template <int N>
__device__ inline uint32_t seen_bits(int at, int limit, int prefix, const u64* mask, int words) {
  uint32_t bits = (1u << N) - 1;
  if (mask != nullptr) {
    const int b = at - prefix;
    if (b > -N) {
      const int first = b < 0 ? 0 : b, word = first >> 6, shift = first & 63;
      u64 x = word < words ? mask[word] >> shift : 0;
      if (shift > 64 - N && word + 1 < words) x |= mask[word + 1] << (64 - shift);
      if (b < 0) x = x << -b | ((1ull << -b) - 1);
      bits &= (uint32_t)x;
    }
  }
  const int left = limit - at;
  return left >= N ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1);
}

// The sequence of tile x and the tile's place in it.  With offsets, sequence i's tiles begin at
// floor((offsets[i] - offsets[0]) group / rows a tile) + i, which leaves room for what each needs.
struct Place {
  int sequence, tile, first, queries;
};
__device__ inline Place place_of(const Call& a, int x, int rows) {
  Place p;
  if (a.offsets == nullptr) {
    const int each = (int)(((i64)a.each * a.group + rows - 1) / rows);
    p.sequence = (unsigned)x / (unsigned)each;
    p.tile = x - p.sequence * each;
    p.first = p.sequence * a.each;
    p.queries = a.each;
    return p;
  }
  const int lane = threadIdx.x & 63;
  const i64 origin = a.offsets[0];
  const auto start = [&](int i) {
    const i64 o = a.offsets[i] - origin;
    const i64 held = o < 0 ? 0 : o > a.tokens ? a.tokens : o;
    return (int)((unsigned)(held * a.group) / (unsigned)rows) + i;
  };
  // 64 probes a turn; the last that starts at or before x
  int low = 0, span = a.n;
  while (span > 1) {
    const int step = (span + 63) >> 6;
    const int at = low + lane * step;
    const bool before = lane * step < span && start(at) <= x;
    const int last = 63 - __clzll((long long)(__ballot(before) | 1));
    span = min(step, low + span - (low + last * step));
    low += last * step;
  }
  p.sequence = __builtin_amdgcn_readfirstlane(low);
  p.tile = x - start(p.sequence);
  const i64 first = a.offsets[p.sequence], end = a.offsets[p.sequence + 1];
  const bool fine = first >= 0 && end <= a.tokens && first < end;
  p.first = fine ? (int)first : 0;
  p.queries = fine ? (int)(end - first) : 0;
  return p;
}

// Stores W consecutive elements.
template <class S, int W>
__device__ inline void store_run(S* p, const float (&x)[W]) {
  struct alignas(sizeof(S) * W) Run {
    S v[W];
  } y;
#pragma unroll
  for (int e = 0; e < W; ++e) y.v[e] = (S)x[e];
  *reinterpret_cast<Run*>(p) = y;
}
template <int W>
__device__ inline void store_floats(float* p, const float (&x)[W]) {
#pragma unroll
  for (int e = 0; e < W; e += W < 4 ? 2 : 4) {
    if constexpr (W < 4) *reinterpret_cast<float2*>(p + e) = make_float2(x[e], x[e + 1]);
    else *reinterpret_cast<float4*>(p + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
  }
}

// One item: a tile of 16 MT rows of a sequence over one key head, or a split of its tokens.  parts =
// 1: an item a wavefront.  parts = 4: an item a workgroup, whose wavefronts take every fourth tile
// of tokens and merge what they have through LDS.
template <class T, int DH, int MT>
__global__ __launch_bounds__(64 * kWaves) void tree_kernel(Call a) {
  using Sh = Shape<T, DH>;
  using S = typename T::storage;
  using Wv = Wave<T, DH, MT>;
  constexpr int KT = Sh::KT, N = Sh::N, NJ = Sh::NJ, KC = Sh::KC;
  constexpr int kRows = 16 * MT;
  extern __shared__ float merged[];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // consecutive items to one XCD (workgroups go round the 8 of them): tiles of one sequence read
  // the same keys
  const unsigned groups = gridDim.x, whole = groups & ~7u;
  const unsigned group = blockIdx.x < whole ? (blockIdx.x & 7) * (whole >> 3) + (blockIdx.x >> 3)
                                            : blockIdx.x;
  const bool together = a.parts > 1;
  const unsigned item = together ? group : group * kWaves + wave;
  if (item >= (unsigned)a.items) return;
  int x, head, split = 0;
  if (together) {
    x = item % (unsigned)a.tiles;
    const unsigned rest = item / (unsigned)a.tiles;
    head = rest % (unsigned)c.kv_heads;
    split = rest / (unsigned)c.kv_heads;
  } else {
    head = item % (unsigned)c.kv_heads;
    x = item / (unsigned)c.kv_heads;
  }
  const Place p = place_of(a, x, kRows);
  const int M = p.queries * a.group;
  const int row0 = p.tile * kRows;
  if (row0 >= M) return;
  // this lane's queries
  bool real[MT];
  int query[MT], token[MT], q_head[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = row0 + 16 * m + r;
    real[m] = row < M;
    query[m] = (unsigned)min(row, M - 1) / (unsigned)a.group;
    token[m] = p.first + query[m];
    q_head[m] = head * a.group + (min(row, M - 1) - query[m] * a.group);
  }
  const i64 cache_row = a.rows ? a.rows[p.sequence] : p.sequence;
  const bool exists = cache_row >= 0 && cache_row < c.rows;
  Wv w;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    w.top[m] = kNegInf;
    w.sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) w.acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (exists) {
    const int length = row_length(c, c.length[cache_row]);
    const i64 given = a.prefix[p.sequence];
    const int prefix = (int)(given < 0 ? 0 : given > length ? length : given);
    // positions that some query of the tile attends end at `end`, those that all do at `full`
    const int q_first = (unsigned)row0 / (unsigned)a.group;
    const int q_last = (unsigned)min(row0 + kRows - 1, M - 1) / (unsigned)a.group;
    const int end = (int)min((i64)length, (i64)prefix + (a.mask ? (i64)64 * a.words : (i64)q_last + 1));
    const int full = min(end, a.mask ? prefix : prefix + q_first + 1);
    const int count = (end + KT - 1) / KT, full_tiles = full / KT;
    const int each = (count + a.splits - 1) / a.splits;
    const int from = split * each, to = min(count, from + each);
    const int step = a.parts;
    const int begin = from + (together ? wave : 0);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const char* at = a.q + token[m] * a.q_stride + (q_head[m] * DH * Sh::E + g * 16);
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        u32x4 y = *reinterpret_cast<const u32x4*>(at + k * 64);
        y ^= a.flip;
        w.q[m][k] = real[m] ? y : u32x4{0, 0, 0, 0};
      }
    }
    const i64 head_offset = a.layer_offset + slot_offset(c, 0, head, 0);
    const char* k_head = c.k + head_offset;
    const char* v_head = c.v + head_offset;
    const int32_t* table = c.table + cache_row * c.width;
    // the pages of the next 64 tiles, one a lane; -1 for none
    int ids0 = -1, ids1 = -1;
    const auto pages_from = [&](int tile) {
      const int mine = tile + lane * step;
      ids0 = ids1 = -1;
      if (mine < to) {
        const int first = mine * KT, last = min(first + KT, end) - 1;
        ids0 = page_of(c, table[first >> c.page_shift]);
        ids1 = page_of(c, table[last >> c.page_shift]);
      }
    };
    typename Wv::Tile now, next;
    int at = 0;  // the current tile among the 64
    int id0 = 0, id1 = 0, next0 = 0, next1 = 0;
    pages_from(begin);
    if (begin < to) {
      id0 = __builtin_amdgcn_readlane(ids0, 0), id1 = __builtin_amdgcn_readlane(ids1, 0);
      Wv::load(c, k_head, v_head, begin, max(id0, 0), max(id1, 0), now);
    }
    for (int tile = begin; tile < to; tile += step) {
      if (++at == 64) {
        at = 0;
        pages_from(tile + step);
      }
      if (tile + step < to) {
        next0 = __builtin_amdgcn_readlane(ids0, at), next1 = __builtin_amdgcn_readlane(ids1, at);
        Wv::load(c, k_head, v_head, tile + step, max(next0, 0), max(next1, 0), next);
      }
      const bool all = tile < full_tiles;
      uint32_t seen[MT];
      const int mine = tile * KT + N * g;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        seen[m] = (1u << N) - 1;
        if (!all) {
          const u64* mask = a.mask ? a.mask + (a.mask_rows == a.tokens ? token[m] : query[m]) * (i64)a.words : nullptr;
          seen[m] = seen_bits<N>(mine, a.mask ? end : min(end, prefix + query[m] + 1), prefix, mask, a.words);
        }
      }
      const bool bad = (!Sh::kWide && g >= 2 ? id1 : id0) < 0;
      w.fold(now, a.scale_log2, all, seen, end - mine, bad);
      now = next;
      id0 = next0, id1 = next1;
    }
  }
  // the lane's rows of O^T: element(j, 4 g + i) of query r
  const auto finish = [&](int m, int i, const f32x4 (&o)[NJ], float total, float top) {
    (void)top;
    if (!real[m]) return;
    const i64 out_row = (i64)token[m] * a.heads + q_head[m];
    if (a.splits > 1) {
      float* po = a.part_o + ((i64)split * a.tokens * a.heads + out_row) * DH;
#pragma unroll
      for (int h = 0; h < Sh::H; ++h) {
        float y[Sh::W];
#pragma unroll
        for (int e = 0; e < Sh::W; ++e) y[e] = o[h * Sh::W + e][i];
        store_floats<Sh::W>(po + Sh::element(h * Sh::W, 4 * g + i), y);
      }
      if (i == 0 && g == 0) {
        float* ml = a.part_ml + ((i64)split * a.tokens * a.heads + out_row) * 2;
        *reinterpret_cast<float2*>(ml) = make_float2(top, total);
      }
      return;
    }
    const float scale = !exists ? __builtin_nanf("") : total == 0.f ? 0.f : 1.f / total;
    S* out = reinterpret_cast<S*>(a.out) + out_row * DH;
#pragma unroll
    for (int h = 0; h < Sh::H; ++h) {
      float y[Sh::W];
#pragma unroll
      for (int e = 0; e < Sh::W; ++e) y[e] = o[h * Sh::W + e][i] * scale;
      store_run<S, Sh::W>(out + Sh::element(h * Sh::W, 4 * g + i), y);
    }
  };
  if (!together) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) finish(m, i, w.acc[m], w.sum[m][0], w.top[m]);
    return;
  }
  // merge: [wave][m][j][i][lane] sums, then [wave][m][2][lane] maxima and totals
  constexpr int kEach = MT * NJ * 4 * 64;
  float* tops = merged + kWaves * kEach;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) merged[wave * kEach + ((m * NJ + j) * 4 + i) * 64 + lane] = w.acc[m][j][i];
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
      float y = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v)
        y += merged[v * kEach + ((m * NJ + j) * 4 + i) * 64 + lane] * less[v];
      o[j] = f32x4{y, y, y, y};
    }
    finish(m, i, o, total, top);
  }
}

// out of split rows: a wavefront's 64 / (DH / 4) rows, four elements a lane.
template <class T, int DH>
__global__ __launch_bounds__(256) void join_kernel(Call a) {
  using S = typename T::storage;
  constexpr int kLanes = DH / 4;
  const i64 rows = (i64)a.tokens * a.heads;
  const i64 row = (i64)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (row >= rows) return;
  if (a.offsets) {
    const i64 token = row / a.heads;
    if (token < a.offsets[0] || token >= a.offsets[a.n]) return;
  }
  const int at = threadIdx.x % kLanes * 4;
  float top = kNegInf;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[(s * rows + row) * 2]);
  float total = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (s * rows + row) * 2);
    const f32x4 y = *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * DH + at);
    const float less = ml.x == kNegInf ? 0.f : exp2_fast(ml.x - top);
    total += ml.y * less;
    o += y * less;
  }
  const float scale = total == 0.f ? 0.f : 1.f / total;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = o[e] * scale;
  store_run<S, 4>(reinterpret_cast<S*>(a.out) + row * DH + at, y);
}

// ------------------------------------------------------------------------------ the host's part

// What a call's launch is: rows a wavefront, wavefronts an item, splits.
struct Plan {
  int mt;
  i64 groups;
};

inline int current_units() {
  int device = 0, count = 0;
  if (hipGetDevice(&device) != hipSuccess ||
      hipDeviceGetAttribute(&count, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess)
    return 256;
  return count > 0 ? count : 256;
}

// Rows a sequence has on the mean decide MT (more rows than it has would be empty); an item a
// wavefront where there are enough of them, else four wavefronts an item, and splits of long
// rows (by the table's width: lengths are on the device) until a compute unit has four workgroups.
inline int plan(Call* a, int dh, Plan* p) {
  const i64 rows = ((i64)a->tokens * a->group + a->n - 1) / a->n;
  const int most = dh == 256 ? (a->c.token_bytes == 1024 ? 1 : 2) : a->c.token_bytes == 512 ? 2 : 4;
  p->mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  if (p->mt > most) p->mt = most;
  const int tile = 16 * p->mt;
  const i64 tiles = a->offsets ? (i64)a->tokens * a->group / tile + a->n
                               : a->n * (((i64)a->each * a->group + tile - 1) / tile);
  const i64 units = tiles * a->c.kv_heads;
  const i64 width = (i64)a->c.width << a->c.page_shift;
  const int cus = current_units();
  i64 splits = 1;
  a->parts = units >= 16 * cus ? 1 : kWaves;
  if (a->parts > 1) {
    const i64 want = (4 * cus + units - 1) / units, longest = width / 512;
    splits = want < longest ? want : longest;
    if (splits < 1) splits = 1;
    if (splits > 64) splits = 64;
  }
  const i64 items = units * splits;
  if (items >= (i64)1 << 24) return -1;
  a->tiles = (int)tiles;
  a->items = (int)items;
  a->splits = (int)splits;
  p->groups = a->parts > 1 ? items : (items + kWaves - 1) / kWaves;
  return 0;
}

inline i64 part_bytes(const Call& a, int dh) {
  return a.splits > 1 ? (i64)a.splits * a.tokens * a.heads * (dh + 2) * (i64)sizeof(float) : 0;
}

template <class T, int DH, int MT>
int launch(const Call& a, i64 groups, hipStream_t stream) {
  using Sh = Shape<T, DH>;
  constexpr size_t kMerge = (size_t)kWaves * MT * 64 * (Sh::NJ * 4 + 2) * sizeof(float);
  const size_t lds = a.parts > 1 ? kMerge : 0;
  if constexpr (kMerge > 64 * 1024) {
    if (lds > 0) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(tree_kernel<T, DH, MT>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)kMerge);
      if (e != hipSuccess) return (int)e;
    }
  }
  hipLaunchKernelGGL((tree_kernel<T, DH, MT>), dim3((unsigned)groups), dim3(64 * kWaves), lds, stream, a);
  if (a.splits > 1) {
    constexpr int kEach = 256 / (DH / 4);
    const i64 rows = (i64)a.tokens * a.heads;
    hipLaunchKernelGGL((join_kernel<T, DH>), dim3((unsigned)((rows + kEach - 1) / kEach)), dim3(256),
                       0, stream, a);
  }
  return (int)hipGetLastError();
}

template <class T, int DH>
int by_rows(const Call& a, const Plan& p, hipStream_t stream) {
  constexpr int kBytes = DH * (int)sizeof(typename T::storage);
  if (p.mt == 1) return launch<T, DH, 1>(a, p.groups, stream);
  if constexpr (kBytes < 1024) {
    if (p.mt == 2) return launch<T, DH, 2>(a, p.groups, stream);
  }
  if constexpr (kBytes < 512) {
    if (p.mt == 4) return launch<T, DH, 4>(a, p.groups, stream);
  }
  return -1;
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
  a->out = static_cast<char*>(p->out);
  a->part_o = a->part_ml = nullptr;
  return 0;
}

}  // namespace paged
}  // namespace cugo_amd

extern "C" {

int64_t cugo_tree_attention_workspace(const CugoTreeAttention* call) {
  using namespace cugo_amd::paged;
  Call a;
  Plan p;
  if (view(call, &a) || a.tokens == 0 || plan(&a, (int)call->cache->dh, &p)) return 0;
  return part_bytes(a, (int)call->cache->dh);
}

int cugo_tree_attention(const CugoTreeAttention* call, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream) {
  using namespace cugo_amd::paged;
  Call a;
  Plan p;
  if (const int bad = view(call, &a)) return bad;
  if (a.tokens == 0) return 0;
  const int dh = (int)call->cache->dh;
  if (const int bad = plan(&a, dh, &p)) return bad;
  if (const int64_t need = part_bytes(a, dh)) {
    if (!workspace) return -1;
    if (!aligned16(workspace)) return -4;
    if (workspace_bytes < need) return -5;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (int64_t)a.splits * a.tokens * a.heads * dh;
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
