// One AdamW step over many tensors in one launch for each 32 of them, behind a launch that
// raises the step counts and, where the gradients are clipped, sums their squares.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   w = (1 - lr d) w - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors' addresses travel in the kernel's arguments (nothing to copy to the device, and a
// captured launch keeps them); a workgroup takes chunks of kChunk values and finds each chunk's
// tensor by bisection.  Memory bounds it: 28 bytes a value with float32 moments and parameters or
// with a bf16 weight, its master and a bf16 gradient, 16 of the latter with 8-bit moments.  35.4M
// values: 174 us (5.7 TB/s, the gradients partly from the last-level cache, which the 48 us of the
// norm's launch filled), with 8-bit moments 118 us (4.8 TB/s).  A whole chunk's loads are all in
// flight before the first is used (187 and 158 us when each access waited for its own).  2M values
// take 14 us, most of it the latencies of a launch in which a wavefront has one chunk.
//
// 8-bit moments: a block of 256 values shares a float32 scale, its largest value; m is kept as
// e4m3 and v, whose values span the squares of the gradients' range, as e5m2.  b2 = 0.999 moves
// v by a thousandth a step where neighbouring codes are 14 to 25 % apart: rounded to nearest, v
// would stay where it is for good.  So both are rounded up or down by chance, with a mean of the
// value itself; the chance is a hash of the seed, the tensor, the step and the value's place.
// A v above 0 is kept at the smallest code at least, so that a weight whose gradient is seldom
// is not divided by eps alone.
#include "learner.h"

#include <math.h>

namespace cugo_amd {
namespace learner {
namespace adamw {

constexpr int kThreads = 256;
constexpr int kEach = 4;                        // values of a thread's access
constexpr int kRounds = 4;                      // accesses of a thread in a chunk
constexpr int kChunk = kThreads * kEach * kRounds;
constexpr int kTable = 32;                      // tensors of a launch: 2.5 KB of arguments
constexpr int kPartials = 1024;                 // most workgroups of a launch
constexpr int kBlock = CUGO_ADAMW_BLOCK;
static_assert(kBlock == 64 * kEach, "a block is one access of a wavefront");
constexpr uint32_t kPlaceStep = 0x9E3779B9u;

// 32 bits mixed: two multiplications by odd constants (the fractions of the golden ratio and of
// the square root of 3) between shifted exclusive ors.
__host__ __device__ inline uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 17)) * 0x9E3779B9u;
  x = (x ^ (x >> 14)) * 0xBB67AE85u;
  return x ^ (x >> 15);
}

struct Tensor {
  void* param;
  const void* grad;
  float* master;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  i64 numel;
  int place;
  int16_t param_dtype, grad_dtype;
};

// What the counting launch leaves for the update, for each tensor.
struct Factors {
  float decay, step_size, root;  // 1 - lr d, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t key;                  // of the rounding words
};

struct Table {
  Tensor tensor[kTable];
  uint32_t chunk_end[kTable];  // chunks of the tensors up to and with this one
  int count;
};

struct CountArgs {
  const void* grad[kTable];
  int64_t* step[kTable];
  i64 numel[kTable];
  double lr[kTable], weight_decay[kTable];
  uint32_t chunk_end[kTable];
  int place[kTable];
  int16_t grad_dtype[kTable];
  int count;
  double beta1, beta2;
  const float* lr_scale;
  uint32_t seed_key;
  bool norm;
  Factors* factors;
  double* partials;
};

// The table's tensor that chunk c belongs to.
__device__ inline int tensor_of(const uint32_t* chunk_end, int count, uint32_t c) {
  int low = 0, high = count - 1;
  while (low < high) {
    const int mid = (low + high) / 2;
    if (chunk_end[mid] > c) high = mid;
    else low = mid + 1;
  }
  return low;
}

// Values i .. i + 3 of a tensor's gradient as float32; `whole`: all four exist, and the address
// is aligned for one access.
template <class T>
__device__ inline void load4_as(const void* p, i64 i, i64 n, bool whole, float (&x)[kEach]) {
  using S = typename T::storage;
  const S* s = static_cast<const S*>(p) + i;
  if (whole) {
    const Vec<S, kEach> v = *reinterpret_cast<const Vec<S, kEach>*>(s);
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = T::to_float(v.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = i + e < n ? T::to_float(s[e]) : 0.0f;
  }
}
__device__ inline void load4(int dtype, const void* p, i64 i, i64 n, bool whole,
                             float (&x)[kEach]) {
  if (dtype == CUGO_DTYPE_F32) load4_as<F32>(p, i, n, whole, x);
  else if (dtype == CUGO_DTYPE_F16) load4_as<F16>(p, i, n, whole, x);
  else load4_as<BF16>(p, i, n, whole, x);
}
template <class T>
__device__ inline void store4_as(void* p, i64 i, i64 n, bool whole, const float (&x)[kEach]) {
  using S = typename T::storage;
  S* s = static_cast<S*>(p) + i;
  if (whole) {
    Vec<S, kEach> v;
#pragma unroll
    for (int e = 0; e < kEach; ++e) v.v[e] = T::from_float(x[e]);
    *reinterpret_cast<Vec<S, kEach>*>(s) = v;
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (i + e < n) s[e] = T::from_float(x[e]);
  }
}
__device__ inline void store4(int dtype, void* p, i64 i, i64 n, bool whole,
                              const float (&x)[kEach]) {
  if (dtype == CUGO_DTYPE_F32) store4_as<F32>(p, i, n, whole, x);
  else if (dtype == CUGO_DTYPE_F16) store4_as<F16>(p, i, n, whole, x);
  else store4_as<BF16>(p, i, n, whole, x);
}

__device__ inline bool aligned(const void* p, int bytes) {
  return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0;
}
__device__ inline int value_bytes(int dtype) { return dtype == CUGO_DTYPE_F32 ? 4 : 2; }

__device__ inline double power(double x, int64_t n) {
  double y = 1.0;
  for (; n > 0; n >>= 1, x *= x)
    if (n & 1) y *= x;
  return y;
}

// The sum over the workgroup, in every thread, in a fixed order.
__device__ inline double workgroup_sum(double x) {
  __shared__ double waves[kThreads / 64];
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = x;
  __syncthreads();
  double total = 0.0;
  for (int k = 0; k < kThreads / 64; ++k) total += waves[k];
  __syncthreads();
  return total;
}

// Raises each tensor's step count and forms the step's factors (the first workgroup); sums the
// squares of the gradients, a partial sum for each workgroup.
__global__ __launch_bounds__(kThreads) void adamw_count_kernel(const CountArgs g) {
  if (blockIdx.x == 0 && (int)threadIdx.x < g.count) {
    const int k = threadIdx.x;
    const int64_t t = ++*g.step[k];
    const double lr = g.lr[k] * (g.lr_scale ? (double)*g.lr_scale : 1.0);
    Factors f;
    f.decay = (float)(1.0 - lr * g.weight_decay[k]);
    f.step_size = (float)(lr / (1.0 - power(g.beta1, t)));
    f.root = (float)(1.0 / sqrt(1.0 - power(g.beta2, t)));
    f.key = mix32(mix32(g.seed_key + (uint32_t)g.place[k]) + (uint32_t)t);
    g.factors[k] = f;
  }
  if (!g.norm) return;
  double sum = 0.0;
  const uint32_t chunks = g.chunk_end[g.count - 1];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int k = tensor_of(g.chunk_end, g.count, c);
    const i64 base = (i64)(c - (k ? g.chunk_end[k - 1] : 0)) * kChunk;
    const void* grad = g.grad[k];
    const i64 n = g.numel[k];
    const int dtype = g.grad_dtype[k];
    const bool fits = aligned(grad, kEach * value_bytes(dtype));
    float x[kRounds][kEach];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const i64 i = base + (r * kThreads + (int)threadIdx.x) * kEach;
      load4(dtype, grad, i, n, fits && i + kEach <= n, x[r]);
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
#pragma unroll
      for (int e = 0; e < kEach; ++e) sum = __builtin_fma((double)x[r][e], (double)x[r][e], sum);
  }
  sum = workgroup_sum(sum);
  if (threadIdx.x == 0) g.partials[blockIdx.x] = sum;
}

struct UpdateArgs {
  Table table;
  float beta1, beta2, rest1, rest2, eps;  // rest: 1 - beta
  double max_norm;                        // 0: not clipped
  const Factors* factors;
  const double* partials;                 // of all the step's counting launches
  int partial_count;
  float* norm_out;
};

// The largest of 64 lanes' x in every lane: within the rows of 16 lanes, then over the rows by
// broadcasts of a row's last lane to the next ones (lane 63 then has it).
__device__ inline uint32_t wavefront_max(uint32_t x) {
  const auto with = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // rows 0, 2 to 1, 3
  x = with(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // rows 1 to 2, 3
  return __builtin_amdgcn_readlane(x, 63);
}

// Four values rounded to codes by chance, and the block's scale.  x >= 0 or NaN where !kE4m3.
// The largest size is found on the bits, where a NaN is above an infinity above all numbers.
template <bool kE4m3>
__device__ inline uint32_t to_codes(const float (&x)[kEach], const uint32_t (&word)[kEach],
                                    float& scale) {
  constexpr float kTop = kE4m3 ? 256.0f : 32768.0f;
  uint32_t most_bits = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
    most_bits = b > most_bits ? b : most_bits;
  }
  most_bits = wavefront_max(most_bits);
  const float most = fmaxf(__uint_as_float(most_bits), 0x1p-100f);
  const float up = kTop / most;
  scale = most_bits >= 0x7f800000u ? NAN : most * (1.0f / kTop);
  uint32_t codes = 0;
  if constexpr (kE4m3) {
    codes = __builtin_amdgcn_cvt_sr_fp8_f32(x[0] * up, word[0], codes, 0);
    codes = __builtin_amdgcn_cvt_sr_fp8_f32(x[1] * up, word[1], codes, 1);
    codes = __builtin_amdgcn_cvt_sr_fp8_f32(x[2] * up, word[2], codes, 2);
    codes = __builtin_amdgcn_cvt_sr_fp8_f32(x[3] * up, word[3], codes, 3);
  } else {
    codes = __builtin_amdgcn_cvt_sr_bf8_f32(x[0] * up, word[0] << 16, codes, 0);
    codes = __builtin_amdgcn_cvt_sr_bf8_f32(x[1] * up, word[1] << 16, codes, 1);
    codes = __builtin_amdgcn_cvt_sr_bf8_f32(x[2] * up, word[2] << 16, codes, 2);
    codes = __builtin_amdgcn_cvt_sr_bf8_f32(x[3] * up, word[3] << 16, codes, 3);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if ((codes & (0xffu << (8 * e))) == 0 && x[e] > 0.0f) codes |= 1u << (8 * e);
  }
  return codes;
}

template <bool kE4m3>
__device__ inline void from_codes(uint32_t codes, float scale, float (&x)[kEach]) {
  const auto low = kE4m3 ? __builtin_amdgcn_cvt_pk_f32_fp8(codes, false)
                         : __builtin_amdgcn_cvt_pk_f32_bf8(codes, false);
  const auto high = kE4m3 ? __builtin_amdgcn_cvt_pk_f32_fp8(codes, true)
                          : __builtin_amdgcn_cvt_pk_f32_bf8(codes, true);
  x[0] = low[0] * scale, x[1] = low[1] * scale, x[2] = high[0] * scale, x[3] = high[1] * scale;
}

__device__ inline uint32_t load_codes(const void* p, i64 i, i64 n, bool whole) {
  const uint8_t* s = static_cast<const uint8_t*>(p) + i;
  if (whole) return *reinterpret_cast<const uint32_t*>(s);
  uint32_t c = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) c |= (i + e < n ? (uint32_t)s[e] : 0u) << (8 * e);
  return c;
}
__device__ inline void store_codes(void* p, i64 i, i64 n, bool whole, uint32_t codes) {
  uint8_t* s = static_cast<uint8_t*>(p) + i;
  if (whole) {
    *reinterpret_cast<uint32_t*>(s) = codes;
    return;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (i + e < n) s[e] = (uint8_t)(codes >> (8 * e));
}

// sqrt(v) to the hardware's last place or so (v_sqrt_f32; its small arguments scaled up first,
// which it would flush).
__device__ inline float root_of(float v) {
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v);
  return small ? r * 0x1p-16f : r;
}

struct Numbers {  // of the step, and of the tensor
  float beta1, beta2, rest1, rest2, eps, clip;
  float decay, step_size, root;
};

// The step of one value.  The moments are formed in separately rounded operations, so that their
// codes follow from IEEE arithmetic; the quotient is the product with the hardware's reciprocal:
// a last place of the step, not of the weight.
__device__ inline void advance(const Numbers& c, float grad, float& w, float& m, float& v) {
  const float x = grad * c.clip;
  m = m * c.beta1 + x * c.rest1;
  v = v * c.beta2 + (x * x) * c.rest2;
  const float by = root_of(v) * c.root + c.eps;
  w = w * c.decay - c.step_size * (m * __builtin_amdgcn_rcpf(by));
}

// The moments of four values as a thread holds them between reading and computing.
template <int kBits>
struct Held;
template <>
struct Held<32> {
  Vec<float, kEach> m, v;
  __device__ void read(const Tensor& t, i64 i) {
    m = *reinterpret_cast<const Vec<float, kEach>*>(static_cast<const float*>(t.m) + i);
    v = *reinterpret_cast<const Vec<float, kEach>*>(static_cast<const float*>(t.v) + i);
  }
};
template <>
struct Held<8> {
  uint32_t m, v;
  float m_scale, v_scale;
  __device__ void read(const Tensor& t, i64 i) {
    m = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.m) + i);
    v = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.v) + i);
    const i64 block = i / kBlock;
    m_scale = t.m_scale[block], v_scale = t.v_scale[block];
  }
};

// A whole chunk of an aligned tensor with P parameters and G gradients: kBatch accesses of each
// stream are in flight before the first is used.
template <int kBits, class P, class G>
__device__ inline void whole_chunk(const Tensor& t, const Numbers& c, i64 base, uint32_t key) {
  using GS = typename G::storage;
  constexpr bool kMaster = sizeof(typename P::storage) == 2;
  constexpr int kBatch = kBits == 8 ? 4 : 2;
  float* w32 = kMaster ? t.master : static_cast<float*>(t.param);
#pragma unroll
  for (int r0 = 0; r0 < kRounds; r0 += kBatch) {
    Vec<GS, kEach> gv[kBatch];
    Vec<float, kEach> wv[kBatch];
    Held<kBits> held[kBatch];
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      const i64 i = base + ((r0 + r) * kThreads + (int)threadIdx.x) * kEach;
      gv[r] = *reinterpret_cast<const Vec<GS, kEach>*>(static_cast<const GS*>(t.grad) + i);
      wv[r] = *reinterpret_cast<const Vec<float, kEach>*>(w32 + i);
      held[r].read(t, i);
    }
#pragma unroll
    for (int r = 0; r < kBatch; ++r) {
      const i64 i = base + ((r0 + r) * kThreads + (int)threadIdx.x) * kEach;
      float w[kEach], m[kEach], v[kEach];
      if constexpr (kBits == 8) {
        from_codes<true>(held[r].m, held[r].m_scale, m);
        from_codes<false>(held[r].v, held[r].v_scale, v);
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        w[e] = wv[r].v[e];
        if constexpr (kBits == 32) m[e] = held[r].m.v[e], v[e] = held[r].v.v[e];
        advance(c, G::to_float(gv[r].v[e]), w[e], m[e], v[e]);
      }
      store4_as<F32>(w32, i, 0, true, w);
      if constexpr (kMaster) store4_as<P>(t.param, i, 0, true, w);
      if constexpr (kBits == 8) {
        uint32_t word[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) word[e] = mix32((uint32_t)(i + e) ^ key);
        float m_scale, v_scale;
        store_codes(t.m, i, 0, true, to_codes<true>(m, word, m_scale));
        store_codes(t.v, i, 0, true, to_codes<false>(v, word, v_scale));
        if (threadIdx.x % 64 == 0) {
          t.m_scale[i / kBlock] = m_scale;
          t.v_scale[i / kBlock] = v_scale;
        }
      } else {
        store4_as<F32>(t.m, i, 0, true, m);
        store4_as<F32>(t.v, i, 0, true, v);
      }
    }
  }
}

// Any chunk, of any types: a tensor's last one, or one whose addresses fit no wide access.
template <int kBits>
__device__ inline void any_chunk(const Tensor& t, const Numbers& c, i64 base, uint32_t key) {
  const i64 n = t.numel;
  float* w32 = t.master ? t.master : static_cast<float*>(t.param);
  for (int r = 0; r < kRounds; ++r) {
    const i64 i = base + (r * kThreads + (int)threadIdx.x) * kEach;
    const i64 block = i / kBlock;  // the same for the wavefront
    if (block * kBlock >= n) continue;
    float gr[kEach], w[kEach], m[kEach], v[kEach];
    load4(t.grad_dtype, t.grad, i, n, false, gr);
    load4_as<F32>(w32, i, n, false, w);
    if constexpr (kBits == 8) {
      from_codes<true>(load_codes(t.m, i, n, false), t.m_scale[block], m);
      from_codes<false>(load_codes(t.v, i, n, false), t.v_scale[block], v);
    } else {
      load4_as<F32>(t.m, i, n, false, m);
      load4_as<F32>(t.v, i, n, false, v);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) advance(c, gr[e], w[e], m[e], v[e]);
    store4_as<F32>(w32, i, n, false, w);
    if (t.master) store4(t.param_dtype, t.param, i, n, false, w);
    if constexpr (kBits == 8) {
      uint32_t word[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        word[e] = mix32((uint32_t)(i + e) ^ key);
        if (i + e >= n) m[e] = v[e] = 0.0f;
      }
      float m_scale, v_scale;
      const uint32_t mc = to_codes<true>(m, word, m_scale);
      const uint32_t vc = to_codes<false>(v, word, v_scale);
      store_codes(t.m, i, n, false, mc);
      store_codes(t.v, i, n, false, vc);
      if (threadIdx.x % 64 == 0) {
        t.m_scale[block] = m_scale;
        t.v_scale[block] = v_scale;
      }
    } else {
      store4_as<F32>(t.m, i, n, false, m);
      store4_as<F32>(t.v, i, n, false, v);
    }
  }
}

template <int kBits, class P>
__device__ inline void whole_chunk_of(const Tensor& t, const Numbers& c, i64 base, uint32_t key) {
  if (t.grad_dtype == CUGO_DTYPE_F32) whole_chunk<kBits, P, F32>(t, c, base, key);
  else if (t.grad_dtype == CUGO_DTYPE_F16) whole_chunk<kBits, P, F16>(t, c, base, key);
  else whole_chunk<kBits, P, BF16>(t, c, base, key);
}

template <int kBits>
__global__ __launch_bounds__(kThreads) void adamw_update_kernel(const UpdateArgs g) {
  Numbers c{g.beta1, g.beta2, g.rest1, g.rest2, g.eps, 1.0f, 0.0f, 0.0f, 0.0f};
  if (g.max_norm > 0.0) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < g.partial_count; i += kThreads) sum += g.partials[i];
    const float norm = (float)sqrt(workgroup_sum(sum));
    const float clip = (float)g.max_norm / (norm + 1e-6f);
    c.clip = clip > 1.0f ? 1.0f : clip;  // a NaN norm stays one, and so do the weights
    if (g.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *g.norm_out = norm;
  }
  const uint32_t chunks = g.table.chunk_end[g.table.count - 1];
  for (uint32_t at = blockIdx.x; at < chunks; at += gridDim.x) {
    const int k = tensor_of(g.table.chunk_end, g.table.count, at);
    const i64 base = (i64)(at - (k ? g.table.chunk_end[k - 1] : 0)) * kChunk;
    const Tensor& t = g.table.tensor[k];
    const Factors f = g.factors[k];
    c.decay = f.decay, c.step_size = f.step_size, c.root = f.root;
    const uint32_t key = mix32(f.key + (uint32_t)((uint64_t)base >> 32) * kPlaceStep);
    const bool fits =
        base + kChunk <= t.numel && aligned(t.grad, kEach * value_bytes(t.grad_dtype)) &&
        aligned(t.param, kEach * value_bytes(t.param_dtype)) && aligned(t.master, 16) &&
        aligned(t.m, kBits == 8 ? 4 : 16) && aligned(t.v, kBits == 8 ? 4 : 16);
    if (!fits) any_chunk<kBits>(t, c, base, key);
    else if (t.param_dtype == CUGO_DTYPE_F32) whole_chunk_of<kBits, F32>(t, c, base, key);
    else if (t.param_dtype == CUGO_DTYPE_F16) whole_chunk_of<kBits, F16>(t, c, base, key);
    else whole_chunk_of<kBits, BF16>(t, c, base, key);
  }
}

inline int groups_for(uint32_t chunks, int most) {
  return chunks < (uint32_t)most ? (int)chunks : most;
}

inline i64 launches_of(i64 count) { return (count + kTable - 1) / kTable; }

}  // namespace adamw
}  // namespace learner
}  // namespace cugo_amd

using namespace cugo_amd::learner;
using namespace cugo_amd::learner::adamw;

extern "C" {

int64_t cugo_adamw_workspace(int64_t count) {
  if (count < 1) return 0;
  return launches_of(count) *
         (int64_t)(kTable * sizeof(Factors) + kPartials * sizeof(double));
}

int cugo_adamw(const CugoAdamwTensor* tensors, int64_t count, int bits, double beta1,
               double beta2, double eps, const float* lr_scale, double max_norm, uint64_t seed,
               float* norm_out, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (count < 0 || (count > 0 && (!tensors || !workspace)) || count > (1 << 20)) return -1;
  if (bits != 8 && bits != 32) return -2;
  if (count > 0 && workspace_bytes < cugo_adamw_workspace(count)) return -3;
  for (int64_t i = 0; i < count; ++i) {
    const CugoAdamwTensor& t = tensors[i];
    if (t.numel < 0 || t.numel > ((int64_t)1 << 36)) return -1;  // chunks count in 32 bits
    if (!dtype_known(t.param_dtype) || !dtype_known(t.grad_dtype)) return -2;
    if (!t.step) return -1;
    if (t.numel > 0 && ((t.param_dtype == CUGO_DTYPE_F32) != (t.master == nullptr))) return -1;
    if (t.numel > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq)) return -1;
    if (t.numel > 0 && bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return -1;
  }
  const i64 launches = launches_of(count);
  double* partials = static_cast<double*>(workspace);
  Factors* factors = reinterpret_cast<Factors*>(partials + launches * kPartials);
  const uint32_t seed_key = mix32((uint32_t)seed ^ mix32((uint32_t)(seed >> 32) + 1u));
  int partial_count = 0;
  for (i64 l = 0; l < launches; ++l) {
    CountArgs g{};
    uint32_t end = 0;
    g.count = (int)(count - l * kTable < kTable ? count - l * kTable : kTable);
    for (int k = 0; k < g.count; ++k) {
      const CugoAdamwTensor& t = tensors[l * kTable + k];
      end += (uint32_t)((t.numel + kChunk - 1) / kChunk);
      g.grad[k] = t.grad, g.step[k] = t.step, g.numel[k] = t.numel, g.lr[k] = t.lr;
      g.weight_decay[k] = t.weight_decay, g.chunk_end[k] = end, g.place[k] = t.place;
      g.grad_dtype[k] = t.grad_dtype;
    }
    g.beta1 = beta1, g.beta2 = beta2, g.lr_scale = lr_scale, g.seed_key = seed_key;
    g.norm = max_norm > 0.0;
    g.factors = factors + l * kTable;
    g.partials = partials + partial_count;
    const int groups = g.norm && end > 0 ? groups_for(end, kPartials) : 1;
    adamw_count_kernel<<<groups, kThreads, 0, stream>>>(g);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    partial_count += g.norm ? groups : 0;
  }
  for (i64 l = 0; l < launches; ++l) {
    UpdateArgs g{};
    uint32_t end = 0;
    g.table.count = (int)(count - l * kTable < kTable ? count - l * kTable : kTable);
    for (int k = 0; k < g.table.count; ++k) {
      const CugoAdamwTensor& t = tensors[l * kTable + k];
      end += (uint32_t)((t.numel + kChunk - 1) / kChunk);
      g.table.chunk_end[k] = end;
      g.table.tensor[k] = Tensor{t.param, t.grad, t.master, t.exp_avg, t.exp_avg_sq,
                                 t.exp_avg_scale, t.exp_avg_sq_scale, t.numel, t.place,
                                 t.param_dtype, t.grad_dtype};
    }
    g.beta1 = (float)beta1, g.beta2 = (float)beta2, g.rest1 = (float)(1.0 - beta1);
    g.rest2 = (float)(1.0 - beta2), g.eps = (float)eps, g.max_norm = max_norm;
    g.factors = factors + l * kTable;
    g.partials = partials, g.partial_count = partial_count;
    g.norm_out = l == 0 ? norm_out : nullptr;
    if (end == 0 && !(l == 0 && norm_out && max_norm > 0.0)) continue;
    const int groups = end > 0 ? groups_for(end, compute_units() * 8) : 1;
    if (bits == 8) adamw_update_kernel<8><<<groups, kThreads, 0, stream>>>(g);
    else adamw_update_kernel<32><<<groups, kThreads, 0, stream>>>(g);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  return 0;
}

}  // extern "C"
