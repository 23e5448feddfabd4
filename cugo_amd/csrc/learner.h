// What the learner's kernels (policy_loss.hip, advantages.hip, adamw.hip) share: the element
// types, loads of consecutive elements at any element's address, and sums over lanes.
#ifndef CUGO_LEARNER_H_
#define CUGO_LEARNER_H_

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/cugo_hip.h"

namespace cugo_amd {
namespace learner {

typedef int64_t i64;

struct F32 {
  using storage = float;
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  __device__ static float to_float(float x) { return x; }
  __device__ static float from_float(float f) { return f; }
};

struct F16 {
  using storage = _Float16;
  static constexpr uint32_t kNone = 0xfc00u;  // -inf
  __device__ static float to_float(_Float16 x) { return (float)x; }
  __device__ static _Float16 from_float(float f) { return (_Float16)f; }
};

struct BF16 {
  using storage = __bf16;
  static constexpr uint32_t kNone = 0xff80u;  // -inf
  __device__ static float to_float(__bf16 x) { return (float)x; }
  // To nearest even in hardware (v_cvt_pk_bf16_f32), as torch rounds.
  __device__ static __bf16 from_float(float f) { return (__bf16)f; }
};

// K consecutive elements, read or written in one access.
template <class S, int K>
struct alignas(sizeof(S) * K) Vec {
  S v[K];
};

// N bytes as they lie in memory, in registers: `Raw` at their own alignment, `RawAny` at any
// (global loads and stores of gfx950 take any alignment).  What is read or written as one of them
// is the elements' memory, so they may alias any type.
typedef uint16_t HalfWord __attribute__((may_alias));
typedef uint32_t Words1 __attribute__((may_alias));
typedef uint32_t Words2 __attribute__((ext_vector_type(2), may_alias));
typedef uint32_t Words4 __attribute__((ext_vector_type(4), may_alias));
template <int N>
struct RawOf;
template <>
struct RawOf<2> {
  using Raw = HalfWord;
};
template <>
struct RawOf<4> {
  using Raw = Words1;
};
template <>
struct RawOf<8> {
  using Raw = Words2;
};
template <>
struct RawOf<16> {
  using Raw = Words4;
};
template <int N>
using Raw = typename RawOf<N>::Raw;
template <int N>
struct __attribute__((packed, aligned(1), may_alias)) RawAny {
  Raw<N> v;
};

// The float32 values of 16 bytes as they are read (8 of 16 bits, or 4 of 32).
template <class T>
__device__ inline void unpack(const Words4& w, float (&f)[16 / sizeof(typename T::storage)]) {
  if constexpr (sizeof(typename T::storage) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = T::to_float(__builtin_bit_cast(typename T::storage, (uint16_t)w[k]));
      f[2 * k + 1] = T::to_float(__builtin_bit_cast(typename T::storage, (uint16_t)(w[k] >> 16)));
    }
  }
}

// x from the lane that the DPP control kCtrl names: within four lanes, or the 16 of a row.
template <int kCtrl>
__device__ inline float exchanged(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xf, 0xf, false));
}

// The sum and the largest over groups of G lanes (4 to 64), the same value in every lane: by
// exchanges within four lanes, within eight (the half row mirrored) or 16 (rotations), and beyond.
// v_max_f32 takes the other operand for a NaN: a NaN shows in the sums of exponentials.
template <int G, class With>
__device__ inline float group_reduce(float x, With with) {
  if constexpr (G <= 8) {
    x = with(x, exchanged<0xb1>(x));
    x = with(x, exchanged<0x4e>(x));
    if constexpr (G == 8) x = with(x, exchanged<0x141>(x));
  } else {
    x = with(x, exchanged<0x128>(x));
    x = with(x, exchanged<0x124>(x));
    x = with(x, exchanged<0x122>(x));
    x = with(x, exchanged<0x121>(x));
  }
  if constexpr (G >= 32) x = with(x, __shfl_xor(x, 16));
  if constexpr (G == 64) x = with(x, __shfl_xor(x, 32));
  return x;
}
template <int G>
__device__ inline float group_sum(float x) {
  return group_reduce<G>(x, [](float a, float b) { return a + b; });
}
template <int G>
__device__ inline float group_max(float x) {
  return group_reduce<G>(x, [](float a, float b) { return fmaxf(a, b); });
}

inline bool dtype_known(int d) {
  return d == CUGO_DTYPE_F32 || d == CUGO_DTYPE_F16 || d == CUGO_DTYPE_BF16;
}

// The current device's compute units (256 where the device does not say).
inline int compute_units() {
  thread_local int device = -1, cus = 256;
  int now = 0;
  if (hipGetDevice(&now) != hipSuccess) return 256;
  if (now != device) {
    int count = 0;
    cus = hipDeviceGetAttribute(&count, hipDeviceAttributeMultiprocessorCount, now) ==
                      hipSuccess && count > 0 ? count : 256;
    device = now;
  }
  return cus;
}

}  // namespace learner
}  // namespace cugo_amd

#endif  // CUGO_LEARNER_H_
