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
  __device__ static float to_float(float x) { return x; }
  __device__ static float from_float(float f) { return f; }
};

struct F16 {
  using storage = _Float16;
  __device__ static float to_float(_Float16 x) { return (float)x; }
  __device__ static _Float16 from_float(float f) { return (_Float16)f; }
};

struct BF16 {
  using storage = __bf16;
  __device__ static float to_float(__bf16 x) { return (float)x; }
  // To nearest even in hardware (v_cvt_pk_bf16_f32), as torch rounds.
  __device__ static __bf16 from_float(float f) { return (__bf16)f; }
};

// K consecutive elements, read or written in one access; `Any` at an address that is only an
// element's (global loads and stores take any alignment on gfx950).
template <class S, int K>
struct alignas(sizeof(S) * K) Vec {
  S v[K];
};
template <class S, int K>
struct __attribute__((packed, aligned(sizeof(S)))) Any {
  S v[K];
};

// x from the lane that kCtrl, a rotation within the 16 lanes of a DPP row, names.
template <int kCtrl>
__device__ inline float rotated(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xf, 0xf, false));
}

// The sum and the largest over groups of G lanes (16 or 64), the same value in every lane.
// v_max_f32 takes the other operand for a NaN: a NaN shows in the sums of exponentials.
template <int G>
__device__ inline float group_sum(float x) {
  x += rotated<0x128>(x);
  x += rotated<0x124>(x);
  x += rotated<0x122>(x);
  x += rotated<0x121>(x);
  if constexpr (G == 64) {
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
  }
  return x;
}
template <int G>
__device__ inline float group_max(float x) {
  x = fmaxf(x, rotated<0x128>(x));
  x = fmaxf(x, rotated<0x124>(x));
  x = fmaxf(x, rotated<0x122>(x));
  x = fmaxf(x, rotated<0x121>(x));
  if constexpr (G == 64) {
    x = fmaxf(x, __shfl_xor(x, 16));
    x = fmaxf(x, __shfl_xor(x, 32));
  }
  return x;
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
