// The element types of the sequence-model operators and the fp32 functions that
// several of them need.
#pragma once

#include "common.h"

namespace myelin {

// VEC: elements of a 16-byte load
struct F32 {
  using T = float;
  static constexpr int VEC = 4;
  __device__ static float get(T v) { return v; }
  __device__ static T put(float v) { return v; }
};
struct BF16 {
  using T = __bf16;
  static constexpr int VEC = 8;
  __device__ static float get(T v) { return static_cast<float>(v); }
  __device__ static T put(float v) { return static_cast<__bf16>(v); }
};

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

// e^d to fp32 accuracy: 2^t with t = d log2(e) rounded, and its rounding error
// put back to first order.  d = -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float exp_f32(float d) {
  const float t = d * kLog2e;
  const float e = __builtin_amdgcn_exp2f(t);
  const float r = __builtin_fmaf(d, kLog2e, -t);
  // (past |t| = 2^24 r may be inf - inf; the exponential is 0 there)
  return t > -200.0f ? __builtin_fmaf(e, r * kLn2, e) : e;
}

}  // namespace myelin
