// Shaped attention scores: a soft cap, x -> cap tanh(x / cap), and a penalty that grows with the distance of query and key.
//
// tanh. For |z| <= kTanhNear it is z P(z^2) with P of degree 4, fitted here to tanh(z)/z with equal relative errors (Lawson's iteration of
// weighted least squares): 5.7e-7, 6.9e-7 with fp32 arithmetic, so cap tanh is as good as an fp32 score. Elsewhere 1 - 2 / (1 + e^(2z)),
// which is off by some 1e-7 in absolute terms, right at +-infinity and for NaN. The hardware's tanh.approx (relative 2^-11) is no
// substitute: at a score of 20 it moves the weight of a key by 1 %.
#pragma once
#include "common/sm100.cuh"

namespace ra {

constexpr float kTanhNear = 0.75f;
constexpr float kTanhC0 = 0.999999463558197f, kTanhC1 = -0.3332825005054474f, kTanhC2 = 0.13258983194828033f,
                kTanhC3 = -0.050056301057338715f, kTanhC4 = 0.01292963232845068f;

// of two values with |z| <= kTanhNear
__device__ __forceinline__ uint64_t tanh_near2(uint64_t z) {
  const uint64_t u = f2_mul(z, z);
  uint64_t p = f2_fma(u, f2_pack(kTanhC4, kTanhC4), f2_pack(kTanhC3, kTanhC3));
  p = f2_fma(p, u, f2_pack(kTanhC2, kTanhC2));
  p = f2_fma(p, u, f2_pack(kTanhC1, kTanhC1));
  p = f2_fma(p, u, f2_pack(kTanhC0, kTanhC0));
  return f2_mul(p, z);
}
// of any value
__device__ __forceinline__ float tanh_any(float z) {
  const float u = z * z;
  float p = fmaf(u, kTanhC4, kTanhC3);
  p = fmaf(p, u, kTanhC2);
  p = fmaf(p, u, kTanhC1);
  p = fmaf(p, u, kTanhC0);
  const float far = 1.f - __fdividef(2.f, 1.f + exp2_approx(z * 2.885390081777927f));  // 2 log2(e)
  return fabsf(z) <= kTanhNear ? p * z : far;
}

}  // namespace ra
