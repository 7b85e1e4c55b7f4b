// Shaped attention scores: a soft cap, x -> cap tanh(x / cap), and a penalty that grows with the distance of query and key.
//
// tanh. For |z| <= kTanhNear it is z P(z^2) with P of degree 4, fitted here to tanh(z)/z with equal relative errors (Lawson's iteration of
// weighted least squares): 5.7e-7, 7.0e-7 with fp32 arithmetic, so cap tanh is as good as an fp32 score. Degree 3 is as good up to kTanhMid (5.4e-7,
// 6.2e-7) and degree 2 up to kTanhSmall (4.0e-7, 5.0e-7). Elsewhere 1 - 2 / (1 + e^(2z)), which is off by some 1e-7 in absolute terms, right at
// +-infinity and for NaN. The hardware's tanh.approx (relative 2^-11) is no substitute: at a score of 20 it moves the weight of a key by 1 %.
#pragma once
#include "common/sm100.cuh"

namespace ra {

constexpr float kTanhNear = 0.75f, kTanhMid = 0.5f, kTanhSmall = 0.25f;
constexpr double kTanhC[5] = {0.999999463558197, -0.3332825005054474, 0.13258983194828033, -0.050056301057338715, 0.01292963232845068};
constexpr double kTanhM[4] = {0.9999994557609966, -0.33326317852948983, 0.1319029553246415, -0.04440219238268648};
constexpr double kTanhS[3] = {0.9999996043326542, -0.33321908045628074, 0.12841609809441018};

// tanh(s * scale) for products s of query and key: the scale is in the coefficients, which saves the product with it.
struct TanhParams {
  float scale;      // softmax scale / cap, 0: no cap
  float near_max, mid_max, small_max;  // largest |s| for which the polynomials are used
  float c[5];       // kTanhC[i] * scale^(2i + 1)
  float s[3];       // the same of kTanhS
  float m[4];       // the same of kTanhM, times cap * log2(e)
};
inline TanhParams tanh_params(float softmax_scale, float cap) {
  TanhParams t = {};
  if (!(cap > 0.f)) return t;
  const double z = static_cast<double>(softmax_scale) / cap, cap_log2 = cap * 1.4426950408889634;
  double power = z;
  for (int i = 0; i < 5; ++i, power *= z * z) {
    t.c[i] = static_cast<float>(kTanhC[i] * power);
    if (i < 4) t.m[i] = static_cast<float>(kTanhM[i] * power * cap_log2);
    if (i < 3) t.s[i] = static_cast<float>(kTanhS[i] * power);
  }
  t.scale = static_cast<float>(z);
  auto largest = [z](double most) { return most / z < 1e18 ? static_cast<float>(most / z) : 1e18f; };  // (its square stays finite)
  t.near_max = largest(kTanhNear);
  t.mid_max = largest(kTanhMid);
  t.small_max = largest(kTanhSmall);
  return t;
}

// of two products with |s| <= near_max
__device__ __forceinline__ uint64_t tanh_near2(uint64_t s, const float (&c)[5]) {
  const uint64_t u = f2_mul(s, s);
  uint64_t p = f2_fma(u, f2_pack(c[4], c[4]), f2_pack(c[3], c[3]));
  p = f2_fma(p, u, f2_pack(c[2], c[2]));
  p = f2_fma(p, u, f2_pack(c[1], c[1]));
  p = f2_fma(p, u, f2_pack(c[0], c[0]));
  return f2_mul(p, s);
}
// the same with |s| <= small_max
__device__ __forceinline__ uint64_t tanh_small2(uint64_t s, const TanhParams& t) {
  const uint64_t u = f2_mul(s, s);
  uint64_t p = f2_fma(u, f2_pack(t.s[2], t.s[2]), f2_pack(t.s[1], t.s[1]));
  p = f2_fma(p, u, f2_pack(t.s[0], t.s[0]));
  return f2_mul(p, s);
}
// cap log2(e) tanh + plus, of two products with |s| <= mid_max
__device__ __forceinline__ uint64_t capped_mid2(uint64_t s, const TanhParams& t, uint64_t plus) {
  const uint64_t u = f2_mul(s, s);
  uint64_t p = f2_fma(u, f2_pack(t.m[3], t.m[3]), f2_pack(t.m[2], t.m[2]));
  p = f2_fma(p, u, f2_pack(t.m[1], t.m[1]));
  p = f2_fma(p, u, f2_pack(t.m[0], t.m[0]));
  return f2_fma(p, s, plus);
}
// tanh of any value
__device__ __forceinline__ float tanh_any(float z) {
  const float u = z * z;
  constexpr float c0 = kTanhC[0], c1 = kTanhC[1], c2 = kTanhC[2], c3 = kTanhC[3], c4 = kTanhC[4];
  float p = fmaf(u, c4, c3);
  p = fmaf(p, u, c2);
  p = fmaf(p, u, c1);
  p = fmaf(p, u, c0);
  const float far = 1.f - __fdividef(2.f, 1.f + exp2_approx(z * 2.885390081777927f));  // 2 log2(e)
  return fabsf(z) <= kTanhNear ? p * z : far;
}
// `columns` columns of scores in TMEM (a multiple of 8) become their tanh, for tiles with a score out of the polynomial's range: a short
// rolled loop, because unrolled beside the common case it costs every tile (instructions that the caches do not hold). Converged warps.
__device__ __forceinline__ void tanh_in_tmem(uint32_t at, int columns, float scale) {
#pragma unroll 1
  for (int c = 0; c < columns; c += 8) {
    uint32_t s[8];
    tmem_ld_x8(at + c, s);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = __float_as_uint(tanh_any(__uint_as_float(s[e]) * scale));
    tmem_st_x8(at + c, s);
  }
  tmem_st_wait();
}

}  // namespace ra
