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

// tanh(s * scale) for products s of query and key: the scale is in the coefficients, which saves the product with it.
struct TanhParams {
  float scale;      // softmax scale / cap, 0: no cap
  float near_max;   // largest |s| for which the polynomial is used
  float c[5];       // kTanhC_i * scale^(2i + 1)
};
inline TanhParams tanh_params(float softmax_scale, float cap) {
  TanhParams t = {};
  if (!(cap > 0.f)) return t;
  const double z = static_cast<double>(softmax_scale) / cap, c[5] = {kTanhC0, kTanhC1, kTanhC2, kTanhC3, kTanhC4};
  double power = z;
  for (int i = 0; i < 5; ++i, power *= z * z) t.c[i] = static_cast<float>(c[i] * power);
  t.scale = static_cast<float>(z);
  const double most = kTanhNear / z;
  t.near_max = most < 1e18 ? static_cast<float>(most) : 1e18f;  // (its square stays finite)
  return t;
}

// of two products with |s| <= near_max
__device__ __forceinline__ uint64_t tanh_near2(uint64_t s, const TanhParams& t) {
  const uint64_t u = f2_mul(s, s);
  uint64_t p = f2_fma(u, f2_pack(t.c[4], t.c[4]), f2_pack(t.c[3], t.c[3]));
  p = f2_fma(p, u, f2_pack(t.c[2], t.c[2]));
  p = f2_fma(p, u, f2_pack(t.c[1], t.c[1]));
  p = f2_fma(p, u, f2_pack(t.c[0], t.c[0]));
  return f2_mul(p, s);
}
// tanh of any value
__device__ __forceinline__ float tanh_any(float z) {
  const float u = z * z;
  float p = fmaf(u, kTanhC4, kTanhC3);
  p = fmaf(p, u, kTanhC2);
  p = fmaf(p, u, kTanhC1);
  p = fmaf(p, u, kTanhC0);
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
