// The Remax of a score, a row's sums apart: shared by the attention kernels that keep no scores.
//
// For a score z ~ N(m, v), a = m / sqrt(v), the Remax (remax.py:33-114) needs the moments of
// max(z, 0) and Phi(a). With x = |a|, phi its density and R(x) = (1 - Phi(x)) / phi(x):
//   f = phi (1 - x R),  q = phi ((1 + x^2) R - x) = phi (R - x (1 - x R))
//   a < 0:  mean = sd f,      var = v (q - f^2),                Phi = phi R
//   a >= 0: mean = sd f + m,  var = v (1 - q - 2 x f - f^2),    Phi = 1 - phi R
// (the second line from the first by z = m + ...: no side subtracts near values but R - x(1 - xR),
// which loses x^2 / 2 of R's rounding; 3e-6 of the variance at x = 4, where the weight is 1e-5 of
// its row). R and 1 - x R are polynomials in t = 1 / (1 + x / 4) (gen_tail_fit.py: relative error
// 1.3e-8 and 2.3e-8, in fp32 4e-7 and 7e-7), so the two tails and both signs run without a branch.
#pragma once
#include "tagi_moments.h"

namespace tagi {

constexpr float kRemaxFloor = 1e-6f;  // of means, variances, weights and their sums
constexpr float kVarFloor = 1e-20f;   // of a score's variance

// In: a score's moments. Out: floored moments of max(z, 0) and Phi.
__device__ __forceinline__ void rectify(float m, float v, float& mm, float& vm, float& cdf) {
  v = fmaxf(v, kVarFloor);
  const float rs = fast_rsqrt(v), sd = v * rs, a = m * rs;
  const float x = fminf(fabsf(a), 1e4f);  // its square stays finite
  const float t = fast_rcp(fmaf(0.25f, x, 1.0f));
  float p = 8.162231129e-02f;
  p = fmaf(p, t, -4.702841742e-01f);
  p = fmaf(p, t, 9.322739078e-01f);
  p = fmaf(p, t, -7.467720368e-01f);
  p = fmaf(p, t, 6.768747605e-01f);
  p = fmaf(p, t, 3.456174901e-03f);
  p = fmaf(p, t, 2.822860731e-01f);
  p = fmaf(p, t, 2.434708960e-01f);
  p = fmaf(p, t, 2.503862088e-01f);
  float u = 2.179881536e-01f;
  u = fmaf(u, t, -1.113959958e+00f);
  u = fmaf(u, t, 2.007446407e+00f);
  u = fmaf(u, t, -1.577014472e+00f);
  u = fmaf(u, t, 1.186129971e+00f);
  u = fmaf(u, t, -1.551880686e-01f);
  u = fmaf(u, t, 2.570016636e-01f);
  u = fmaf(u, t, 1.145055705e-01f);
  u = fmaf(u, t, 6.309070943e-02f);
  const float R = p * t, u1 = u * t * t;
  // exp(-x^2 / 2): the exponent's rounding is x^2 2^-25 of the value, as that of x itself
  const float pdf = INV_SQRT_2PI * __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  const float f = pdf * u1, q = pdf * fmaf(-x, u1, R), tail = pdf * R;
  const bool up = a >= 0.0f;
  const float mean = fmaf(sd, f, fmaxf(m, 0.0f));
  const float var = fmaf(-f, f, up ? fmaf(-2.0f * x, f, 1.0f - q) : q);
  cdf = up ? 1.0f - tail : tail;
  mm = fmaxf(mean, kRemaxFloor);
  // where the floor lifts the mean, the variance is taken about the lifted one (as rect_moments)
  vm = fmaxf(fmaf(mean - mm, fmaf(-2.0f, m, mean + mm), v * var), kRemaxFloor);
}

// A row's sums of mm and vm, as the weights use them.
struct RowSums {
  float inv_mt, y, c_mt;
};
__device__ __forceinline__ RowSums row_sums(float mt, float vt) {
  RowSums r;
  r.inv_mt = fast_rcp(fmaxf(mt, kRemaxFloor));
  r.y = fmaxf(vt, kRemaxFloor) * r.inv_mt * r.inv_mt;
  r.c_mt = r.inv_mt * (1.0f + r.y);
  return r;
}

// A score's weight before its row's normalisation, w, and its variance over w^2 (k = num rw^2);
// xw, rw feed the Jacobian (the log-normal stage in closed form, as remax_row).
__device__ __forceinline__ void weigh(float mm, float vm, const RowSums& r, float& w, float& k, float& xw, float& rw) {
  const float rm = fast_rcp(mm), vr = vm * rm, x = vr * rm, ww = vr * r.inv_mt;
  rw = fast_rcp(1.0f + ww);
  w = fmaxf(mm * r.c_mt * rw, kRemaxFloor);
  xw = x - ww;
  k = fmaxf((xw + (r.y - ww)) + fmaf(x, r.y, -(ww * ww)), 0.0f) * rw * rw;
}

// J = cov(weight, z) / v of the normalised weight mua.
__device__ __forceinline__ float remax_jacobian(float v, float mm, float cdf, float mua, float k, float xw, float rw) {
  v = fmaxf(v, kVarFloor);
  const float cov = fmaxf(xw, 0.0f) * rw * mua * mm * fast_rcp(fmaxf(cdf, kRemaxFloor));
  return fminf(__builtin_amdgcn_sqrtf(k * mua * mua * v), cov) * fast_rcp(v);
}

}  // namespace tagi
