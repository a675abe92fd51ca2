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
// 1.3e-8 and 2.3e-8, in fp32 4e-7 and 7e-7), so the two tails and both signs run without a branch:
// the vector ALUs bound the attention kernels, and this is half of their work.
#pragma once
#include "tagi_moments.h"

namespace tagi {

constexpr float kRemaxFloor = 1e-6f;  // of means, variances, weights and their sums
// Added to a score's variance: a stays finite for means up to 1e28, and a variance above 1e-13 does
// not change.
constexpr float kVarFloor = 1e-20f;

// The greater of the two, NaN where x is (fmaxf would give the floor): a mean and a weight that are NaN
// reach the outputs.
__device__ __forceinline__ float floored(float x, float floor) { return __builtin_elementwise_maximum(x, floor); }

struct Rectified {
  float mm, vm;   // moments of max(z, 0), floored
  float cdf, rs;  // Phi(a), 1 / sqrt(v)
};
__device__ __forceinline__ Rectified rectify(float m, float v) {
  Rectified o;
  v += kVarFloor;
  o.rs = fast_rsqrt(v);
  const float sd = v * o.rs, a = m * o.rs, x = fabsf(a);
  const float t = fast_rcp(fmaf(0.25f, x, 1.0f));
  float p = 3.256259095e-02f;  // R / (t sqrt(2 pi))
  p = fmaf(p, t, -1.876162406e-01f);
  p = fmaf(p, t, 3.719234782e-01f);
  p = fmaf(p, t, -2.979189386e-01f);
  p = fmaf(p, t, 2.700339600e-01f);
  p = fmaf(p, t, 1.378814559e-03f);
  p = fmaf(p, t, 1.126158497e-01f);
  p = fmaf(p, t, 9.713083447e-02f);
  p = fmaf(p, t, 9.988964513e-02f);
  float u = 8.696469113e-02f;  // (1 - x R) / (t^2 sqrt(2 pi))
  u = fmaf(u, t, -4.444057261e-01f);
  u = fmaf(u, t, 8.008552477e-01f);
  u = fmaf(u, t, -6.291377500e-01f);
  u = fmaf(u, t, 4.731973958e-01f);
  u = fmaf(u, t, -6.191108207e-02f);
  u = fmaf(u, t, 1.025288298e-01f);
  u = fmaf(u, t, 4.568111342e-02f);
  u = fmaf(u, t, 2.516955149e-02f);
  // exp(-x^2 / 2) t: the exponent's rounding is x^2 2^-25 of the value, as that of x itself
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f) * t, ut = u * t;
  const float f = e * ut, q = e * fmaf(-x, ut, p), tail = e * p;
  const bool up = a >= 0.0f;
  const float mean = fmaf(sd, f, up ? m : 0.0f);
  const float var = fmaf(-f, f, up ? 1.0f - fmaf(2.0f * x, f, q) : q);
  o.cdf = up ? 1.0f - tail : tail;
  o.mm = floored(mean, kRemaxFloor);
  // where the floor lifts the mean by d, the variance is taken about the lifted one: less 2 d (mm -
  // m) and d^2, of which 2 d mm and d^2 are below 2e-6 of the variance's own floor
  o.vm = fmaxf(fmaf(-2.0f * m, mean - o.mm, v * var), kRemaxFloor);
  return o;
}

// A row's sums of mm and vm, as the weights use them.
struct RowSums {
  float inv_mt, vt, c_mt;  // 1 / mt, vt, (1 + vt / mt^2) / mt
};
__device__ __forceinline__ RowSums row_sums(float mt, float vt) {
  RowSums r;
  r.inv_mt = fast_rcp(floored(mt, kRemaxFloor));
  r.vt = fmaxf(vt, kRemaxFloor);
  r.c_mt = fmaf(r.vt * r.inv_mt, r.inv_mt, 1.0f) * r.inv_mt;
  return r;
}

// A score's weight before its row's normalisation and the weight's relative variance: the
// log-normal stage in closed form (remax_row) with x = vm / mm^2 and w = vm / (mm mt) multiplied out,
//   weight = mm c_mt / (1 + w) = mm^2 c_mt / d,  d = mm + s,  s = vm / mt
//   k = [(1 + x)(1 + vt / mt^2) - (1 + w)^2] / (1 + w)^2 = [vm u^2 + (vt - vm) (p^2 + s / mt)] / d^2,
//       p = mm / mt, u = 1 - p
// (what cancels is taken out by hand: a row of one key has u = 0, vt = vm and no variance, and with
// few keys a difference of the products would lose what their roundings are of it).
struct Weight {
  float w, k, rd, u;  // rd = 1 / d
};
__device__ __forceinline__ Weight weigh(const Rectified& z, const RowSums& r) {
  Weight o;
  const float s = z.vm * r.inv_mt, d = z.mm + s;
  o.rd = fast_rcp(d);
  o.w = floored(z.mm * o.rd * z.mm * r.c_mt, kRemaxFloor);
  const float p = z.mm * r.inv_mt;
  o.u = 1.0f - p;
  const float num = fmaf(r.vt - z.vm, fmaf(p, p, s * r.inv_mt), z.vm * (o.u * o.u));
  o.k = fmaxf(num, 0.0f) * o.rd * o.rd;
  return o;
}

// J = cov(weight, z) / v of the normalised weight a: a times the lesser of sqrt(k / v) and
// (x - w) / (1 + w) mm / (Phi v), (x - w) / (1 + w) mm = vm (1 - mm / mt) / d.
__device__ __forceinline__ float remax_jacobian(const Rectified& z, const Weight& w, float a) {
  const float cov = fmaxf(w.u, 0.0f) * (z.vm * w.rd) * fast_rcp(fmaxf(z.cdf, kRemaxFloor));
  return a * z.rs * fminf(__builtin_amdgcn_sqrtf(w.k), cov * z.rs);
}

}  // namespace tagi
