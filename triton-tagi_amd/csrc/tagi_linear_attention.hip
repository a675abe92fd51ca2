// Linear attention with a decay for each head, on Gaussian moments.
//
// A head carries a D x D state of independent Gaussians (means M, variances P). With g its
// decay and c the scale, every token advances it and reads it (the product moments of
// independent Gaussians, exactly):
//   M_t = g M_{t-1} + k v^T            P_t = g^2 P_{t-1} + Sk (v^2 + Sv)^T + (k^2) Sv^T
//   mo  = c M_t^T q                    So  = c^2 [P_t^T (Sq + q^2) + (M_t.M_t)^T Sq]
// Backward, each product's other operand held at its mean (as the attention layer does),
// with d = c dmo, e = c^2 dSo:
//   dq = M_t d,  dSq = (M_t.M_t) e
//   G_t = g G_{t+1} + q d^T,  N_t = g^2 N_{t+1} + (q^2) e^T      (last token first)
//   dk = G_t v,  dSk = N_t (v^2);   dv = G_t^T k,  dSv = N_t^T (k^2)
//
// The squared state (M_t.M_t) is needed at every token and has no form as a matrix product
// over a chunk, so the state advances token by token on the vector ALUs, and that is the
// bound: 7 operations per state element and token forward. Every pass is one scan,
//   X_t = g X_{t-1} + u_t w_t^T (one or two such states),  y_t[o] = sum_i r_t[i] f(X_t[i][o]),
// whose columns o are independent: a wavefront keeps 32 columns of the state in registers
// (8 lane groups over i, 8 over o, a lane holding DI x EO elements), reads the token's
// vectors from LDS and adds its 8 partial sums over i in three exchanges that halve the
// values each lane keeps.
//
// Decay without a multiplication per token: inside a group of 8 tokens the state is kept
// divided by g^j (token j), the powers go into the token's vectors when they are staged,
// and the state is multiplied by g^8 (as a two-part float: its rounding would repeat every
// group) between groups. |g| < 0.05 would overflow the powers and decays token by token.
#include "tagi_common.h"

namespace tagi {
namespace {

constexpr int kTok = 8;          // tokens per stage, and per decay group
constexpr float kGroupMin = 0.05f;
constexpr int kMaxHeadDim = 128;

enum Mode { FWD = 0, DQ = 1, DK = 2, DV = 3 };
// vectors staged per token, over i and over o
constexpr int n_ivec(int m) { return m == FWD ? 6 : (m == DQ ? 3 : 4); }
constexpr int n_ovec(int m) { return m == FWD ? 3 : (m == DQ ? 1 : 2); }

struct Args {
  // DQ/DK/DV read the means and the deltas (dm, dS) only
  const float *mq, *Sq, *mk, *Sk, *mv, *Sv, *dm, *dS;
  tagi_heads lq, lk, lv, ld, lo;  // strides; lo of the outputs
  float *om, *oS;
  const float* decay;
  const void* lengths;
  int len_bytes;
  int64_t B, T;
  int H, D;
  float c, c2;
  int64_t L;     // tokens per chunk, a multiple of kTok
  int64_t nch;
  const float *pre_m, *pre_S;  // state before each chunk (nch > 1), [bh][chunk][D][D]
  int pre_t;                   // pre is stored [o][i]
  const float *init_m, *init_S;  // state before the first token, or null
  float *end_m, *end_S;          // state after the last token, or null
  float *sum_m, *sum_S;          // SUM kernels: each chunk's own contribution, [bh][chunk][i][o]
};

__device__ __forceinline__ int64_t seq_len(const Args& a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.len_bytes == 8 ? static_cast<const int64_t*>(a.lengths)[b]
                                     : (int64_t)static_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// x^n in float64, n >= 0
__device__ __forceinline__ double ipow(double x, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1, x *= x)
    if (n & 1) r *= x;
  return r;
}

struct Two {
  float hi, lo;
};
__device__ __forceinline__ Two two(double x) {
  Two t;
  t.hi = (float)x;
  t.lo = (float)(x - (double)t.hi);
  if (!(fabsf(t.hi) < 3.0e38f)) t.lo = 0.f;
  return t;
}
__device__ __forceinline__ float scaled(const Two& t, float x) { return fmaf(t.hi, x, t.lo * x); }

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kXor7 = 0x141;  // quad_perm, quad_perm, row_half_mirror

// Sums over the 8 lanes of a group (lane & 7) of EO means and EO variances per lane. Lanes
// with bit 2 set end with variances, the others with means; of the EO values the lane's
// bit 0 (and, with four, bit 1) says which.
template <int EO>
__device__ __forceinline__ float group_sums(const float* pm, const float* ps, int lane) {
  float r[EO];
  const bool b2 = lane & 4, b0 = lane & 1, b1 = lane & 2;
#pragma unroll
  for (int e = 0; e < EO; ++e) {
    const float keep = b2 ? ps[e] : pm[e], give = b2 ? pm[e] : ps[e];
    r[e] = keep + dpp<kXor7>(give);
  }
  float h[EO / 2];
#pragma unroll
  for (int e = 0; e < EO / 2; ++e) {
    const float keep = b0 ? r[EO / 2 + e] : r[e], give = b0 ? r[e] : r[EO / 2 + e];
    h[e] = keep + dpp<kXor1>(give);
  }
  if constexpr (EO == 4) {
    const float keep = b1 ? h[1] : h[0], give = b1 ? h[0] : h[1];
    return keep + dpp<kXor2>(give);
  } else {
    return h[0] + dpp<kXor2>(h[0]);
  }
}

// Four consecutive values of a token's head row (zeros past D).
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int c, int D) {
  if constexpr (VEC) return *reinterpret_cast<const float4*>(p + c);
  float4 r = make_float4(p[c], 0.f, 0.f, 0.f);
  if (c + 1 < D) r.y = p[c + 1];
  if (c + 2 < D) r.z = p[c + 2];
  if (c + 3 < D) r.w = p[c + 3];
  return r;
}

__device__ __forceinline__ float4 mul4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) {
  return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w);
}
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// The scan of one (sequence, head, chunk) per block. SUM: no outputs, the chunk's own
// contribution to the state is written instead.
template <int MODE, int DI, int EO, bool VEC, bool SUM>
__global__ void __launch_bounds__(DI <= 4 ? 64 : DI * 16) scan_kernel(Args a) {
  constexpr int IP = 8 * DI;                     // padded head dimension
  constexpr int NT = DI <= 4 ? 64 : DI * 16;     // threads: a wave per 8 * EO columns
  constexpr bool REV = MODE >= DK, TWO_STATES = MODE != DQ;
  constexpr int NI = SUM ? (MODE == FWD ? 3 : (MODE == DQ ? 1 : 2)) : n_ivec(MODE), NO = n_ovec(MODE);
  constexpr int C4 = IP / 4;                     // float4 chunks of a row
  __shared__ float4 iv[NI][kTok][C4];
  __shared__ float4 ov[NO][kTok][C4];

  const int64_t bid = blockIdx.x, ch = bid % a.nch, bh = bid / a.nch, b = bh / a.H;
  const int h = (int)(bh % a.H), D = a.D;
  const int64_t n = seq_len(a, b), t0 = ch * a.L, t1 = min(a.T, t0 + a.L), live = min(n, t1);
  const int cnt = live > t0 ? (int)(live - t0) : 0;  // live tokens of the chunk
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ig = lane & 7, og = lane >> 3;

  const float g = a.decay[h];
  const bool grouped = fabsf(g) >= kGroupMin;
  const int per = grouped ? kTok : 1;  // tokens between decays
  const double gd = (double)g;
  const Two gm = two(ipow(gd, per)), gS = two(ipow(gd, 2 * per));  // between groups

  // this thread's part of a stage: token st, values 4 sc .. 4 sc + 3
  const int st = tid / C4, sc = tid % C4;
  const bool stager = st < kTok, inside = 4 * sc < D;
  float up = 1.f, up2 = 1.f, dn = 1.f, dn2 = 1.f;  // g^-j, g^-2j, g^j, g^2j
  if (grouped && stager) {
    const double p = ipow(gd, st);
    dn = (float)p, dn2 = (float)(p * p), up = (float)(1.0 / p), up2 = (float)(1.0 / (p * p));
  }
  const float4 z4 = make_float4(0.f, 0.f, 0.f, 0.f);

  const int64_t qb = b * a.lq.sb + h * a.lq.sh, kb = b * a.lk.sb + h * a.lk.sh, vb = b * a.lv.sb + h * a.lv.sh,
                db = b * a.ld.sb + h * a.ld.sh, ob = b * a.lo.sb + h * a.lo.sh;

  auto tok = [&](int r) -> int64_t { return REV ? live - 1 - r : t0 + r; };  // r-th token of the scan

  float4 x0 = z4, x1 = z4, x2 = z4, x3 = z4, x4 = z4, x5 = z4;
  auto fetch = [&](int s0) {
    const int r = s0 + st;
    if (stager && inside && r < cnt) {
      const int64_t t = tok(r);
      const int c = 4 * sc;
      if constexpr (MODE == FWD) {
        x2 = load4<VEC>(a.mk + kb + t * a.lk.st, c, D), x3 = load4<VEC>(a.Sk + kb + t * a.lk.st, c, D);
        x4 = load4<VEC>(a.mv + vb + t * a.lv.st, c, D), x5 = load4<VEC>(a.Sv + vb + t * a.lv.st, c, D);
        if constexpr (!SUM)
          x0 = load4<VEC>(a.mq + qb + t * a.lq.st, c, D), x1 = load4<VEC>(a.Sq + qb + t * a.lq.st, c, D);
      } else if constexpr (MODE == DQ) {
        x0 = load4<VEC>(a.mv + vb + t * a.lv.st, c, D), x1 = load4<VEC>(a.mk + kb + t * a.lk.st, c, D);
        if constexpr (!SUM)
          x2 = load4<VEC>(a.dm + db + t * a.ld.st, c, D), x3 = load4<VEC>(a.dS + db + t * a.ld.st, c, D);
      } else {
        x0 = load4<VEC>(a.mq + qb + t * a.lq.st, c, D);
        x1 = load4<VEC>(a.dm + db + t * a.ld.st, c, D), x2 = load4<VEC>(a.dS + db + t * a.ld.st, c, D);
        if constexpr (!SUM)
          x3 = MODE == DK ? load4<VEC>(a.mv + vb + t * a.lv.st, c, D) : load4<VEC>(a.mk + kb + t * a.lk.st, c, D);
      }
    } else {
      x0 = x1 = x2 = x3 = x4 = x5 = z4;  // nothing to add, and a dead token's output is zero
    }
  };
  auto stage = [&]() {
    if (!stager) return;
    if constexpr (MODE == FWD) {
      iv[0][st][sc] = mul4(x2, up);
      iv[1][st][sc] = mul4(x3, up2);
      iv[2][st][sc] = mul4(mul4(x2, x2), up2);
      ov[0][st][sc] = x4;
      ov[1][st][sc] = add4(mul4(x4, x4), x5);
      ov[2][st][sc] = x5;
      if constexpr (!SUM) {
        iv[3][st][sc] = mul4(x0, a.c * dn);
        iv[4][st][sc] = mul4(add4(x1, mul4(x0, x0)), a.c2 * dn2);
        iv[5][st][sc] = mul4(x1, a.c2 * dn2);
      }
    } else if constexpr (MODE == DQ) {
      iv[0][st][sc] = mul4(x0, up);
      ov[0][st][sc] = x1;
      if constexpr (!SUM) {
        iv[1][st][sc] = mul4(x2, a.c * dn);
        iv[2][st][sc] = mul4(x3, a.c2 * dn2);
      }
    } else {
      const float4 d = mul4(x1, a.c), e = mul4(x2, a.c2), q2 = mul4(x0, x0);
      if constexpr (MODE == DK) {
        iv[0][st][sc] = mul4(d, up), iv[1][st][sc] = mul4(e, up2);
        ov[0][st][sc] = x0, ov[1][st][sc] = q2;
      } else {
        iv[0][st][sc] = mul4(x0, up), iv[1][st][sc] = mul4(q2, up2);
        ov[0][st][sc] = d, ov[1][st][sc] = e;
      }
      if constexpr (!SUM) iv[2][st][sc] = mul4(x3, dn), iv[3][st][sc] = mul4(mul4(x3, x3), dn2);
    }
  };

  // state element (i, o): i = 32 (k / 4) + 4 ig + k % 4 (EO == 4), the o of this wave
  auto idx_i = [&](int k) { return EO == 4 ? 32 * (k >> 2) + 4 * ig + (k & 3) : DI * ig + k; };
  auto idx_o = [&](int e) { return 8 * EO * wave + EO * og + e; };
  float X[DI][EO], Y[TWO_STATES ? DI : 1][EO];
#pragma unroll
  for (int k = 0; k < DI; ++k)
#pragma unroll
    for (int e = 0; e < EO; ++e) {
      X[k][e] = 0.f;
      if constexpr (TWO_STATES) Y[k][e] = 0.f;
    }
  const bool from_pre = !SUM && a.nch > 1;
  const float* sm = from_pre ? a.pre_m : (SUM ? nullptr : a.init_m);
  const float* sS = from_pre ? a.pre_S : (SUM ? nullptr : a.init_S);
  if (sm) {
    const int64_t base = (from_pre ? bh * a.nch + ch : bh) * (int64_t)D * D;
    const bool tr = from_pre && a.pre_t;
#pragma unroll
    for (int k = 0; k < DI; ++k)
#pragma unroll
      for (int e = 0; e < EO; ++e) {
        const int i = idx_i(k), o = idx_o(e);
        if (i < D && o < D) {
          const int64_t at = base + (tr ? (int64_t)o * D + i : (int64_t)i * D + o);
          X[k][e] = sm[at];
          if constexpr (TWO_STATES) Y[k][e] = sS[at];
        }
      }
  }

  fetch(0);
  for (int s0 = 0; s0 < cnt; s0 += kTok) {
    __syncthreads();
    stage();
    __syncthreads();
    fetch(s0 + kTok);
    const int m = min(kTok, cnt - s0);
    for (int j = 0; j < m; ++j) {
      if (!grouped || j == 0) {  // the state before the token, decayed
#pragma unroll
        for (int k = 0; k < DI; ++k)
#pragma unroll
          for (int e = 0; e < EO; ++e) {
            // the first group starts from the true state: one decay, not a group's
            X[k][e] = (s0 == 0 && j == 0) ? g * X[k][e] : scaled(gm, X[k][e]);
            if constexpr (TWO_STATES) Y[k][e] = (s0 == 0 && j == 0) ? g * (g * Y[k][e]) : scaled(gS, Y[k][e]);
          }
      }
      float w[NO][EO];
#pragma unroll
      for (int v = 0; v < NO; ++v) {
        const float* p = reinterpret_cast<const float*>(&ov[v][j][0]) + 8 * EO * wave + EO * og;
#pragma unroll
        for (int e = 0; e < EO; ++e) w[v][e] = p[e];
      }
      float pm[EO] = {}, ps[EO] = {};
#pragma unroll
      for (int k0 = 0; k0 < DI; k0 += (EO == 4 ? 4 : DI)) {
        constexpr int KN = EO == 4 ? 4 : DI;
        float u[NI][KN];
#pragma unroll
        for (int v = 0; v < NI; ++v) {
          const float* p = reinterpret_cast<const float*>(&iv[v][j][0]) + idx_i(k0);
#pragma unroll
          for (int k = 0; k < KN; ++k) u[v][k] = p[k];
        }
#pragma unroll
        for (int k = 0; k < KN; ++k)
#pragma unroll
          for (int e = 0; e < EO; ++e) {
            float& x = X[k0 + k][e];
            x = fmaf(u[0][k], w[0][e], x);
            if constexpr (MODE == FWD) {
              float& y = Y[k0 + k][e];
              y = fmaf(u[1][k], w[1][e], y);
              y = fmaf(u[2][k], w[2][e], y);
              if constexpr (!SUM) {
                pm[e] = fmaf(u[3][k], x, pm[e]);
                ps[e] = fmaf(u[4][k], y, ps[e]);
                ps[e] = fmaf(u[5][k], x * x, ps[e]);
              }
            } else if constexpr (MODE == DQ) {
              if constexpr (!SUM) {
                pm[e] = fmaf(u[1][k], x, pm[e]);
                ps[e] = fmaf(u[2][k], x * x, ps[e]);
              }
            } else {
              float& y = Y[k0 + k][e];
              y = fmaf(u[1][k], w[1][e], y);
              if constexpr (!SUM) {
                pm[e] = fmaf(u[2][k], x, pm[e]);
                ps[e] = fmaf(u[3][k], y, ps[e]);
              }
            }
          }
      }
      if constexpr (!SUM) {
        const float r = group_sums<EO>(pm, ps, lane);
        const int o = idx_o(0) + (EO == 4 ? 2 * (lane & 1) + ((lane >> 1) & 1) : (lane & 1));
        const bool mine = EO == 4 || (lane & 2) == 0;
        if (mine && o < D) ((lane & 4) ? a.oS : a.om)[ob + tok(s0 + j) * a.lo.st + o] = r;
      }
    }
  }

  // back to the true state: the last token's power
  const int last = (grouped && cnt > 0) ? (cnt - 1) % kTok : 0;
  const Two fm = two(ipow(gd, last)), fS = two(ipow(gd, 2 * last));
  float* em = SUM ? a.sum_m : a.end_m;
  float* eS = SUM ? a.sum_S : a.end_S;
  // the chunk of the last live token (the first one without any) holds the final state
  const bool writes = SUM || (em && ch == (n > 0 ? (n - 1) / a.L : 0));
  if (writes) {
    const int64_t base = (SUM ? bh * a.nch + ch : bh) * (int64_t)D * D;
#pragma unroll
    for (int k = 0; k < DI; ++k)
#pragma unroll
      for (int e = 0; e < EO; ++e) {
        const int i = idx_i(k), o = idx_o(e);
        if (i < D && o < D) {
          em[base + (int64_t)i * D + o] = scaled(fm, X[k][e]);
          if constexpr (TWO_STATES) eS[base + (int64_t)i * D + o] = scaled(fS, Y[k][e]);
        }
      }
  }
  if constexpr (!SUM) {  // tokens past the sequence's end
    const int64_t dead0 = max(t0, min(t1, n));
    for (int64_t q = tid; q < (t1 - dead0) * D; q += NT) {
      const int64_t at = ob + (dead0 + q / D) * a.lo.st + q % D;
      a.om[at] = 0.f;
      a.oS[at] = 0.f;
    }
  }
}

// Chunk contributions to the states before each chunk, in place: run = g^n run + sum (n the
// chunk's live tokens; fewer than L only where every later chunk in scan order is empty, or,
// last token first, where run is still zero).
template <bool REV>
__global__ void __launch_bounds__(256) carry_kernel(Args a, int two_states) {
  const int64_t DD = (int64_t)a.D * a.D, per = (DD + 255) / 256, bh = blockIdx.x / per, b = bh / a.H;
  const int64_t el = (blockIdx.x % per) * 256 + threadIdx.x;
  if (el >= DD) return;
  const int64_t n = seq_len(a, b);
  const double gL = ipow((double)a.decay[bh % a.H], a.L);
  for (int s = 0; s < (two_states ? 2 : 1); ++s) {
    const Two f = two(s ? gL * gL : gL);
    float* x = (s ? a.sum_S : a.sum_m) + bh * a.nch * DD + el;
    const float* init = s ? a.init_S : a.init_m;
    float run = init ? init[bh * DD + el] : 0.f;
    for (int64_t k = 0; k < a.nch; ++k) {
      const int64_t ch = REV ? a.nch - 1 - k : k;
      const bool live = ch * a.L < n, more = k + 1 < a.nch;
      const float own = live && more ? x[ch * DD] : 0.f;  // the last chunk's is not formed
      x[ch * DD] = run;
      if (live) run = scaled(f, run) + own;
    }
  }
}

// One token of every sequence: the state is read, advanced and written once.
template <bool VEC>
__global__ void __launch_bounds__(256) step_kernel(Args a, const uint8_t* __restrict__ active, float* __restrict__ M,
                                                   float* __restrict__ P) {
  __shared__ float vec[6][kMaxHeadDim];
  __shared__ float red[2][32][32];
  const int D = a.D, tid = threadIdx.x;
  const int64_t bh = blockIdx.x, b = bh / a.H;
  const int h = (int)(bh % a.H), c0 = (int)blockIdx.y * 32;
  const bool on = !active || active[b];
  const int64_t qb = b * a.lq.sb + h * a.lq.sh, kb = b * a.lk.sb + h * a.lk.sh, vb = b * a.lv.sb + h * a.lv.sh,
                ob = b * a.lo.sb + h * a.lo.sh;
  if (!on) {
    if (tid < 32 && c0 + tid < D) a.om[ob + c0 + tid] = 0.f, a.oS[ob + c0 + tid] = 0.f;
    return;
  }
  for (int i = tid; i < D; i += 256) {
    const float q = a.mq[qb + i], Sq = a.Sq[qb + i], k = a.mk[kb + i];
    vec[0][i] = a.c * q;
    vec[1][i] = a.c2 * (Sq + q * q);
    vec[2][i] = a.c2 * Sq;
    vec[3][i] = k;
    vec[4][i] = a.Sk[kb + i];
    vec[5][i] = k * k;
  }
  const float g = a.decay[h];
  const int cq = tid & 7, rg = tid >> 3, col = c0 + 4 * cq;
  float v[4], v2[4], Sv[4], pm[4] = {}, ps[4] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool ok = col + e < D;
    v[e] = ok ? a.mv[vb + col + e] : 0.f;
    Sv[e] = ok ? a.Sv[vb + col + e] : 0.f;
    v2[e] = v[e] * v[e] + Sv[e];
  }
  __syncthreads();
  for (int i = rg; i < D; i += 32) {
    const int64_t at = (bh * D + i) * D + col;
    float x[4], y[4];
    if constexpr (VEC) {
      float4 xm = make_float4(0.f, 0.f, 0.f, 0.f), xS = xm;
      if (col < D) xm = *reinterpret_cast<const float4*>(M + at), xS = *reinterpret_cast<const float4*>(P + at);
      x[0] = xm.x, x[1] = xm.y, x[2] = xm.z, x[3] = xm.w, y[0] = xS.x, y[1] = xS.y, y[2] = xS.z, y[3] = xS.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = col + e < D ? M[at + e] : 0.f;
        y[e] = col + e < D ? P[at + e] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = fmaf(vec[3][i], v[e], g * x[e]);
      y[e] = fmaf(vec[5][i], Sv[e], fmaf(vec[4][i], v2[e], g * (g * y[e])));
      pm[e] = fmaf(vec[0][i], x[e], pm[e]);
      ps[e] = fmaf(vec[1][i], y[e], fmaf(vec[2][i], x[e] * x[e], ps[e]));
    }
    if constexpr (VEC) {
      if (col < D) {
        *reinterpret_cast<float4*>(M + at) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(P + at) = make_float4(y[0], y[1], y[2], y[3]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < D) M[at + e] = x[e], P[at + e] = y[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[0][rg][4 * cq + e] = pm[e], red[1][rg][4 * cq + e] = ps[e];
  __syncthreads();
  if (tid < 64) {
    const int w = tid >> 5, cc = tid & 31;
    float s = 0.f;
    for (int r = 0; r < 32; ++r) s += red[w][r][cc];
    if (c0 + cc < D) (w ? a.oS : a.om)[ob + c0 + cc] = s;
  }
}

inline bool al16a(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline bool al4(const tagi_heads& s) { return s.sb % 4 == 0 && s.st % 4 == 0 && s.sh % 4 == 0; }

// Tokens per chunk. One chunk is one pass over the data, but a wavefront per (sequence, head,
// 32 columns) leaves the GPU's 1024 SIMDs idle where these are few; chunks cost a pass that
// sums each one's contribution and 16 bytes of state traffic an element. Two wavefronts for
// each SIMD, chunks of 32 tokens at least. One prompt of 32768 tokens, 8 heads of 64 (us):
// one chunk 22514, 1024 wavefronts 686, 2048 468, 4096 630.
constexpr int64_t kWaves = 2048, kMinChunk = 32;
int64_t chunk_len(int64_t heads, int64_t T, int64_t D) {
  const int64_t waves = heads * cdiv(D, 32);
  int64_t nch = cdiv(kWaves, waves);
  if (nch > cdiv(T, kMinChunk)) nch = cdiv(T, kMinChunk);
  if (nch < 1) nch = 1;
  return cdiv(cdiv(T > 0 ? T : 1, nch), kTok) * kTok;
}

struct Chunks {
  int64_t L, nch;
};
Chunks chunks(int64_t B, int64_t T, int64_t H, int64_t D) {
  Chunks c;
  c.L = chunk_len(B * H, T, D);
  c.nch = T > 0 ? cdiv(T, c.L) : 1;
  return c;
}

template <int MODE, bool SUM, bool VEC>
void launch_scan_v(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * a.H * a.nch));
  if (a.D <= 16)
    hipLaunchKernelGGL((scan_kernel<MODE, 2, 2, VEC, SUM>), grid, dim3(64), 0, s, a);
  else if (a.D <= 32)
    hipLaunchKernelGGL((scan_kernel<MODE, 4, 4, VEC, SUM>), grid, dim3(64), 0, s, a);
  else if (a.D <= 64)
    hipLaunchKernelGGL((scan_kernel<MODE, 8, 4, VEC, SUM>), grid, dim3(128), 0, s, a);
  else if (a.D <= 96)
    hipLaunchKernelGGL((scan_kernel<MODE, 12, 4, VEC, SUM>), grid, dim3(192), 0, s, a);
  else
    hipLaunchKernelGGL((scan_kernel<MODE, 16, 4, VEC, SUM>), grid, dim3(256), 0, s, a);
}
template <int MODE, bool SUM>
void launch_scan(const Args& a, bool vec, hipStream_t s) {
  vec ? launch_scan_v<MODE, SUM, true>(a, s) : launch_scan_v<MODE, SUM, false>(a, s);
}
template <bool REV>
void launch_carry(const Args& a, bool two_states, hipStream_t s) {
  const int64_t DD = (int64_t)a.D * a.D;
  hipLaunchKernelGGL(carry_kernel<REV>, dim3((unsigned)(cdiv(DD, 256) * a.B * a.H)), dim3(256), 0, s, a,
                     (int)two_states);
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t H, int64_t D) {
  TAGI_REQUIRE(B >= 0 && T >= 0 && H > 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(B < (1ll << 24) && H < (1ll << 24) && B * H < (1ll << 24) && T < (1ll << 31), "%s: too large", what);
  if (D > kMaxHeadDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxHeadDim);
  return TAGI_OK;
}

int64_t state_floats(int64_t B, int64_t H, int64_t D, int64_t nch) { return (B * H * nch * D * D + 3) / 4 * 4; }

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_linear_attention_fwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || D <= 0) return 0;
  const Chunks c = chunks(B, T, H, D);
  return c.nch > 1 ? 2 * state_floats(B, H, D, c.nch) * 4 : 0;
}

extern "C" int64_t tagi_linear_attention_bwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || D <= 0) return 0;
  const Chunks c = chunks(B, T, H, D);
  return c.nch > 1 ? 3 * state_floats(B, H, D, c.nch) * 4 : 0;
}

extern "C" int tagi_linear_attention_fwd(const float* mq, const float* Sq, const float* mk, const float* Sk,
                                         const float* mv, const float* Sv, const tagi_heads* lq, const tagi_heads* lk,
                                         const tagi_heads* lv, const float* decay, const void* lengths, int len_bytes,
                                         const float* init_m, const float* init_S, float* mo, float* So,
                                         const tagi_heads* lo, float* end_m, float* end_S, int64_t B, int64_t T,
                                         int64_t H, int64_t D, double scale, void* ws, int64_t ws_bytes,
                                         tagi_stream_t stream) {
  const char* what = "tagi_linear_attention_fwd";
  if (int rc = check_sizes(what, B, T, H, D)) return rc;
  if (B == 0) return TAGI_OK;
  TAGI_REQUIRE(lq && lk && lv && lo && decay, "%s: null pointer", what);
  TAGI_REQUIRE(T == 0 || (mq && Sq && mk && Sk && mv && Sv && mo && So), "%s: null pointer", what);
  TAGI_REQUIRE((init_m == nullptr) == (init_S == nullptr) && (end_m == nullptr) == (end_S == nullptr),
               "%s: a state is means and variances together", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  const Chunks c = chunks(B, T, H, D);
  TAGI_REQUIRE(B * H * c.nch < (1ll << 31), "%s: too large", what);
  TAGI_REQUIRE(c.nch == 1 || (ws && ws_bytes >= tagi_linear_attention_fwd_ws_bytes(B, T, H, D)),
               "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 15.0 * B * T * H * D * D, 32.0 * B * T * H * D);
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv;
  a.lq = *lq, a.lk = *lk, a.lv = *lv, a.lo = *lo;
  a.om = mo, a.oS = So, a.decay = decay, a.lengths = lengths, a.len_bytes = len_bytes;
  a.B = B, a.T = T, a.H = (int)H, a.D = (int)D, a.c = (float)scale, a.c2 = (float)(scale * scale);
  a.L = c.L, a.nch = c.nch, a.init_m = init_m, a.init_S = init_S, a.end_m = end_m, a.end_S = end_S;
  const bool vec = D % 4 == 0 && al4(*lq) && al4(*lk) && al4(*lv) && al16a(mq) && al16a(Sq) && al16a(mk) && al16a(Sk) &&
                   al16a(mv) && al16a(Sv);
  if (c.nch > 1) {
    a.sum_m = static_cast<float*>(ws);
    a.sum_S = a.sum_m + state_floats(B, H, D, c.nch);
    launch_scan<FWD, true>(a, vec, s);
    launch_carry<false>(a, true, s);
    a.pre_m = a.sum_m, a.pre_S = a.sum_S, a.pre_t = 0;
  }
  launch_scan<FWD, false>(a, vec, s);
  return check_launch(what);
}

extern "C" int tagi_linear_attention_bwd(const float* mq, const float* mk, const float* mv, const tagi_heads* lq,
                                         const tagi_heads* lk, const tagi_heads* lv, const float* dmo,
                                         const float* dSo, const tagi_heads* ld, const float* decay,
                                         const void* lengths, int len_bytes, float* dmq, float* dSq, float* dmk,
                                         float* dSk, float* dmv, float* dSv, const tagi_heads* lo, int64_t B,
                                         int64_t T, int64_t H, int64_t D, double scale, void* ws, int64_t ws_bytes,
                                         tagi_stream_t stream) {
  const char* what = "tagi_linear_attention_bwd";
  if (int rc = check_sizes(what, B, T, H, D)) return rc;
  if (B == 0 || T == 0) return TAGI_OK;
  TAGI_REQUIRE(lq && lk && lv && ld && lo && decay && mq && mk && mv && dmo && dSo && dmq && dSq && dmk && dSk && dmv &&
                   dSv, "%s: null pointer", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  const Chunks c = chunks(B, T, H, D);
  TAGI_REQUIRE(B * H * c.nch < (1ll << 31), "%s: too large", what);
  TAGI_REQUIRE(c.nch == 1 || (ws && ws_bytes >= tagi_linear_attention_bwd_ws_bytes(B, T, H, D)),
               "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 22.0 * B * T * H * D * D, 44.0 * B * T * H * D);
  Args a{};
  a.mq = mq, a.mk = mk, a.mv = mv, a.dm = dmo, a.dS = dSo;
  a.lq = *lq, a.lk = *lk, a.lv = *lv, a.ld = *ld, a.lo = *lo;
  a.decay = decay, a.lengths = lengths, a.len_bytes = len_bytes;
  a.B = B, a.T = T, a.H = (int)H, a.D = (int)D, a.c = (float)scale, a.c2 = (float)(scale * scale);
  a.L = c.L, a.nch = c.nch;
  const bool vec = D % 4 == 0 && al4(*lq) && al4(*lk) && al4(*lv) && al4(*ld) && al16a(mq) && al16a(mk) && al16a(mv) &&
                   al16a(dmo) && al16a(dSo);
  float *wM = nullptr, *wG = nullptr, *wN = nullptr;
  if (c.nch > 1) {
    const int64_t n = state_floats(B, H, D, c.nch);
    wM = static_cast<float*>(ws), wG = wM + n, wN = wG + n;
    a.sum_m = wM;
    launch_scan<DQ, true>(a, vec, s);
    launch_carry<false>(a, false, s);
    a.sum_m = wG, a.sum_S = wN;
    launch_scan<DV, true>(a, vec, s);
    launch_carry<true>(a, true, s);
  }
  a.pre_m = wM, a.pre_t = 0, a.om = dmq, a.oS = dSq;  // the transposed state, as DQ's own sums left it
  launch_scan<DQ, false>(a, vec, s);
  a.pre_m = wG, a.pre_S = wN, a.pre_t = 1, a.om = dmk, a.oS = dSk;
  launch_scan<DK, false>(a, vec, s);
  a.pre_t = 0, a.om = dmv, a.oS = dSv;
  launch_scan<DV, false>(a, vec, s);
  return check_launch(what);
}

extern "C" int tagi_linear_attention_step(const float* mq, const float* Sq, const float* mk, const float* Sk,
                                          const float* mv, const float* Sv, const tagi_heads* lq,
                                          const tagi_heads* lk, const tagi_heads* lv, const float* decay,
                                          const uint8_t* active, float* state_m, float* state_S, float* mo, float* So,
                                          const tagi_heads* lo, int64_t B, int64_t H, int64_t D, double scale,
                                          tagi_stream_t stream) {
  const char* what = "tagi_linear_attention_step";
  if (int rc = check_sizes(what, B, 1, H, D)) return rc;
  if (B == 0) return TAGI_OK;
  TAGI_REQUIRE(lq && lk && lv && lo && decay && mq && Sq && mk && Sk && mv && Sv && state_m && state_S && mo && So,
               "%s: null pointer", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 15.0 * B * H * D * D, 16.0 * B * H * D * D);
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv;
  a.lq = *lq, a.lk = *lk, a.lv = *lv, a.lo = *lo, a.om = mo, a.oS = So, a.decay = decay;
  a.B = B, a.T = 1, a.H = (int)H, a.D = (int)D, a.c = (float)scale, a.c2 = (float)(scale * scale);
  const dim3 grid((unsigned)(B * H), (unsigned)cdiv(D, 32));
  if (D % 4 == 0 && al16a(state_m) && al16a(state_S))
    hipLaunchKernelGGL(step_kernel<true>, grid, dim3(256), 0, s, a, active, state_m, state_S);
  else
    hipLaunchKernelGGL(step_kernel<false>, grid, dim3(256), 0, s, a, active, state_m, state_S);
  return check_launch(what);
}
