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
// over a chunk, so the state advances token by token on the vector ALUs: 7 operations per state
// element and token forward, 12 backward. Three of each serve the squared state; the others,
// linear in their states, are taken along and not formed as matrix products over chunks. Every
// pass is one scan,
//   X_t = g X_{t-1} + u_t w_t^T (one or two such states),  y_t[o] = sum_i r_t[i] f(X_t[i][o]),
// whose columns o are independent: a wavefront keeps 32 columns of the state in registers
// (4 or 8 lanes share a column, each with as many of its rows; 16 or 8 columns where waves are
// few), reads the token's vectors from LDS and adds the partial sums over i in exchanges that
// halve the values each lane keeps: 2 x 4096 tokens, 16 heads of 64, forward and backward 461 us.
// Counters of that layout (forward, 64 features): 260 vector instructions a token and wave, 224
// of them products; the vector ALUs are active in 1.07 of a CU's busy cycles (2 where two waves'
// instructions run side by side all the time), LDS in 0.47, no bank conflicts. Backward: 1.12
// and 0.49. Neither unit is full: two waves a SIMD wait for each other's LDS reads and sums.
// A fp32 MFMA has the rate of the vector ALUs and does not run beside them: with the rank-one
// update as 4 x 4 x 1 MFMAs the same took 496 us where fmas took 474.
//
// Decay without a multiplication per token: inside a group of 8 tokens the state is kept
// divided by g^j (token j), the powers go into the token's vectors when they are staged, and
// the state is multiplied by g^8 between groups. Below |g| = 1/4 the squared powers (4^14 at
// most above it) would eat into the floats' range: such heads decay token by token.
#include "tagi_common.h"

namespace tagi {
namespace {

constexpr int kTok = 8;          // tokens per stage, and per decay group
constexpr float kGroupMin = 0.25f;
constexpr int kMaxHeadDim = 128;
constexpr double kCacheTwice = 512e6;  // bytes: twice the last-level cache

enum Mode { FWD = 0, DQ = 1, DK = 2, DV = 3 };
// vectors staged per token, over i and over o
constexpr int n_ivec(int m) { return m == FWD ? 6 : (m == DQ ? 3 : 4); }
constexpr int n_ovec(int m) { return m == FWD ? 3 : (m == DQ ? 1 : 2); }
constexpr int scan_threads(int ip, int ig, int eo) { return ip * ig / eo; }  // 64 per 64 eo / ig columns

struct Args {
  // DQ/DK/DV read the means and the deltas (dm, dS) only
  const float *mq, *Sq, *mk, *Sk, *mv, *Sv, *dm, *dS;
  tagi_heads lq, lk, lv, ld, lo;  // strides; lo of the outputs
  float *om, *oS, *km, *kS, *vm, *vS;  // outputs (backward: of the queries, keys and values)
  const float* decay;
  const void* lengths;
  int len_bytes;
  int64_t B, T;
  int H, D;
  float c, c2;
  int64_t L;     // tokens per chunk, a multiple of kTok
  int64_t nch;
  // states before each chunk (nch > 1), [bh][chunk][D][D]: M, P; last token first: G, N
  float *pre_m, *pre_S, *pre_g, *pre_n;
  const float *init_m, *init_S;  // state before the first token, or null
  float *end_m, *end_S;          // state after the last token, or null
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

// Sums over the IG lanes of a group (consecutive lanes) of EO means and EO variances per lane,
// each exchange halving the values a lane keeps: lanes whose bit IG / 2 is set end with
// variances, the others with means, of the column that column_of says. Lanes that differ in
// bits left over agree, and first_of picks one.
template <int IG, int EO>
__device__ __forceinline__ float group_sums(const float* pm, const float* ps, int lane) {
  const bool var = lane & (IG / 2), b0 = lane & 1, b1 = lane & 2;
  float r[EO];
#pragma unroll
  for (int e = 0; e < EO; ++e) {
    const float keep = var ? ps[e] : pm[e], give = var ? pm[e] : ps[e];
    r[e] = keep + dpp<IG == 8 ? kXor7 : kXor2>(give);
  }
  float h[EO > 1 ? EO / 2 : 1];
  if constexpr (EO == 1) {
    h[0] = r[0] + dpp<kXor1>(r[0]);
  } else {
#pragma unroll
    for (int e = 0; e < EO / 2; ++e) {
      const float keep = b0 ? r[EO / 2 + e] : r[e], give = b0 ? r[e] : r[EO / 2 + e];
      h[e] = keep + dpp<kXor1>(give);
    }
  }
  if constexpr (IG == 4) return h[0];
  if constexpr (EO < 4) return h[0] + dpp<kXor2>(h[0]);
  const float keep = b1 ? h[EO / 2 - 1] : h[0], give = b1 ? h[0] : h[EO / 2 - 1];
  return keep + dpp<kXor2>(give);
}
template <int IG, int EO>
__device__ __forceinline__ int column_of(int lane) {
  return EO == 4 ? 2 * (lane & 1) + ((lane >> 1) & 1) : (EO == 2 ? lane & 1 : 0);
}
template <int IG, int EO>
__device__ __forceinline__ bool first_of(int lane) {
  return (lane & (IG / 2 - 1) & ~(EO - 1)) == 0;
}

// Four consecutive values of a token's head row, of which `left` are there (zeros for the others).
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int left) {
  if constexpr (VEC) return *reinterpret_cast<const float4*>(p);
  float4 r = make_float4(p[0], 0.f, 0.f, 0.f);
  if (left > 1) r.y = p[1];
  if (left > 2) r.z = p[2];
  if (left > 3) r.w = p[3];
  return r;
}

__device__ __forceinline__ float4 mul4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) {
  return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w);
}
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// The scan of one (sequence, head, chunk), one block.
template <int MODE, int IP, int IG, int EO, bool VEC>
__device__ __forceinline__ void scan(const Args& a, float4* lds, int64_t bid) {
  // IP: the padded head dimension. A lane holds DI rows and EO columns of the state, IG lanes
  // share a column, a wave takes CW columns
  constexpr int DI = IP / IG, CW = EO * 64 / IG, NT = scan_threads(IP, IG, EO);
  static_assert((IG == 4 && EO <= 2) || (IG == 8 && EO <= 4), "layouts of group_sums");
  constexpr bool REV = MODE >= DK, TWO_STATES = MODE != DQ;
  constexpr int NI = n_ivec(MODE), NO = n_ovec(MODE);
  constexpr int C4 = IP / 4;                  // float4 chunks of a row
  // staged vectors: [vector][token][chunk], those over i, then those over o
  auto iv = [&](int v, int t, int c) -> float4& { return lds[(v * kTok + t) * C4 + c]; };
  auto ov = [&](int v, int t, int c) -> float4& { return lds[((NI + v) * kTok + t) * C4 + c]; };

  const int64_t ch = bid % a.nch, bh = bid / a.nch, b = bh / a.H;
  const int h = (int)(bh % a.H), D = a.D;
  const int64_t n = seq_len(a, b), t0 = ch * a.L, t1 = min(a.T, t0 + a.L), live = min(n, t1);
  const int cnt = live > t0 ? (int)(live - t0) : 0;  // live tokens of the chunk
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ig = lane % IG, og = lane / IG;

  const float g = a.decay[h];
  const bool grouped = fabsf(g) >= kGroupMin;
  // Between groups the state is multiplied by the float nearest g^8. What that rounds off
  // would repeat every group, so it is kept: the true state is the kept one times r (its
  // square for the variances), and r goes into the staged powers like g^j does. A decay that
  // goes token by token needs none of this: what it rounds off is gone a token later.
  const int per = grouped ? kTok : 1;  // tokens between decays
  const double gd = (double)g, gp = ipow(gd, per);
  const float s1 = (float)gp, s2 = (float)(gp * gp);
  const double e1 = grouped ? gp / (double)s1 : 1.0, e2 = grouped ? gp * gp / (double)s2 : 1.0;
  const double i1 = 1.0 / e1, i2 = 1.0 / e2;
  double r1 = 1.0, r2 = 1.0, q1 = 1.0, q2 = 1.0;  // r, r of the variances, and their inverses

  // this thread's part of a stage: token st, values 4 sc .. 4 sc + 3
  const int st = tid / C4, sc = tid % C4;
  const bool stager = st < kTok, inside = 4 * sc < D;
  const double pj = grouped && stager ? ipow(gd, st) : 1.0, ij = 1.0 / pj;  // g^j, g^-j
  const float4 z4 = make_float4(0.f, 0.f, 0.f, 0.f);

  const int64_t ob = b * a.lo.sb + h * a.lo.sh;
  auto tok = [&](int r) -> int64_t { return REV ? live - 1 - r : t0 + r; };  // r-th token of the scan

  // this thread's place in each operand, moved on by a stage at a time
  const auto place = [&](const tagi_heads& l) { return b * l.sb + h * l.sh + tok(st) * l.st + 4 * sc; };
  const auto stride = [&](const tagi_heads& l) { return (REV ? -kTok : kTok) * l.st; };
  int64_t qo = place(a.lq), ko = place(a.lk), vo = place(a.lv), dO = place(a.ld);
  float4 x0 = z4, x1 = z4, x2 = z4, x3 = z4, x4 = z4, x5 = z4;
  auto fetch = [&](int s0) {
    if (stager && inside && s0 + st < cnt) {
      const int left = D - 4 * sc;
      if constexpr (MODE == FWD) {
        x0 = load4<VEC>(a.mq + qo, left), x1 = load4<VEC>(a.Sq + qo, left);
        x2 = load4<VEC>(a.mk + ko, left), x3 = load4<VEC>(a.Sk + ko, left);
        x4 = load4<VEC>(a.mv + vo, left), x5 = load4<VEC>(a.Sv + vo, left);
      } else if constexpr (MODE == DQ) {
        x0 = load4<VEC>(a.mv + vo, left), x1 = load4<VEC>(a.mk + ko, left);
        x2 = load4<VEC>(a.dm + dO, left), x3 = load4<VEC>(a.dS + dO, left);
      } else {
        x0 = load4<VEC>(a.mq + qo, left);
        x1 = load4<VEC>(a.dm + dO, left), x2 = load4<VEC>(a.dS + dO, left);
        x3 = MODE == DK ? load4<VEC>(a.mv + vo, left) : load4<VEC>(a.mk + ko, left);
      }
    } else {
      x0 = x1 = x2 = x3 = x4 = x5 = z4;  // nothing to add, and a dead token's output is zero
    }
    qo += stride(a.lq), ko += stride(a.lk), vo += stride(a.lv), dO += stride(a.ld);
  };
  auto stage = [&]() {
    if (!stager) return;
    const float dn = (float)(pj * r1), dn2 = (float)(pj * pj * r2);
    const float up = (float)(ij * q1), up2 = (float)(ij * ij * q2);
    if constexpr (MODE == FWD) {
      iv(0, st, sc) = mul4(x2, up);
      iv(1, st, sc) = mul4(x3, up2);
      iv(2, st, sc) = mul4(mul4(x2, x2), up2);
      iv(3, st, sc) = mul4(x0, a.c * dn);
      iv(4, st, sc) = mul4(add4(x1, mul4(x0, x0)), a.c2 * dn2);
      iv(5, st, sc) = mul4(x1, a.c2 * (dn * dn));  // of the squared means
      ov(0, st, sc) = x4;
      ov(1, st, sc) = add4(mul4(x4, x4), x5);
      ov(2, st, sc) = x5;
    } else if constexpr (MODE == DQ) {
      iv(0, st, sc) = mul4(x0, up);
      iv(1, st, sc) = mul4(x2, a.c * dn);
      iv(2, st, sc) = mul4(x3, a.c2 * (dn * dn));
      ov(0, st, sc) = x1;
    } else {
      const float4 d = mul4(x1, a.c), e = mul4(x2, a.c2), q2 = mul4(x0, x0);
      if constexpr (MODE == DK) {
        iv(0, st, sc) = mul4(d, up), iv(1, st, sc) = mul4(e, up2);
        ov(0, st, sc) = x0, ov(1, st, sc) = q2;
      } else {
        iv(0, st, sc) = mul4(x0, up), iv(1, st, sc) = mul4(q2, up2);
        ov(0, st, sc) = d, ov(1, st, sc) = e;
      }
      iv(2, st, sc) = mul4(x3, dn), iv(3, st, sc) = mul4(mul4(x3, x3), dn2);
    }
  };

  // state element (i, o): rows in fours (DI a multiple of 4), the o of this wave
  constexpr int KN = DI % 4 == 0 ? 4 : DI;
  auto idx_i = [&](int k) { return KN * IG * (k / KN) + KN * ig + k % KN; };
  auto idx_o = [&](int e) { return CW * wave + EO * og + e; };
  float X[DI][EO], Y[TWO_STATES ? DI : 1][EO];
#pragma unroll
  for (int k = 0; k < DI; ++k)
#pragma unroll
    for (int e = 0; e < EO; ++e) {
      X[k][e] = 0.f;
      if constexpr (TWO_STATES) Y[k][e] = 0.f;
    }
  fetch(0);
  const bool from_pre = a.nch > 1;
  const bool tr = from_pre && MODE != FWD && MODE != DV;  // DQ and DK hold the transposed state
  const float* sm = from_pre ? (MODE == DQ || MODE == FWD ? a.pre_m : a.pre_g) : (MODE == FWD ? a.init_m : nullptr);
  const float* sS = from_pre ? (MODE == FWD ? a.pre_S : a.pre_n) : (MODE == FWD ? a.init_S : nullptr);
  if (sm) {
    const int64_t base = (from_pre ? bh * a.nch + ch : bh) * (int64_t)D * D;
    const float d1 = cnt > 0 ? g : 1.f;  // to before the first token; an empty chunk hands on what it got
#pragma unroll
    for (int k = 0; k < DI; ++k)
#pragma unroll
      for (int e = 0; e < EO; ++e) {
        const int i = idx_i(k), o = idx_o(e);
        if (i < D && o < D) {
          const int64_t at = base + (tr ? (int64_t)o * D + i : (int64_t)i * D + o);
          X[k][e] = d1 * sm[at];
          if constexpr (TWO_STATES) Y[k][e] = d1 * (d1 * sS[at]);
        }
      }
  }

  auto token = [&](int s0, int j) {
    float w[NO][EO];
#pragma unroll
    for (int v = 0; v < NO; ++v) {
      const float* p = reinterpret_cast<const float*>(&ov(v, j, 0)) + idx_o(0);
#pragma unroll
      for (int e = 0; e < EO; ++e) w[v][e] = p[e];
    }
    float pm[EO] = {}, ps[EO] = {};
#pragma unroll
    for (int k0 = 0; k0 < DI; k0 += KN) {
      float u[NI][KN];
#pragma unroll
      for (int v = 0; v < NI; ++v) {
        const float* p = reinterpret_cast<const float*>(&iv(v, j, 0)) + idx_i(k0);
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
            pm[e] = fmaf(u[3][k], x, pm[e]);
            ps[e] = fmaf(u[4][k], y, ps[e]);
            ps[e] = fmaf(u[5][k], x * x, ps[e]);
          } else if constexpr (MODE == DQ) {
            pm[e] = fmaf(u[1][k], x, pm[e]);
            ps[e] = fmaf(u[2][k], x * x, ps[e]);
          } else {
            float& y = Y[k0 + k][e];
            y = fmaf(u[1][k], w[1][e], y);
            pm[e] = fmaf(u[2][k], x, pm[e]);
            ps[e] = fmaf(u[3][k], y, ps[e]);
          }
        }
    }
    const float r = group_sums<IG, EO>(pm, ps, lane);
    const int o = idx_o(0) + column_of<IG, EO>(lane);
    const bool mine = first_of<IG, EO>(lane);
    float* om = MODE == DK ? a.km : (MODE == DV ? a.vm : a.om);
    float* oS = MODE == DK ? a.kS : (MODE == DV ? a.vS : a.oS);
    if (mine && o < D) ((lane & (IG / 2)) ? oS : om)[ob + tok(s0 + j) * a.lo.st + o] = r;
  };

  for (int s0 = 0; s0 < cnt; s0 += kTok) {
    __syncthreads();
    stage();
    __syncthreads();
    fetch(s0 + kTok);
    const int m = min(kTok, cnt - s0);
#pragma unroll 1
    for (int j0 = 0; j0 < m; j0 += per) {
      if (s0 + j0) {
#pragma unroll
        for (int k = 0; k < DI; ++k)
#pragma unroll
          for (int e = 0; e < EO; ++e) {
            X[k][e] *= s1;
            if constexpr (TWO_STATES) Y[k][e] *= s2;
          }
      }
      const int j1 = min(j0 + per, m);
#pragma unroll 1
      for (int j = j0; j < j1; ++j) token(s0, j);
    }
    r1 *= e1, r2 *= e2, q1 *= i1, q2 *= i2;  // of the next group
  }

  if constexpr (MODE == FWD) {
    // the chunk of the last live token (the first one without any) holds the final state
    if (a.end_m && ch == (n > 0 ? (n - 1) / a.L : 0)) {
      const int last = (grouped && cnt > 0) ? (cnt - 1) % kTok : 0;
      double f1 = 1.0, f2 = 1.0;  // back to the true state; r is one group ahead
      if (grouped && cnt > 0) f1 = ipow(gd, last) * (r1 * i1), f2 = ipow(gd, 2 * last) * (r2 * i2);
      const Two w1 = two(f1), w2 = two(f2);
      const int64_t base = bh * (int64_t)D * D;
#pragma unroll
      for (int k = 0; k < DI; ++k)
#pragma unroll
        for (int e = 0; e < EO; ++e) {
          const int i = idx_i(k), o = idx_o(e);
          if (i < D && o < D) {
            a.end_m[base + (int64_t)i * D + o] = scaled(w1, X[k][e]);
            a.end_S[base + (int64_t)i * D + o] = scaled(w2, Y[k][e]);
          }
        }
    }
  }
  // tokens past the sequence's end
  float* om = MODE == DK ? a.km : (MODE == DV ? a.vm : a.om);
  float* oS = MODE == DK ? a.kS : (MODE == DV ? a.vS : a.oS);
  const int64_t dead0 = max(t0, min(t1, n));
  for (int64_t q = tid; q < (t1 - dead0) * D; q += NT) {
    const int64_t at = ob + (dead0 + q / D) * a.lo.st + q % D;
    om[at] = 0.f;
    oS[at] = 0.f;
  }
}

template <int IP, int IG, int EO, bool VEC>
__global__ void __launch_bounds__(scan_threads(IP, IG, EO)) scan_fwd_kernel(Args a) {
  __shared__ float4 lds[(n_ivec(FWD) + n_ovec(FWD)) * kTok * IP / 4];
  scan<FWD, IP, IG, EO, VEC>(a, lds, blockIdx.x);
}
// The three backward scans are independent and read the same tensors: one launch, the three
// blocks of a chunk 8 block numbers apart, so that they run at about the same time on one of
// the 8 XCDs and find each other's reads in its L2.
template <int IP, int IG, int EO, bool VEC>
__global__ void __launch_bounds__(scan_threads(IP, IG, EO)) scan_bwd_kernel(Args a) {
  __shared__ float4 lds[(n_ivec(DK) + n_ovec(DK)) * kTok * IP / 4];
  const int64_t x = blockIdx.x, q = x >> 3, bid = (q / 3) * 8 + (x & 7);
  if (bid >= a.B * a.H * a.nch) return;
  if (q % 3 == 0)
    scan<DK, IP, IG, EO, VEC>(a, lds, bid);
  else if (q % 3 == 1)
    scan<DV, IP, IG, EO, VEC>(a, lds, bid);
  else
    scan<DQ, IP, IG, EO, VEC>(a, lds, bid);
}

// ------------------------------------------------------------------- chunk contributions
// A chunk's own share of the state after it, sum_t g^(tokens still to come) u_t w_t^T, is a
// matrix product over the chunk's tokens: fp32 MFMAs (32 x 32 x 2, a token for each half of
// the wave), operands straight from memory, 32 floats of a token per half wave. A wave forms
// 32 rows and NO 32-column tiles. The powers of the decay run from the token that keeps 1,
// in float64, so that neither a small decay nor a long chunk leaves the floats' range early.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool REV, bool SECOND, int NO>
__device__ __forceinline__ void chunk_sum(const Args& a, int it, int ot) {
  const int64_t bid = blockIdx.x, ch = bid % a.nch, bh = bid / a.nch, b = bh / a.H;
  if (ch == (REV ? 0 : a.nch - 1)) return;  // no chunk comes after it
  const int h = (int)(bh % a.H), D = a.D, lane = threadIdx.x & 63, half = lane >> 5, l5 = lane & 31;
  const int64_t n = seq_len(a, b), t0 = ch * a.L, t1 = min(a.T, t0 + a.L), live = min(n, t1);
  if (live <= t0) return;  // the carry does not read it
  const int cnt = (int)(live - t0);
  const int i = 32 * it + l5;
  const bool iok = i < D;
  // u: keys (REV: queries), w: values (REV: deltas), with their variances' counterparts
  const tagi_heads lu = REV ? a.lq : a.lk, lw = REV ? a.ld : a.lv;
  const float* um = (REV ? a.mq : a.mk) + b * lu.sb + h * lu.sh + i;
  const float* uS = REV ? nullptr : a.Sk + b * lu.sb + h * lu.sh + i;
  const float* wm = (REV ? a.dm : a.mv) + b * lw.sb + h * lw.sh;
  const float* wS = (REV ? a.dS : a.Sv) + b * lw.sb + h * lw.sh;
  const double g = (double)a.decay[h];
  double p = half ? g : 1.0;
  const double gg = g * g;
  f32x16 X[NO] = {}, Y[NO] = {};
  constexpr int U = 4;  // pairs of tokens a stage; a stage's loads run during the one before
  struct Stage {
    float ku[U], ks[U], wv[U][NO], ws[U][NO];
  };
  auto fetch = [&](Stage& f, int r0) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int r = r0 + 2 * q + half;
      const bool on = r < cnt;
      const int64_t t = REV ? t0 + r : live - 1 - r;
      f.ku[q] = on && iok ? um[t * lu.st] : 0.f;
      if constexpr (SECOND && !REV) f.ks[q] = on && iok ? uS[t * lu.st] : 0.f;
#pragma unroll
      for (int o = 0; o < NO; ++o) {
        const int oc = 32 * (ot + o) + l5;
        const bool ok = on && oc < D;
        f.wv[q][o] = ok ? wm[t * lw.st + oc] : 0.f;
        if constexpr (SECOND) f.ws[q][o] = ok ? wS[t * lw.st + oc] : 0.f;
      }
    }
  };
  auto product = [&](const Stage& f) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const float f1 = (float)p, f2 = (float)(p * p);
      p *= gg;
      const float c1 = REV ? a.c : 1.f, c2 = REV ? a.c2 : 1.f;
      const float x = f.ku[q] * f1, k2 = f.ku[q] * f.ku[q] * f2;
#pragma unroll
      for (int o = 0; o < NO; ++o) {
        X[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, c1 * f.wv[q][o], X[o], 0, 0, 0);
        if constexpr (SECOND) {
          Y[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(k2, c2 * f.ws[q][o], Y[o], 0, 0, 0);
          if constexpr (!REV)
            Y[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(f.ks[q] * f2, f.wv[q][o] * f.wv[q][o] + f.ws[q][o], Y[o], 0, 0,
                                                        0);
        }
      }
    }
  };
  Stage f0, f1;
  fetch(f0, 0);
  for (int r0 = 0; r0 < cnt; r0 += 4 * U) {  // fetches past the chunk's tokens are zeros
    fetch(f1, r0 + 2 * U);
    product(f0);
    fetch(f0, r0 + 4 * U);
    product(f1);
  }
  float* sm = REV ? a.pre_g : a.pre_m;
  float* sS = REV ? a.pre_n : a.pre_S;
  const int64_t base = (bh * a.nch + ch) * (int64_t)D * D;
#pragma unroll
  for (int o = 0; o < NO; ++o)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = 32 * it + 8 * (e >> 2) + 4 * half + (e & 3), col = 32 * (ot + o) + l5;
      if (row < D && col < D) {
        sm[base + (int64_t)row * D + col] = X[o][e];
        if constexpr (SECOND) sS[base + (int64_t)row * D + col] = Y[o][e];
      }
    }
}

template <int NO>
__global__ void __launch_bounds__(64) sum_fwd_kernel(Args a) {
  chunk_sum<false, true, NO>(a, blockIdx.y, blockIdx.z * NO);
}
// Keys and values into the mean state, queries and deltas into the adjoint ones.
template <int NO>
__global__ void __launch_bounds__(64) sum_bwd_kernel(Args a) {
  const int tiles = (a.D + 31) / 32;
  if ((int)blockIdx.y < tiles)
    chunk_sum<false, false, NO>(a, blockIdx.y, blockIdx.z * NO);
  else
    chunk_sum<true, true, NO>(a, blockIdx.y - tiles, blockIdx.z * NO);
}

// Chunk contributions to the states before each chunk, in place: run = g^L run + sum. A chunk
// with fewer live tokens than L has only empty ones after it, or (last token first) an empty
// run before it, so its own power is never needed.
// A: chunks in flight, whose loads do not wait for each other's carry (128 chunks of 8 heads
// of 64: 95 us one by one, 22 us sixteen at a time).
template <bool REV, int A>
__device__ __forceinline__ void carry(const Args& a, float* x, const float* init, bool second) {
  const int64_t DD = (int64_t)a.D * a.D, per = (DD + 255) / 256, bh = blockIdx.x / per, b = bh / a.H;
  const int64_t el = (blockIdx.x % per) * 256 + threadIdx.x;
  if (el >= DD) return;
  const int64_t n = seq_len(a, b);
  const double gL = ipow((double)a.decay[bh % a.H], a.L);
  const Two f = two(second ? gL * gL : gL);
  x += bh * a.nch * DD + el;
  float run = init ? init[bh * DD + el] : 0.f;
  for (int64_t k0 = 0; k0 < a.nch; k0 += A) {
    float own[A];
#pragma unroll
    for (int j = 0; j < A; ++j) {
      const int64_t ch = REV ? a.nch - 1 - k0 - j : k0 + j;
      const bool use = k0 + j + 1 < a.nch && ch * a.L < n;  // the last chunk's is not formed
      own[j] = use ? x[ch * DD] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < A; ++j) {
      if (k0 + j >= a.nch) break;
      const int64_t ch = REV ? a.nch - 1 - k0 - j : k0 + j;
      x[ch * DD] = run;
      if (ch * a.L < n) run = scaled(f, run) + own[j];
    }
  }
}
template <int A>
__global__ void __launch_bounds__(256) carry_fwd_kernel(Args a) {
  carry<false, A>(a, blockIdx.y ? a.pre_S : a.pre_m, blockIdx.y ? a.init_S : a.init_m, blockIdx.y);
}
template <int A>
__global__ void __launch_bounds__(256) carry_bwd_kernel(Args a) {
  if (blockIdx.y == 0)
    carry<false, A>(a, a.pre_m, nullptr, false);
  else
    carry<true, A>(a, blockIdx.y == 1 ? a.pre_g : a.pre_n, nullptr, blockIdx.y == 2);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
template <bool NT>
__device__ __forceinline__ f32x4 ld_state(const float* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
  return *reinterpret_cast<const f32x4*>(p);
}
template <bool NT>
__device__ __forceinline__ void st_state(float* p, f32x4 v) {
  if constexpr (NT)
    __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
  else
    *reinterpret_cast<f32x4*>(p) = v;
}

// One token of every sequence: the state is read, advanced and written once, 32 columns of a
// head a block. HBM bound: 64 sequences of 16 heads of 128, whose states the cache holds, 44 us
// (6.1 TB/s read and written), 256 of them 198 us (5.4).
template <bool VEC, bool NT>
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
      f32x4 xm = {0.f, 0.f, 0.f, 0.f}, xS = xm;
      if (col < D) xm = ld_state<NT>(M + at), xS = ld_state<NT>(P + at);
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
        st_state<NT>(M + at, f32x4{x[0], x[1], x[2], x[3]});
        st_state<NT>(P + at, f32x4{y[0], y[1], y[2], y[3]});
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

// Columns of a wavefront and tokens of a chunk. A wave per (sequence, head, 32 columns) is the
// least work, but few of them leave the GPU's 1024 SIMDs idle. Narrower waves (16 or 8
// columns) read the token's vectors more often; chunks cost a pass that sums each one's
// contribution, the state traffic, and two launches. Measured (us, forward / backward; "n x c":
// n chunks, c columns):
//   64 x 256 tokens, 8 heads of 32:  1 x 8 64 / 114, 1 x 16 81 / 91, 1 x 32 101 / 93, 4 x 32 75 / 105
//   32 x 128 tokens, 8 heads of 64:  1 x 8 48 / 78, 1 x 16 56 / 65, 2 x 16 77 / 103, 4 x 32 73 / 122
//   2 x 4096 tokens, 16 heads of 64: 32 x 32 181 / 301, 16 x 32 276 / 280, 16 x 16 191 / 303
//   1 x 512 tokens, 8 heads of 64:   16 x 8 34 / 37, 16 x 16 37 / 39, 16 x 32 48 / 47
//   1 x 2048 tokens, 4 heads of 128: 64 x 16 75 / 131, 32 x 32 126 / 115, 64 x 32 94 / 138
//   1 x 64 tokens, 8 heads of 32:    1 x 8 18 / 24, 1 x 16 21 / 24, 2 x 8 22 / 31
//   3 x 339 tokens, 1 head of 128:   11 x 16 56 / 49, 9 x 16 64 / 55, 6 x 16 85 / 67
//   32 x 2048 tokens, 8 heads of 64: 1 x 8 729 / 1218, 1 x 16 851 / 1012, 4 x 32 624 / 1055
//   16 x 512 tokens, 8 heads of 128: 1 x 8 479 / -, 1 x 16 413 / 564, 4 x 32 326 / 554
// So: no chunks where the widest waves that do reach 2048 (backward, whose three scans run side
// by side: 1024); forward they may have 8 columns for few tokens, and long heads' have 16 at
// least, since narrow waves spend their time reading LDS. No chunks below 128 tokens; else as
// many as bring 32-column waves there, of 32 tokens at least (backward: and of half a head's
// features, its three states' traffic, where those are waves enough), with narrower waves
// where that falls short. Whole groups of kTok tokens make chunks longer than T / n: 3 x 339
// tokens get 9 of 40, not 11 of 32.
struct Chunks {
  int64_t L, nch;
  int cols;
};
Chunks chunks(int64_t B, int64_t T, int64_t H, int64_t D, bool bwd) {
  // three-wave blocks (65 to 96 features) fit a CU twice, not 2 2/3 times: 512 of them at once.
  // Chunk counts are rounded up, so that a few more may be launched (7 x 777 tokens, 6 heads of
  // 80: 11 chunks, 462 blocks, 152; 13, which this takes, 546 blocks, 152; 14, 588 blocks, 181)
  const int64_t heads = B * H, full = D > 64 && D <= 96 ? 1536 : 2048, target = bwd ? 1024 : full;
  const int64_t enough = bwd ? 512 : full;
  const int narrowest = D > 64 ? 16 : 8;
  const auto waves = [&](int cols) { return heads * cdiv(D, cols); };
  Chunks c{cdiv(T > 0 ? T : 1, kTok) * kTok, 1, narrowest};
  for (int cols = 32; cols >= (bwd || T >= 512 ? 16 : narrowest); cols /= 2)
    if (waves(cols) >= target) {
      c.cols = cols;
      return c;
    }
  if (T < 128) return c;
  const int64_t least = bwd && D > 64 && T / (D / 2) * waves(32) >= enough ? D / 2 : 32;
  int64_t n = cdiv(target, waves(32));
  if (n > T / least) n = T / least;
  c.L = cdiv(cdiv(T, n), kTok) * kTok;
  c.nch = cdiv(T, c.L);
  for (c.cols = 32; c.cols > narrowest && c.nch * waves(c.cols) < enough;) c.cols /= 2;
  return c;
}

template <bool BWD, bool VEC>
void launch_scan_v(const Args& a, int cols, hipStream_t s) {
  const int64_t n = a.B * a.H * a.nch;
  const dim3 grid((unsigned)(BWD ? cdiv(n, 8) * 24 : n));
#define TAGI_SCAN(IP, IG, EO)                                                                                     \
  do {                                                                                                            \
    if constexpr (BWD)                                                                                            \
      hipLaunchKernelGGL((scan_bwd_kernel<IP, IG, EO, VEC>), grid, dim3(scan_threads(IP, IG, EO)), 0, s, a);      \
    else                                                                                                          \
      hipLaunchKernelGGL((scan_fwd_kernel<IP, IG, EO, VEC>), grid, dim3(scan_threads(IP, IG, EO)), 0, s, a);      \
    return;                                                                                                       \
  } while (0)
  // Lanes to a column: 4 leave the shorter sum, 8 read half as much from LDS, which bounds 16
  // columns of more than 32 features (backward 32 x 512 tokens, 8 heads of 64: 265 against 245
  // us, forward 3 x 339, one head of 128: 69 and 63; 64 x 256, 8 heads of 32: 90 and 93) and the
  // backward of 32 columns of more than 64 (16 x 512, 8 heads of 128: 645 and 570).
#define TAGI_SCAN_COLS(IP)                        \
  do {                                            \
    constexpr int G16 = IP > 32 ? 8 : 4;          \
    constexpr int G32 = BWD && IP > 64 ? 8 : 4;   \
    if constexpr (IP <= 64)                       \
      if (cols == 8) TAGI_SCAN(IP, 8, 1);         \
    if (cols == 16)                               \
      TAGI_SCAN(IP, G16, G16 / 4);                \
    else                                          \
      TAGI_SCAN(IP, G32, G32 / 2);                \
  } while (0)
  if (a.D <= 16) {
    if (cols == 8)
      TAGI_SCAN(16, 8, 1);
    else
      TAGI_SCAN(16, 4, 1);
  } else if (a.D <= 32) {
    TAGI_SCAN_COLS(32);
  } else if (a.D <= 64) {
    TAGI_SCAN_COLS(64);
  } else if (a.D <= 96) {
    TAGI_SCAN_COLS(96);
  } else {
    TAGI_SCAN_COLS(128);
  }
#undef TAGI_SCAN
#undef TAGI_SCAN_COLS
}

// The states before every chunk, then the scans.
template <bool BWD>
void launch_all(const Args& a, int cols, bool vec, hipStream_t s) {
  if (a.nch > 1) {
    const int tiles = (int)cdiv(a.D, 32);
    const unsigned x = (unsigned)(a.B * a.H * a.nch), y = BWD ? 2 * tiles : tiles;
    if (tiles % 2 == 0) {
      const dim3 grid(x, y, tiles / 2);
      if constexpr (BWD)
        hipLaunchKernelGGL(sum_bwd_kernel<2>, grid, dim3(64), 0, s, a);
      else
        hipLaunchKernelGGL(sum_fwd_kernel<2>, grid, dim3(64), 0, s, a);
    } else {
      const dim3 grid(x, y, tiles);
      if constexpr (BWD)
        hipLaunchKernelGGL(sum_bwd_kernel<1>, grid, dim3(64), 0, s, a);
      else
        hipLaunchKernelGGL(sum_fwd_kernel<1>, grid, dim3(64), 0, s, a);
    }
    const dim3 grid((unsigned)(cdiv((int64_t)a.D * a.D, 256) * a.B * a.H), BWD ? 3 : 2);
    if constexpr (BWD) {
      if (a.nch <= 4)
        hipLaunchKernelGGL(carry_bwd_kernel<4>, grid, dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL(carry_bwd_kernel<16>, grid, dim3(256), 0, s, a);
    } else {
      if (a.nch <= 4)
        hipLaunchKernelGGL(carry_fwd_kernel<4>, grid, dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL(carry_fwd_kernel<16>, grid, dim3(256), 0, s, a);
    }
  }
  vec ? launch_scan_v<BWD, true>(a, cols, s) : launch_scan_v<BWD, false>(a, cols, s);
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t H, int64_t D) {
  TAGI_REQUIRE(B >= 0 && T >= 0 && H > 0 && D > 0, "%s: bad sizes", what);
  // a launch has fewer than 2^32 threads: three blocks of 256 for a head
  TAGI_REQUIRE(B < (1ll << 22) && H < (1ll << 22) && B * H < (1ll << 22) && T < (1ll << 31), "%s: too large", what);
  if (D > kMaxHeadDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxHeadDim);
  return TAGI_OK;
}

int64_t state_floats(int64_t B, int64_t H, int64_t D, int64_t nch) { return (B * H * nch * D * D + 3) / 4 * 4; }

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_linear_attention_fwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || D <= 0) return 0;
  const Chunks c = chunks(B, T, H, D, false);
  return c.nch > 1 ? 2 * state_floats(B, H, D, c.nch) * 4 : 0;
}

extern "C" int64_t tagi_linear_attention_bwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || D <= 0) return 0;
  const Chunks c = chunks(B, T, H, D, true);
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
  const Chunks c = chunks(B, T, H, D, false);
  TAGI_REQUIRE(B * H * c.nch < (1ll << 22), "%s: too large", what);
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
    a.pre_m = static_cast<float*>(ws);
    a.pre_S = a.pre_m + state_floats(B, H, D, c.nch);
  }
  launch_all<false>(a, c.cols, vec, s);
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
  const Chunks c = chunks(B, T, H, D, true);
  TAGI_REQUIRE(B * H * c.nch < (1ll << 22), "%s: too large", what);
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
  a.om = dmq, a.oS = dSq, a.km = dmk, a.kS = dSk, a.vm = dmv, a.vS = dSv;
  if (c.nch > 1) {
    const int64_t n = state_floats(B, H, D, c.nch);
    a.pre_m = static_cast<float*>(ws);
    a.pre_g = a.pre_m + n, a.pre_n = a.pre_g + n;
  }
  launch_all<true>(a, c.cols, vec, s);
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
  // states well beyond the last-level cache: the nontemporal policy reaches further (537 MB of
  // states, 1.07 GB read and written: 217 -> 198 us; 268 MB: 91 -> 94)
  const bool vec = D % 4 == 0 && al16a(state_m) && al16a(state_S), nt = 8.0 * B * H * D * D > kCacheTwice;
  const auto kernel = !vec ? step_kernel<false, false> : (nt ? step_kernel<true, true> : step_kernel<true, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, active, state_m, state_S);
  return check_launch(what);
}
