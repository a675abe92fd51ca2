// RMSNorm of every query and key head and its rotation by position, on Gaussian moments.
//
// For one head of one token, with its moments (m, S), the weight's (g, Sg) and the pair of
// features (a, b) that turns by the angle t = position * frequency:
//   inv = 1 / sqrt(mean(m^2 + S) + eps)
//   n = m inv g,  N = inv^2 (S (g^2 + Sg) + Sg m^2)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t) of the means n,
//   (A, B) -> (A cos^2 t + B sin^2 t, A sin^2 t + B cos^2 t) of the variances N
// (the features stay independent Gaussians: the pair's covariance is dropped, as everywhere).
// Backward, with inv held: the deltas turn back (the transposed maps), then
//   dm = dn inv g, dS = dN (inv g)^2;  dg = Sg sum dn inv m, dSg = Sg^2 sum dN (inv m)^2.
//
// HBM bound: a row is read once, its statistic and its pairs stay in registers, and it is
// written once; queries and keys share the launch, and the angles of a token (in 64 bits up to
// the reduced turn, since positions reach millions) are formed once for all of its heads. Measured:
// 8 x 2048 tokens, 16 query and 16 key heads of 128, forward 196 us and backward 260, 5.3 TB/s of
// 2.4 GB, where a copy has 5.4.
#include "tagi_common.h"

namespace tagi {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kMaxAxes = 4;
// The backward: each block has its own column sums. 1024 of them fill the GPU; beyond, one thread adds up at
// most kMostRows rows in fp32 (2^30 rows of one feature: 6e-5 wrong with 4096 rows a thread).
constexpr int kMaxBlocks = 1024, kMostRows = 512;

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

struct Args {
  // forward: moments in, moments out. Backward: dq/dk deltas in, mq/mk the forward's means
  const float *mq, *Sq, *mk, *Sk, *dmq, *dSq, *dmk, *dSk;
  tagi_heads lq, lk, ldq, ldk, loq, lok;  // lo: the backward's outputs
  float *oqm, *oqS, *okm, *okS, *inv;
  const float *wqm, *wqS, *wkm, *wkS;  // NULL: no norm
  const void* positions;
  int pos_bytes, axes, pairs, interleaved;
  int bound[kMaxAxes];  // pairs below bound[i] belong to axis i or an earlier one
  const double* freq;
  int64_t T, tokens;
  int H, G, D, L, TB;  // L lanes hold a row; a block takes TB tokens at a time
  float eps;
  float* part;  // backward: [4][D][blocks]
};

// Features of a lane's four pairs. Pairs that turn: (u, u + pairs) or (2u, 2u + 1); the others
// are (2u, 2u + 1) in either layout, the last one alone where the head is odd.
struct Unit {
  int a, b;  // b < 0: no such feature; a < 0: no such pair
  bool turns;
};
__device__ __forceinline__ Unit unit(const Args& A, int u) {
  Unit x;
  x.turns = u < A.pairs;
  if (x.turns && !A.interleaved) {
    x.a = u, x.b = u + A.pairs;
  } else {
    x.a = 2 * u < A.D ? 2 * u : -1;
    x.b = 2 * u + 1 < A.D ? 2 * u + 1 : -1;
  }
  return x;
}

// A lane's eight features of one row, a[4] and b[4]. VEC: four neighbouring pairs (all turning or
// none, where a pair's features lie apart) in two 16-byte accesses; otherwise pairs lane, lane + L, ... one feature at a time.
template <bool VEC>
__device__ __forceinline__ void load_row(const Args& A, const float* p, int lane, float (&a)[4], float (&b)[4]) {
  if constexpr (VEC) {
    const int u = 4 * lane;
    f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (2 * u < A.D) {
      if (u < A.pairs && !A.interleaved) {
        x = *reinterpret_cast<const f4*>(p + u), y = *reinterpret_cast<const f4*>(p + u + A.pairs);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = x[j], b[j] = y[j];
        return;
      }
      x = *reinterpret_cast<const f4*>(p + 2 * u), y = *reinterpret_cast<const f4*>(p + 2 * u + 4);
    }
    a[0] = x[0], b[0] = x[1], a[1] = x[2], b[1] = x[3];
    a[2] = y[0], b[2] = y[1], a[3] = y[2], b[3] = y[3];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Unit x = unit(A, lane + A.L * j);
      a[j] = x.a >= 0 ? p[x.a] : 0.f;
      b[j] = x.b >= 0 ? p[x.b] : 0.f;
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void store_row(const Args& A, float* p, int lane, const float (&a)[4], const float (&b)[4]) {
  if constexpr (VEC) {
    const int u = 4 * lane;
    if (2 * u >= A.D) return;
    if (u < A.pairs && !A.interleaved) {
      *reinterpret_cast<f4*>(p + u) = f4{a[0], a[1], a[2], a[3]};
      *reinterpret_cast<f4*>(p + u + A.pairs) = f4{b[0], b[1], b[2], b[3]};
    } else {
      *reinterpret_cast<f4*>(p + 2 * u) = f4{a[0], b[0], a[1], b[1]};
      *reinterpret_cast<f4*>(p + 2 * u + 4) = f4{a[2], b[2], a[3], b[3]};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Unit x = unit(A, lane + A.L * j);
      if (x.a >= 0) p[x.a] = a[j];
      if (x.b >= 0) p[x.b] = b[j];
    }
  }
}

// cos and sin of the block's tokens' pairs into LDS. The turn position * frequency / 2 pi is
// reduced in float64: its error is 2^-53 of the turns, 1e-10 at a million of them.
__device__ __forceinline__ void angles(const Args& A, int64_t token0, int n, float2* cs) {
  for (int i = threadIdx.x; i < n * A.pairs; i += kThreads) {
    const int tok = i / A.pairs, u = i % A.pairs;
    int axis = 0;
#pragma unroll
    for (int k = 0; k + 1 < kMaxAxes; ++k) axis += k + 1 < A.axes && u >= A.bound[k];
    const int64_t at = (token0 + tok) * A.axes + axis;
    const double pos = A.pos_bytes == 8 ? (double)static_cast<const int64_t*>(A.positions)[at]
                                        : (double)static_cast<const int32_t*>(A.positions)[at];
    double turn = pos * A.freq[u] * 0.15915494309189533577;
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    cs[i] = make_float2(c, s);
  }
}

__device__ __forceinline__ float row_sum(float x, int L) {
  for (int w = L >> 1; w > 0; w >>= 1) x += __shfl_xor(x, w);
  return x;
}

template <bool VEC>
__device__ __forceinline__ void lane_turns(const Args& A, const float2* cs, int lane, float (&c)[4], float (&s)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int u = VEC ? 4 * lane + j : lane + A.L * j;
    const float2 t = u < A.pairs ? cs[u] : make_float2(1.f, 0.f);
    c[j] = t.x, s[j] = t.y;
  }
}
// The lane's weights; zeros where it holds no feature
template <bool VEC>
__device__ __forceinline__ void lane_weights(const Args& A, const float* w, int lane, float (&a)[4], float (&b)[4]) {
  load_row<VEC>(A, w, lane, a, b);
}

__device__ __forceinline__ int64_t head_at(const tagi_heads& l, int64_t b, int64_t t, int h) {
  return b * l.sb + t * l.st + h * l.sh;
}

// The token's batch element: a division of 64 bits takes as long as a row's products.
__device__ __forceinline__ int64_t batch_of(const Args& A, int64_t token) {
  return A.tokens >> 31 ? token / A.T : (int64_t)((uint32_t)token / (uint32_t)A.T);
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) qk_rotary_fwd_kernel(const Args A) {
  extern __shared__ float2 cs[];
  const int lane = threadIdx.x & (A.L - 1), heads = A.H + A.G, groups = kThreads / A.L;
  const int64_t token0 = (int64_t)blockIdx.x * A.TB;
  const int n = (int)(A.tokens - token0 < A.TB ? A.tokens - token0 : A.TB);
  angles(A, token0, n, cs);
  __syncthreads();
  // all of a wave's lanes run the same number of rows: the row sums cross lanes
  for (int base = 0; base < n * heads; base += groups) {
    const int r = base + (int)threadIdx.x / A.L;
    const bool on = r < n * heads;
    const int tok = on ? r / heads : 0, h = on ? r % heads : 0;
    const int64_t token = token0 + tok, b = batch_of(A, token), t = token - b * A.T;
    const bool q = h < A.H;
    const int64_t at = q ? head_at(A.lq, b, t, h) : head_at(A.lk, b, t, h - A.H);
    float ma[4], mb[4], Sa[4], Sb[4];
    load_row<VEC>(A, (q ? A.mq : A.mk) + at, lane, ma, mb);
    load_row<VEC>(A, (q ? A.Sq : A.Sk) + at, lane, Sa, Sb);
    if (A.wqm) {
      float ga[4], gb[4], ha[4], hb[4], x = 0.f;
      lane_weights<VEC>(A, q ? A.wqm : A.wkm, lane, ga, gb);
      lane_weights<VEC>(A, q ? A.wqS : A.wkS, lane, ha, hb);
#pragma unroll
      for (int j = 0; j < 4; ++j) x += (ma[j] * ma[j] + Sa[j]) + (mb[j] * mb[j] + Sb[j]);
      const float inv = 1.f / sqrtf(row_sum(x, A.L) / (float)A.D + A.eps);
      if (on && lane == 0) A.inv[token * heads + h] = inv;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float na = ma[j] * inv, nb = mb[j] * inv;
        Sa[j] = inv * inv * (Sa[j] * (ga[j] * ga[j] + ha[j])) + ha[j] * (na * na);
        Sb[j] = inv * inv * (Sb[j] * (gb[j] * gb[j] + hb[j])) + hb[j] * (nb * nb);
        ma[j] = na * ga[j], mb[j] = nb * gb[j];
      }
    }
    float c[4], s[4];
    lane_turns<VEC>(A, cs + tok * A.pairs, lane, c, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = ma[j], y = mb[j], X = Sa[j], Y = Sb[j], c2 = c[j] * c[j], s2 = s[j] * s[j];
      ma[j] = x * c[j] - y * s[j], mb[j] = x * s[j] + y * c[j];
      Sa[j] = X * c2 + Y * s2, Sb[j] = X * s2 + Y * c2;
    }
    if (!on) continue;
    const int64_t o = q ? (token * A.H + h) * A.D : (token * A.G + h - A.H) * A.D;
    store_row<VEC>(A, (q ? A.oqm : A.okm) + o, lane, ma, mb);
    store_row<VEC>(A, (q ? A.oqS : A.okS) + o, lane, Sa, Sb);
  }
}

// The column sums of the weights' deltas: a thread's rows in registers (at most kMostRows, or a token's),
// a block's threads in a fixed order through LDS, the blocks' in float64 (column_sums_kernel).
template <bool VEC>
__global__ void __launch_bounds__(kThreads) qk_rotary_bwd_kernel(const Args A) {
  extern __shared__ float2 cs[];
  float* red = reinterpret_cast<float*>(cs + A.TB * A.pairs);  // kThreads * 8 floats
  const int lane = threadIdx.x & (A.L - 1), heads = A.H + A.G, groups = kThreads / A.L;
  float gm[2][8] = {}, gS[2][8] = {};  // [queries, keys][a, b]
  for (int64_t token0 = (int64_t)blockIdx.x * A.TB; token0 < A.tokens; token0 += (int64_t)gridDim.x * A.TB) {
    const int n = (int)(A.tokens - token0 < A.TB ? A.tokens - token0 : A.TB);
    __syncthreads();  // the angles of the tokens before are read no more
    angles(A, token0, n, cs);
    __syncthreads();
    for (int r = (int)threadIdx.x / A.L; r < n * heads; r += groups) {
      const int tok = r / heads, h = r % heads;
      const int64_t token = token0 + tok, b = batch_of(A, token), t = token - b * A.T;
      const bool q = h < A.H;
      const int64_t at = q ? head_at(A.ldq, b, t, h) : head_at(A.ldk, b, t, h - A.H);
      float da[4], db[4], ea[4], eb[4], c[4], s[4];
      load_row<VEC>(A, (q ? A.dmq : A.dmk) + at, lane, da, db);
      load_row<VEC>(A, (q ? A.dSq : A.dSk) + at, lane, ea, eb);
      lane_turns<VEC>(A, cs + tok * A.pairs, lane, c, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = da[j], y = db[j], X = ea[j], Y = eb[j], c2 = c[j] * c[j], s2 = s[j] * s[j];
        da[j] = x * c[j] + y * s[j], db[j] = y * c[j] - x * s[j];
        ea[j] = X * c2 + Y * s2, eb[j] = X * s2 + Y * c2;
      }
      if (A.wqm) {
        const int64_t in = q ? head_at(A.lq, b, t, h) : head_at(A.lk, b, t, h - A.H);
        const float inv = A.inv[token * heads + h];
        float ma[4], mb[4], ga[4], gb[4];
        load_row<VEC>(A, (q ? A.mq : A.mk) + in, lane, ma, mb);
        lane_weights<VEC>(A, q ? A.wqm : A.wkm, lane, ga, gb);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float na = ma[j] * inv, nb = mb[j] * inv, wa = inv * ga[j], wb = inv * gb[j];
          const float xa = da[j] * na, xb = db[j] * nb, ya = ea[j] * (na * na), yb = eb[j] * (nb * nb);
          gm[0][j] += q ? xa : 0.f, gm[0][4 + j] += q ? xb : 0.f, gm[1][j] += q ? 0.f : xa, gm[1][4 + j] += q ? 0.f : xb;
          gS[0][j] += q ? ya : 0.f, gS[0][4 + j] += q ? yb : 0.f, gS[1][j] += q ? 0.f : ya, gS[1][4 + j] += q ? 0.f : yb;
          da[j] *= wa, db[j] *= wb, ea[j] *= wa * wa, eb[j] *= wb * wb;
        }
      }
      // the features that this lane has read: the outputs may be the deltas themselves
      const int64_t o = q ? head_at(A.loq, b, t, h) : head_at(A.lok, b, t, h - A.H);
      store_row<VEC>(A, (q ? A.oqm : A.okm) + o, lane, da, db);
      store_row<VEC>(A, (q ? A.oqS : A.okS) + o, lane, ea, eb);
    }
  }
  if (!A.part) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // dgq, dSgq, dgk, dSgk
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x * 8 + j] = (k & 1) ? gS[k >> 1][j] : gm[k >> 1][j];
    __syncthreads();
    for (int i = threadIdx.x; i < A.L * 8; i += kThreads) {
      const int ln = i / 8, j = i % 8, u = VEC ? 4 * ln + (j & 3) : ln + A.L * (j & 3);
      const Unit x = unit(A, u);
      const int d = j < 4 ? x.a : x.b;
      if (d < 0 || d >= A.D) continue;
      float sum = 0.f;
      for (int g = 0; g < groups; ++g) sum += red[(g * A.L + ln) * 8 + j];
      A.part[((int64_t)k * A.D + d) * gridDim.x + blockIdx.x] = sum;
    }
  }
}

// One wave per sum: the blocks' partial sums in float64, times Sg or Sg^2.
__global__ void __launch_bounds__(64) column_sums_kernel(const float* part, int blocks, int D, const float* wqS,
                                                         const float* wkS, float* dwq, float* dSwq, float* dwk,
                                                         float* dSwk) {
  const int k = blockIdx.x / D, d = blockIdx.x % D;
  const float* p = part + (int64_t)blockIdx.x * blocks;
  double sum = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 64) sum += (double)p[i];
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
  if (threadIdx.x != 0) return;
  const double S = (double)(k < 2 ? wqS : wkS)[d];
  float* out = k == 0 ? dwq : (k == 1 ? dSwq : (k == 2 ? dwk : dSwk));
  out[d] = (float)(sum * ((k & 1) ? S * S : S));
}

int lanes_of(int64_t D) {  // four pairs a lane
  int L = 1;
  while (8 * L < D) L *= 2;
  return L;
}
// Tokens of a block at a time: enough rows for its threads, one at least.
int tokens_of(int64_t heads, int L) {
  const int64_t rows = kThreads / L;
  return (int)(heads >= rows ? 1 : cdiv(rows, heads));
}
int64_t bwd_blocks(int64_t tokens, int64_t heads, int64_t D) {
  const int L = lanes_of(D), TB = tokens_of(heads, L);
  const int64_t n = cdiv(tokens, TB), rows = cdiv(TB * heads, kThreads / L);  // rows of a thread a turn
  const int64_t turns = rows < kMostRows ? kMostRows / rows : 1, most = cdiv(n, turns);
  const int64_t blocks = most > kMaxBlocks ? most : kMaxBlocks;
  return n < blocks ? n : blocks;
}

int fill(const char* what, Args& a, int64_t B, int64_t T, int64_t H, int64_t G, int64_t D, const void* positions,
         int pos_bytes, int64_t axes, const int64_t* sections, const double* freq, int64_t pairs, int interleaved) {
  TAGI_REQUIRE(B >= 0 && T >= 0 && H > 0 && G >= 0 && D > 0, "%s: bad sizes", what);
  if (D > kMaxDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxDim);
  TAGI_REQUIRE(H + G < (1 << 20) && (T == 0 || B < (1ll << 31) / T), "%s: too large", what);
  TAGI_REQUIRE(pairs >= 0 && 2 * pairs <= D, "%s: %lld pairs in %lld features", what, (long long)pairs, (long long)D);
  a.pairs = (int)pairs, a.axes = (int)axes, a.interleaved = interleaved != 0;
  if (pairs > 0) {
    TAGI_REQUIRE(axes >= 1 && axes <= kMaxAxes && sections, "%s: positions have 1 to %d axes", what, kMaxAxes);
    TAGI_REQUIRE(pos_bytes == 4 || pos_bytes == 8, "%s: positions are int32 or int64", what);
    int64_t sum = 0;
    for (int i = 0; i < axes; ++i) {
      TAGI_REQUIRE(sections[i] >= 0 && sections[i] <= pairs, "%s: bad sections", what);
      sum += sections[i];
      a.bound[i] = (int)(sum < pairs ? sum : pairs);
    }
    TAGI_REQUIRE(sum == pairs, "%s: sections add up to %lld of %lld pairs", what, (long long)sum, (long long)pairs);
    TAGI_REQUIRE(B * T == 0 || (positions && freq), "%s: null pointer", what);
  }
  a.positions = positions, a.pos_bytes = pos_bytes, a.freq = freq;
  a.T = T, a.tokens = B * T, a.H = (int)H, a.G = (int)G, a.D = (int)D;
  a.L = lanes_of(D), a.TB = tokens_of(H + G, a.L);
  return TAGI_OK;
}
// four neighbouring pairs turn together or not at all, and rows end with a lane
bool vec_rows(const Args& a) { return a.D % 8 == 0 && (a.interleaved || a.pairs % 4 == 0); }

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int tagi_qk_rotary_fwd(const float* mq, const float* Sq, const tagi_heads* lq, const float* mk,
                                  const float* Sk, const tagi_heads* lk, const float* wqm, const float* wqS,
                                  const float* wkm, const float* wkS, const void* positions, int pos_bytes,
                                  int64_t axes, const int64_t* sections, const double* freq, int64_t pairs,
                                  int interleaved, float eps, float* oqm, float* oqS, float* okm, float* okS,
                                  float* inv, int64_t B, int64_t T, int64_t H, int64_t G, int64_t D,
                                  tagi_stream_t stream) {
  const char* what = "tagi_qk_rotary_fwd";
  Args a{};
  if (int rc = fill(what, a, B, T, H, G, D, positions, pos_bytes, axes, sections, freq, pairs, interleaved)) return rc;
  TAGI_REQUIRE(!!wqm == !!wqS && !!wqm == !!wkm && !!wqm == !!wkS, "%s: a norm has four weight moments", what);
  if (a.tokens == 0) return TAGI_OK;
  TAGI_REQUIRE(mq && Sq && lq && oqm && oqS && (G == 0 || (mk && Sk && lk && okm && okS)) && (!wqm || inv),
               "%s: null pointer", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_RMSNORM, s, 0.0, 16.0 * a.tokens * (H + G) * D);
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.lq = *lq;
  if (G) a.lk = *lk;
  a.wqm = wqm, a.wqS = wqS, a.wkm = wkm, a.wkS = wkS, a.eps = eps;
  a.oqm = oqm, a.oqS = oqS, a.okm = okm, a.okS = okS, a.inv = inv;
  const size_t lds = sizeof(float2) * a.TB * (a.pairs ? a.pairs : 1);
  const dim3 grid((unsigned)cdiv(a.tokens, a.TB));
  TAGI_REQUIRE((int64_t)grid.x * kThreads < (1ll << 32), "%s: too large", what);
  if (vec_rows(a))
    hipLaunchKernelGGL(qk_rotary_fwd_kernel<true>, grid, dim3(kThreads), lds, s, a);
  else
    hipLaunchKernelGGL(qk_rotary_fwd_kernel<false>, grid, dim3(kThreads), lds, s, a);
  return check_launch(what);
}

extern "C" int64_t tagi_qk_rotary_bwd_ws_bytes(int64_t B, int64_t T, int64_t H, int64_t G, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || G < 0 || D <= 0 || D > kMaxDim) return 0;
  return 16 * D * bwd_blocks(B * T, H + G, D);
}

extern "C" int tagi_qk_rotary_bwd(const float* dmq, const float* dSq, const tagi_heads* ldq, const float* dmk,
                                  const float* dSk, const tagi_heads* ldk, const float* mq, const tagi_heads* lq,
                                  const float* mk, const tagi_heads* lk, const float* inv, const float* wqm,
                                  const float* wqS, const float* wkm, const float* wkS, const void* positions,
                                  int pos_bytes, int64_t axes, const int64_t* sections, const double* freq,
                                  int64_t pairs, int interleaved, float* oqm, float* oqS, const tagi_heads* loq,
                                  float* okm, float* okS, const tagi_heads* lok, float* dwq, float* dSwq, float* dwk, float* dSwk, int64_t B, int64_t T, int64_t H,
                                  int64_t G, int64_t D, void* ws, int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_qk_rotary_bwd";
  Args a{};
  if (int rc = fill(what, a, B, T, H, G, D, positions, pos_bytes, axes, sections, freq, pairs, interleaved)) return rc;
  TAGI_REQUIRE(!!wqm == !!wqS && !!wqm == !!wkm && !!wqm == !!wkS, "%s: a norm has four weight moments", what);
  TAGI_REQUIRE(!wqm || (dwq && dSwq && dwk && dSwk), "%s: null pointer", what);
  TAGI_REQUIRE(a.tokens == 0 || (dmq && dSq && ldq && oqm && oqS && loq), "%s: null pointer", what);
  TAGI_REQUIRE(a.tokens == 0 || G == 0 || (dmk && dSk && ldk && okm && okS && lok), "%s: null pointer", what);
  TAGI_REQUIRE(a.tokens == 0 || !wqm || (mq && lq && inv && (G == 0 || (mk && lk))), "%s: null pointer", what);
  const int64_t nblk = a.tokens ? bwd_blocks(a.tokens, H + G, D) : 0;
  TAGI_REQUIRE(nblk * kThreads < (1ll << 32), "%s: too large", what);
  TAGI_REQUIRE(!wqm || !nblk || (ws && ws_bytes >= tagi_qk_rotary_bwd_ws_bytes(B, T, H, G, D)),
               "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_RMSNORM, s, 0.0, 20.0 * a.tokens * (H + G) * D);
  if (nblk) {
    a.dmq = dmq, a.dSq = dSq, a.dmk = dmk, a.dSk = dSk, a.ldq = *ldq, a.loq = *loq, a.mq = mq, a.mk = mk;
    if (G) a.ldk = *ldk, a.lok = *lok;
    if (lq) a.lq = *lq;
    if (lk) a.lk = *lk;
    a.wqm = wqm, a.wqS = wqS, a.wkm = wkm, a.wkS = wkS, a.inv = const_cast<float*>(inv);
    a.oqm = oqm, a.oqS = oqS, a.okm = okm, a.okS = okS;
    a.part = wqm ? static_cast<float*>(ws) : nullptr;
    const size_t lds = sizeof(float2) * a.TB * a.pairs + sizeof(float) * 8 * kThreads;
    if (vec_rows(a))
      hipLaunchKernelGGL(qk_rotary_bwd_kernel<true>, dim3((unsigned)nblk), dim3(kThreads), lds, s, a);
    else
      hipLaunchKernelGGL(qk_rotary_bwd_kernel<false>, dim3((unsigned)nblk), dim3(kThreads), lds, s, a);
  }
  if (wqm)  // no tokens: sums of nothing
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)(4 * D)), dim3(64), 0, s, static_cast<const float*>(ws),
                       (int)nblk, (int)D, wqS, wkS, dwq, dSwq, dwk, dSwk);
  return check_launch(what);
}
