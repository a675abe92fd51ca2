// Attention with Remax scores over sequences of any length, forward and backward, without
// storing a score.
//
// With c the scale, for query i and the keys j it sees (remax.py:33-114 over them):
//   m_ij = c q_i.k_j,  v_ij = c^2 [Sq_i.(k_j^2 + Sk_j) + q_i^2.Sk_j]
//   (mm, vm, Phi)_ij: moments of max(z_ij, 0);  mt_i = sum mm, vt_i = sum vm
//   w_ij, k_ij: weight and its relative variance from (mm, vm)_ij and (mt, vt)_i;  s_i = sum w
//   a = w / s,  mo_i = sum a v_j,  So_i = sum a^2 [k (v_j^2 + Sv_j) + Sv_j]
// The weights need the row's sums first, so a row's keys are walked twice: once for mt and vt,
// once for the outputs, which are linear in w and w^2 and are divided by s at the end.
// Backward, each product's other operand at its mean, with J_ij the Remax Jacobian:
//   e_ij = c J (dm_i.v_j),  E_ij = c^2 J^2 (dS_i.v_j^2)
//   dq = e k, dSq = E k^2;  dk = e^T q, dSk = E^T q^2;  dv = a^T dm, dSv = (a^2)^T dS
// Queries and keys are formed again from (mt, vt, s): one kernel walks keys for each query (dq),
// one walks queries for each key (dk, dv); no atomics, every sum's order is fixed by the sizes.
//
// The queries of the H / G heads that share a key head are one list of rows, token by token.
// Every product is 16 x 16 x 4 fp32 MFMAs with the walked side in the rows, so a lane holds the
// scores of one row (or key) and its sums need no exchange until the end; and the tile's
// registers are the next product's right operand as they are: lane group g holds rows 4 g + r,
// and a sum over rows may take them in any order.
#include "tagi_remax.h"

namespace tagi {
namespace {

typedef float v4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kRows = 16 * kWaves;  // rows (or keys) of a block
constexpr int kTile = 32;           // keys (or rows) walked at a time
constexpr int kMaxDim = 128;

struct Args {
  const float *mq, *Sq, *mk, *Sk, *mv, *Sv, *dm, *dS;
  tagi_heads lq, lk, lv, ld, loq, lokv;
  const void *lengths, *starts;
  int len_bytes, start_bytes, causal;
  float *mo, *So, *rows, *dmk, *dSk, *dmv, *dSv;  // mo, So: dmq, dSq in the backward
  float *sums, *parts;  // workspace: [split][2][BG][M], [split][BG][M][2 D + 1]
  int64_t B, M;         // M = T R rows of a key head
  int T, N, H, G, R, D, splits, chunk;
  float c, c2;
};

__device__ __forceinline__ v4 mfma(float a, float b, v4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int64_t int_at(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// A sequence: its keys, and where its first query stands.
struct Seq {
  int64_t start;
  int len;
};
__device__ __forceinline__ Seq sequence(const Args& A, int64_t b) {
  Seq s{0, A.N};
  if (A.lengths) {
    const int64_t n = int_at(A.lengths, A.len_bytes, b);
    s.len = (int)(n < 0 ? 0 : (n < A.N ? n : A.N));
  }
  if (A.starts) {  // positions beyond 2^32 either way see nothing, or everything, alike
    const int64_t p = int_at(A.starts, A.start_bytes, b), far = 1ll << 32;
    s.start = p < -far ? -far : (p > far ? far : p);
  }
  return s;
}
// Keys that row rho of its key head sees: those below this.
__device__ __forceinline__ int row_limit(const Args& A, const Seq& s, int64_t rho) {
  if (rho >= A.M) return 0;
  const int64_t pos = s.start + rho / A.R;
  if (pos < 0 || pos >= s.len) return 0;
  return A.causal ? (int)pos + 1 : s.len;
}
// No row of [rho0, rho0 + n) sees a key from here on.
__device__ __forceinline__ int block_limit(const Args& A, const Seq& s, int64_t rho0, int n) {
  const int64_t last = (rho0 + n < A.M ? rho0 + n : A.M) - 1;
  const int64_t first_pos = s.start + rho0 / A.R, pos = s.start + last / A.R;
  if (first_pos >= s.len || pos < 0) return 0;
  return A.causal ? (int)(pos + 1 < s.len ? pos + 1 : s.len) : s.len;
}

__device__ __forceinline__ int64_t row_at(const Args& A, const tagi_heads& l, int64_t b, int g, int64_t rho) {
  const int64_t t = rho / A.R;
  return b * l.sb + t * l.st + (g * A.R + (rho - t * A.R)) * l.sh;
}

// kTile rows of an operand into LDS, zeros where there is none: nothing behind `end` is read.
template <int DP>
__device__ __forceinline__ void stage_keys(const Args& A, const float* p, const tagi_heads& l, int64_t b, int g, int key0,
                                           int end, float (*to)[DP + 1]) {
  for (int i = threadIdx.x; i < kTile * DP; i += 64 * kWaves) {
    const int r = i / DP, d = i % DP;
    to[r][d] = key0 + r < end && d < A.D ? p[b * l.sb + (int64_t)(key0 + r) * l.st + g * l.sh + d] : 0.f;
  }
}

// The right operand of a wave's 16 rows: lane group k4 of step s holds feature 4 s + k4.
template <int DP>
__device__ __forceinline__ void load_right(const Args& A, const float* p, int64_t at, bool on, float (&x)[DP / 4]) {
  const int k4 = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int s = 0; s < DP / 4; ++s) x[s] = on && 4 * s + k4 < A.D ? p[at + 4 * s + k4] : 0.f;
}

// Score moments of 16 walked rows (LDS) against the wave's 16, queries on the right.
template <int DP>
__device__ __forceinline__ void scores(const Args& A, const float (*km)[DP + 1], const float (*kS)[DP + 1], int r0,
                                       const float (&qm)[DP / 4], const float (&qS)[DP / 4], v4& m, v4& v) {
  const int i = r0 + (threadIdx.x & 15), k4 = (threadIdx.x & 63) >> 4;
  m = v4{0, 0, 0, 0}, v = m;
#pragma unroll
  for (int s = 0; s < DP / 4; ++s) {
    const float a = km[i][4 * s + k4], b = kS[i][4 * s + k4];
    m = mfma(a, qm[s], m);
    v = mfma(fmaf(a, a, b), qS[s], v);
    v = mfma(b, qm[s] * qm[s], v);
  }
  m *= A.c, v *= A.c2;
}

// The sum over the four lane groups that share a column.
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

struct Place {
  int64_t b, bg, rho0;
  int g, split;
};
// Rows of late tokens first where they are the longest.
__device__ __forceinline__ Place place(const Args& A) {
  Place p;
  const int64_t blocks = (A.M + kRows - 1) / kRows;
  const int64_t i = A.causal ? blocks - 1 - blockIdx.x : blockIdx.x;
  p.rho0 = i * kRows;
  p.bg = (int64_t)blockIdx.y;
  p.split = blockIdx.z;
  p.b = p.bg / A.G;
  p.g = (int)(p.bg - p.b * A.G);
  return p;
}

template <int DP>
__global__ void __launch_bounds__(64 * kWaves) stats_kernel(const Args A) {
  __shared__ float km[kTile][DP + 1], kS[kTile][DP + 1];
  const Place p = place(A);
  const Seq s = sequence(A, p.b);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g4 = lane >> 4;
  const int64_t rho = p.rho0 + wave * 16 + (lane & 15);
  const int lim = row_limit(A, s, rho);
  float qm[DP / 4], qS[DP / 4];
  const int64_t at = lim ? row_at(A, A.lq, p.b, p.g, rho) : 0;
  load_right<DP>(A, A.mq, at, lim > 0, qm);
  load_right<DP>(A, A.Sq, at, lim > 0, qS);
  const int from = p.split * A.chunk, all = block_limit(A, s, p.rho0, kRows);
  const int to = all < from + A.chunk ? all : from + A.chunk;
  float mt = 0.f, vt = 0.f;
  for (int key0 = from; key0 < to; key0 += kTile) {
    __syncthreads();
    stage_keys<DP>(A, A.mk, A.lk, p.b, p.g, key0, to, km);
    stage_keys<DP>(A, A.Sk, A.lk, p.b, p.g, key0, to, kS);
    __syncthreads();
#pragma unroll
    for (int r0 = 0; r0 < kTile; r0 += 16) {
      v4 m, v;
      scores<DP>(A, km, kS, r0, qm, qS, m, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float mm, vm, cdf;
        rectify(m[r], v[r], mm, vm, cdf);
        const bool seen = key0 + r0 + 4 * g4 + r < lim;
        mt += seen ? mm : 0.f, vt += seen ? vm : 0.f;
      }
    }
  }
  mt = group_sum(mt), vt = group_sum(vt);
  if (g4 == 0 && rho < A.M) {
    float* o = A.sums + ((int64_t)p.split * 2 * A.B * A.G + p.bg) * A.M + rho;
    o[0] = mt, o[A.B * A.G * A.M] = vt;
  }
}

__device__ __forceinline__ void store_rows(const Args& A, int64_t b, int g, int64_t rho, int q, float x) {
  const int64_t t = rho / A.R, h = g * A.R + (rho - t * A.R);
  A.rows[((q * A.B + b) * A.H + h) * A.T + t] = x;
}
__device__ __forceinline__ float load_rows(const Args& A, int64_t b, int g, int64_t rho, int q) {
  const int64_t t = rho / A.R, h = g * A.R + (rho - t * A.R);
  return A.rows[((q * A.B + b) * A.H + h) * A.T + t];
}

template <int DP>
__global__ void __launch_bounds__(64 * kWaves) outputs_kernel(const Args A) {
  __shared__ float km[kTile][DP + 1], kS[kTile][DP + 1], vm_[kTile][DP + 1], vS_[kTile][DP + 1];
  const Place p = place(A);
  const Seq s = sequence(A, p.b);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g4 = lane >> 4, col = lane & 15;
  const int64_t rho = p.rho0 + wave * 16 + col;
  const int lim = row_limit(A, s, rho);
  float qm[DP / 4], qS[DP / 4];
  const int64_t at = lim ? row_at(A, A.lq, p.b, p.g, rho) : 0;
  load_right<DP>(A, A.mq, at, lim > 0, qm);
  load_right<DP>(A, A.Sq, at, lim > 0, qS);
  float mt = 0.f, vt = 0.f;
  if (rho < A.M) {
    const float* o = A.sums + p.bg * A.M + rho;
    const int64_t step = A.B * A.G * A.M;
    for (int i = 0; i < A.splits; ++i, o += 2 * step) mt += o[0], vt += o[step];
    if (p.split == 0 && g4 == 0) store_rows(A, p.b, p.g, rho, 0, mt), store_rows(A, p.b, p.g, rho, 1, vt);
  }
  const RowSums rs = row_sums(mt, vt);
  const int from = p.split * A.chunk, all = block_limit(A, s, p.rho0, kRows);
  const int to = all < from + A.chunk ? all : from + A.chunk;
  float sum = 0.f;
  v4 om[DP / 16], oS[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) om[d] = oS[d] = v4{0, 0, 0, 0};
  for (int key0 = from; key0 < to; key0 += kTile) {
    __syncthreads();
    stage_keys<DP>(A, A.mk, A.lk, p.b, p.g, key0, to, km);
    stage_keys<DP>(A, A.Sk, A.lk, p.b, p.g, key0, to, kS);
    stage_keys<DP>(A, A.mv, A.lv, p.b, p.g, key0, to, vm_);
    stage_keys<DP>(A, A.Sv, A.lv, p.b, p.g, key0, to, vS_);
    __syncthreads();
#pragma unroll
    for (int r0 = 0; r0 < kTile; r0 += 16) {
      v4 m, v;
      scores<DP>(A, km, kS, r0, qm, qS, m, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float mm, vm, cdf, w, k, xw, rw;
        rectify(m[r], v[r], mm, vm, cdf);
        weigh(mm, vm, rs, w, k, xw, rw);
        const int j = r0 + 4 * g4 + r;
        w = key0 + j < lim ? w : 0.f;
        sum += w;
        const float w2 = w * w, kw = k * w2;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const float a = vm_[j][16 * d + col], b = vS_[j][16 * d + col];
          om[d] = mfma(a, w, om[d]);
          oS[d] = mfma(fmaf(a, a, b), kw, oS[d]);
          oS[d] = mfma(b, w2, oS[d]);
        }
      }
    }
  }
  sum = group_sum(sum);
  if (rho >= A.M) return;
  if (A.splits > 1) {
    float* o = A.parts + (((int64_t)p.split * A.B * A.G + p.bg) * A.M + rho) * (2 * A.D + 1);
    if (g4 == 0) o[2 * A.D] = sum;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * d + 4 * g4 + r;
        if (f < A.D) o[f] = om[d][r], o[A.D + f] = oS[d][r];
      }
    return;
  }
  if (g4 == 0) store_rows(A, p.b, p.g, rho, 2, sum);
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor)), inv2 = inv * inv;
  const int64_t o = row_at(A, A.loq, p.b, p.g, rho);
#pragma unroll
  for (int d = 0; d < DP / 16; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * d + 4 * g4 + r;
      if (f < A.D) A.mo[o + f] = om[d][r] * inv, A.So[o + f] = oS[d][r] * inv2;
    }
}

// The splits of a row added in order; a wave to a row.
__global__ void __launch_bounds__(256) join_kernel(const Args A) {
  const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= A.B * A.G * A.M) return;
  const int64_t bg = i / A.M, rho = i - bg * A.M, b = bg / A.G, step = A.B * A.G * A.M * (2 * A.D + 1);
  const int g = (int)(bg - b * A.G), lane = threadIdx.x & 63;
  const float* p = A.parts + i * (2 * A.D + 1);
  float sum = 0.f;
  for (int k = 0; k < A.splits; ++k) sum += p[k * step + 2 * A.D];
  if (lane == 0) store_rows(A, b, g, rho, 2, sum);
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor)), inv2 = inv * inv;
  const int64_t o = row_at(A, A.loq, b, g, rho);
  for (int f = lane; f < A.D; f += 64) {
    float x = 0.f, y = 0.f;
    for (int k = 0; k < A.splits; ++k) x += p[k * step + f], y += p[k * step + A.D + f];
    A.mo[o + f] = x * inv, A.So[o + f] = y * inv2;
  }
}

// Deltas of the queries.
template <int DP>
__global__ void __launch_bounds__(64 * kWaves) dq_kernel(const Args A) {
  __shared__ float km[kTile][DP + 1], kS[kTile][DP + 1], vm_[kTile][DP + 1];
  const Place p = place(A);
  const Seq s = sequence(A, p.b);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g4 = lane >> 4, col = lane & 15;
  const int64_t rho = p.rho0 + wave * 16 + col;
  const int lim = row_limit(A, s, rho);
  float qm[DP / 4], qS[DP / 4], dm[DP / 4], dS[DP / 4];
  const int64_t at = lim ? row_at(A, A.lq, p.b, p.g, rho) : 0, dat = lim ? row_at(A, A.ld, p.b, p.g, rho) : 0;
  load_right<DP>(A, A.mq, at, lim > 0, qm);
  load_right<DP>(A, A.Sq, at, lim > 0, qS);
  load_right<DP>(A, A.dm, dat, lim > 0, dm);
  load_right<DP>(A, A.dS, dat, lim > 0, dS);
  float mt = 0.f, vt = 0.f, sum = 0.f;
  if (lim) mt = load_rows(A, p.b, p.g, rho, 0), vt = load_rows(A, p.b, p.g, rho, 1), sum = load_rows(A, p.b, p.g, rho, 2);
  const RowSums rs = row_sums(mt, vt);
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor));
  const int to = block_limit(A, s, p.rho0, kRows);
  v4 om[DP / 16], oS[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) om[d] = oS[d] = v4{0, 0, 0, 0};
  for (int key0 = 0; key0 < to; key0 += kTile) {
    __syncthreads();
    stage_keys<DP>(A, A.mk, A.lk, p.b, p.g, key0, to, km);
    stage_keys<DP>(A, A.Sk, A.lk, p.b, p.g, key0, to, kS);
    stage_keys<DP>(A, A.mv, A.lv, p.b, p.g, key0, to, vm_);
    __syncthreads();
#pragma unroll
    for (int r0 = 0; r0 < kTile; r0 += 16) {
      v4 m, v, e = {0, 0, 0, 0}, E = e;
      scores<DP>(A, km, kS, r0, qm, qS, m, v);
#pragma unroll
      for (int i = 0; i < DP / 4; ++i) {
        const float a = vm_[r0 + col][4 * i + g4];
        e = mfma(a, dm[i], e);
        E = mfma(a * a, dS[i], E);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float mm, vm, cdf, w, k, xw, rw;
        rectify(m[r], v[r], mm, vm, cdf);
        weigh(mm, vm, rs, w, k, xw, rw);
        const int j = r0 + 4 * g4 + r;
        const float J = remax_jacobian(v[r], mm, cdf, w * inv, k, xw, rw) * A.c;
        const float x = key0 + j < lim ? e[r] * J : 0.f, X = key0 + j < lim ? E[r] * J * J : 0.f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const float a = km[j][16 * d + col];
          om[d] = mfma(a, x, om[d]);
          oS[d] = mfma(a * a, X, oS[d]);
        }
      }
    }
  }
  if (rho >= A.M) return;
  const int64_t o = row_at(A, A.loq, p.b, p.g, rho);
#pragma unroll
  for (int d = 0; d < DP / 16; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * d + 4 * g4 + r;
      if (f < A.D) A.mo[o + f] = om[d][r], A.So[o + f] = oS[d][r];
    }
}

// Deltas of the keys and values: a wave holds 16 keys and walks the rows that see them.
template <int DP>
__global__ void __launch_bounds__(64 * kWaves) dkv_kernel(const Args A) {
  __shared__ float qm[kTile][DP + 1], qS[kTile][DP + 1], dm[kTile][DP + 1], dS[kTile][DP + 1];
  __shared__ float stat[5][kTile];  // inv_mt, y, c_mt, 1 / s; limit
  const int64_t bg = blockIdx.y, b = bg / A.G;
  const int g = (int)(bg - b * A.G);
  const Seq s = sequence(A, b);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g4 = lane >> 4, col = lane & 15;
  const int key0 = blockIdx.x * kRows, key = key0 + wave * 16 + col;
  float km[DP / 4], kS[DP / 4], vm_[DP / 4];
  const bool on = key < s.len;
  load_right<DP>(A, A.mk, b * A.lk.sb + (int64_t)key * A.lk.st + g * A.lk.sh, on, km);
  load_right<DP>(A, A.Sk, b * A.lk.sb + (int64_t)key * A.lk.st + g * A.lk.sh, on, kS);
  load_right<DP>(A, A.mv, b * A.lv.sb + (int64_t)key * A.lv.st + g * A.lv.sh, on, vm_);
  v4 okm[DP / 16], okS[DP / 16], ovm[DP / 16], ovS[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) okm[d] = okS[d] = ovm[d] = ovS[d] = v4{0, 0, 0, 0};
  // rows of positions [max(0, first key's if causal), len)
  int64_t first = (A.causal ? key0 : 0) - s.start, last = s.len - s.start;
  if (first < 0) first = 0;
  if (first < -s.start) first = -s.start;
  if (last > A.T) last = A.T;
  const int64_t end = key0 < s.len ? last * A.R : 0;
  for (int64_t rho0 = first * A.R; rho0 < end; rho0 += kTile) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * DP; i += 64 * kWaves) {
      const int r = i / DP, d = i % DP;
      const int64_t rho = rho0 + r;
      const bool in = rho < end && d < A.D;
      const int64_t qa = in ? row_at(A, A.lq, b, g, rho) + d : 0, da = in ? row_at(A, A.ld, b, g, rho) + d : 0;
      qm[r][d] = in ? A.mq[qa] : 0.f, qS[r][d] = in ? A.Sq[qa] : 0.f;
      dm[r][d] = in ? A.dm[da] : 0.f, dS[r][d] = in ? A.dS[da] : 0.f;
    }
    if (threadIdx.x < kTile) {
      const int64_t rho = rho0 + threadIdx.x;
      const int lim = rho < end ? row_limit(A, s, rho) : 0;
      float mt = 0.f, vt = 0.f, sum = 0.f;
      if (lim) mt = load_rows(A, b, g, rho, 0), vt = load_rows(A, b, g, rho, 1), sum = load_rows(A, b, g, rho, 2);
      const RowSums rs = row_sums(mt, vt);
      stat[0][threadIdx.x] = rs.inv_mt, stat[1][threadIdx.x] = rs.y, stat[2][threadIdx.x] = rs.c_mt;
      stat[3][threadIdx.x] = fast_rcp(fmaxf(sum, kRemaxFloor));
      stat[4][threadIdx.x] = __int_as_float(lim);
    }
    __syncthreads();
#pragma unroll
    for (int r0 = 0; r0 < kTile; r0 += 16) {
      v4 m = {0, 0, 0, 0}, v = m, e = m, E = m;
#pragma unroll
      for (int i = 0; i < DP / 4; ++i) {
        const float a = qm[r0 + col][4 * i + g4], c = qS[r0 + col][4 * i + g4];
        m = mfma(a, km[i], m);
        v = mfma(c, fmaf(km[i], km[i], kS[i]), v);
        v = mfma(a * a, kS[i], v);
        e = mfma(dm[r0 + col][4 * i + g4], vm_[i], e);
        E = mfma(dS[r0 + col][4 * i + g4], vm_[i] * vm_[i], E);
      }
      m *= A.c, v *= A.c2;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = r0 + 4 * g4 + r;
        const RowSums rs{stat[0][j], stat[1][j], stat[2][j]};
        float mm, vm, cdf, w, k, xw, rw;
        rectify(m[r], v[r], mm, vm, cdf);
        weigh(mm, vm, rs, w, k, xw, rw);
        const bool seen = key < __float_as_int(stat[4][j]);
        const float a = seen ? w * stat[3][j] : 0.f, a2 = a * a;
        const float J = remax_jacobian(v[r], mm, cdf, w * stat[3][j], k, xw, rw) * A.c;
        const float x = seen ? e[r] * J : 0.f, X = seen ? E[r] * J * J : 0.f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const float q = qm[j][16 * d + col];
          okm[d] = mfma(q, x, okm[d]);
          okS[d] = mfma(q * q, X, okS[d]);
          ovm[d] = mfma(dm[j][16 * d + col], a, ovm[d]);
          ovS[d] = mfma(dS[j][16 * d + col], a2, ovS[d]);
        }
      }
    }
  }
  if (key >= A.N) return;
  const int64_t o = b * A.lokv.sb + (int64_t)key * A.lokv.st + g * A.lokv.sh;
#pragma unroll
  for (int d = 0; d < DP / 16; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * d + 4 * g4 + r;
      if (f < A.D)
        A.dmk[o + f] = okm[d][r], A.dSk[o + f] = okS[d][r], A.dmv[o + f] = ovm[d][r], A.dSv[o + f] = ovS[d][r];
    }
}

int splits_of(int64_t B, int64_t T, int64_t N, int64_t H, int64_t G) {
  const int64_t blocks = cdiv(T * (H / G), kRows) * B * G;
  int64_t s = cdiv(1024, blocks);
  if (s > cdiv(N, 256)) s = cdiv(N, 256);
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t N, int64_t H, int64_t G, int64_t D) {
  TAGI_REQUIRE(B >= 0 && T >= 0 && N >= 0 && H > 0 && G > 0 && D > 0 && H % G == 0, "%s: bad sizes", what);
  if (D > kMaxDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxDim);
  TAGI_REQUIRE(B < 65536 && G < 65536 && B * G < 65536 && H < (1 << 20) && T < (1 << 30) && N < (1 << 30) &&
                   T * (H / G) < (1ll << 30), "%s: too large", what);
  return TAGI_OK;
}
int64_t part_floats(int64_t B, int64_t G, int64_t M, int64_t D, int splits) {
  return splits > 1 ? splits * B * G * M * (2 * D + 1) : 0;
}

#define BY_DIM(kernel, grid)                                                       \
  do {                                                                             \
    const dim3 threads(64 * kWaves);                                               \
    if (D <= 32)                                                                   \
      hipLaunchKernelGGL(kernel<32>, grid, threads, 0, s, a);                      \
    else if (D <= 64)                                                              \
      hipLaunchKernelGGL(kernel<64>, grid, threads, 0, s, a);                      \
    else                                                                           \
      hipLaunchKernelGGL(kernel<128>, grid, threads, 0, s, a);                     \
  } while (0)

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_remax_attention_fwd_ws_bytes(int64_t B, int64_t T, int64_t N, int64_t H, int64_t G,
                                                     int64_t D) {
  if (B <= 0 || T <= 0 || N < 0 || H <= 0 || G <= 0 || D <= 0 || H % G) return 0;
  const int splits = splits_of(B, T, N, H, G);
  return 4 * (2 * splits * B * H * T + part_floats(B, G, T * (H / G), D, splits));
}

extern "C" int tagi_remax_attention_fwd(const float* mq, const float* Sq, const tagi_heads* lq, const float* mk,
                                        const float* Sk, const tagi_heads* lk, const float* mv, const float* Sv,
                                        const tagi_heads* lv, const void* lengths, int len_bytes, const void* starts,
                                        int start_bytes, int causal, float* mo, float* So, float* rows, int64_t B,
                                        int64_t T, int64_t N, int64_t H, int64_t G, int64_t D, double scale, void* ws,
                                        int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_remax_attention_fwd";
  if (int rc = check_sizes(what, B, T, N, H, G, D)) return rc;
  if (B == 0 || T == 0) return TAGI_OK;
  TAGI_REQUIRE(mq && Sq && lq && mo && So && rows && (N == 0 || (mk && Sk && lk && mv && Sv && lv)),
               "%s: null pointer", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(!starts || start_bytes == 4 || start_bytes == 8, "%s: starts are int32 or int64", what);
  TAGI_REQUIRE(ws && ws_bytes >= tagi_remax_attention_fwd_ws_bytes(B, T, N, H, G, D), "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 18.0 * B * H * T * N * D * (causal && T == N ? 0.5 : 1.0),
               16.0 * D * B * (T * H + N * G));
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv, a.lq = *lq;
  if (N) a.lk = *lk, a.lv = *lv;
  a.lengths = lengths, a.len_bytes = len_bytes, a.starts = starts, a.start_bytes = start_bytes, a.causal = causal != 0;
  a.mo = mo, a.So = So, a.rows = rows, a.loq = tagi_heads{T * H * D, H * D, D};
  a.B = B, a.T = (int)T, a.N = (int)N, a.H = (int)H, a.G = (int)G, a.R = (int)(H / G), a.D = (int)D, a.M = T * (H / G);
  a.c = (float)scale, a.c2 = (float)(scale * scale);
  a.splits = splits_of(B, T, N, H, G);
  a.chunk = (int)(cdiv(cdiv(N, a.splits), kTile) * kTile);
  a.sums = static_cast<float*>(ws), a.parts = a.sums + 2 * a.splits * B * H * T;
  const dim3 grid((unsigned)cdiv(a.M, kRows), (unsigned)(B * G), (unsigned)a.splits);
  BY_DIM(stats_kernel, grid);
  BY_DIM(outputs_kernel, grid);
  if (a.splits > 1) {
    const int64_t blocks = cdiv(B * G * a.M, 4), x = blocks < (1 << 20) ? blocks : (1 << 20);
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)x, (unsigned)cdiv(blocks, x)), dim3(256), 0, s, a);
  }
  return check_launch(what);
}

extern "C" int64_t tagi_remax_attention_bwd_ws_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int tagi_remax_attention_bwd(const float* mq, const float* Sq, const tagi_heads* lq, const float* mk,
                                        const float* Sk, const tagi_heads* lk, const float* mv, const tagi_heads* lv,
                                        const float* dmo, const float* dSo, const tagi_heads* ldo, const float* rows,
                                        const void* lengths, int len_bytes, const void* starts, int start_bytes,
                                        int causal, float* dmq, float* dSq, const tagi_heads* ldq, float* dmk,
                                        float* dSk, float* dmv, float* dSv, const tagi_heads* ldkv, int64_t B,
                                        int64_t T, int64_t N, int64_t H, int64_t G, int64_t D, double scale, void* ws,
                                        int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_remax_attention_bwd";
  if (int rc = check_sizes(what, B, T, N, H, G, D)) return rc;
  if (B == 0) return TAGI_OK;
  TAGI_REQUIRE(T == 0 || (mq && Sq && lq && dmo && dSo && ldo && rows && dmq && dSq && ldq), "%s: null pointer", what);
  TAGI_REQUIRE(N == 0 || (mk && Sk && lk && mv && lv && dmk && dSk && dmv && dSv && ldkv), "%s: null pointer", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(!starts || start_bytes == 4 || start_bytes == 8, "%s: starts are int32 or int64", what);
  (void)ws, (void)ws_bytes;
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 28.0 * B * H * T * N * D * (causal && T == N ? 0.5 : 1.0),
               D * B * (24.0 * T * H + 28.0 * N * G));
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.dm = dmo, a.dS = dSo;
  if (T) a.lq = *lq, a.ld = *ldo, a.loq = *ldq;
  if (N) a.lk = *lk, a.lv = *lv, a.lokv = *ldkv;
  a.lengths = lengths, a.len_bytes = len_bytes, a.starts = starts, a.start_bytes = start_bytes, a.causal = causal != 0;
  a.mo = dmq, a.So = dSq, a.rows = const_cast<float*>(rows), a.dmk = dmk, a.dSk = dSk, a.dmv = dmv, a.dSv = dSv;
  a.B = B, a.T = (int)T, a.N = (int)N, a.H = (int)H, a.G = (int)G, a.R = (int)(H / G), a.D = (int)D, a.M = T * (H / G);
  a.c = (float)scale, a.c2 = (float)(scale * scale);
  a.splits = 1;
  if (T) {
    const dim3 grid((unsigned)cdiv(a.M, kRows), (unsigned)(B * G));
    BY_DIM(dq_kernel, grid);
  }
  if (N) {
    const dim3 grid((unsigned)cdiv(N, kRows), (unsigned)(B * G));
    BY_DIM(dkv_kernel, grid);
  }
  return check_launch(what);
}
