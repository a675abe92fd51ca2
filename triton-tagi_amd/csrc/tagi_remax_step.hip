// Remax attention of one query of every sequence over the pages of its cache.
//
// The formulas of tagi_remax_attention.hip with one row per head. A sequence's tokens are split
// over blocks; a weight needs the sums over all of them first, so there are three launches:
//   scores: the keys' pages once; moments of the rectified scores (mm, vm) to the workspace, and
//           each wave's sums of them
//   values: those sums added in order, weights, the values' pages once; each split's sums
//   join:   the splits' sums added in order and normalised
// HBM bound: the cache is read once, straight into the registers that feed the matrix cores, and
// the scores between the launches are 16 bytes a token and head beside 4 D cells a token and key
// head. The query heads that share a key head are the columns of the products, 16 at a time (a
// column that no head has is computed and dropped: 9 to 18 MFMAs for 32 features of 16 tokens take
// less time than the cells' way from HBM). Products: tagi_split_bf16.h; cells of 8 and 16 bits are
// one part, so only the queries and weights are split.
#include "tagi_kv_cache.h"
#include "tagi_remax.h"
#include "tagi_split_bf16.h"

namespace tagi {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveKeys = 256;  // most keys of a wave: their slots and scales stay in LDS

// Parts of a cell's value and of its square.
template <typename Cell>
struct CellParts;
template <>
struct CellParts<F32Cell> {
  static constexpr int one = 3, two = 3;
};
template <>
struct CellParts<Bf16Cell> {
  static constexpr int one = 1, two = 2;
};
template <>
struct CellParts<Fp8Cell> {
  static constexpr int one = 1, two = 1;
};

struct Args {
  const float *mq, *Sq;
  tagi_heads lq;
  CacheView c;
  const void* lengths;
  int len_bytes;
  float *mo, *So;
  float2* scores;  // (B, H, max_len): (mm, vm), mm = 0 where there is no token
  float* sums;     // (B, H, splits * kWaves, 2)
  float* parts;    // (B, H, splits, 2 D + 1)
  int64_t B;
  int H, R, max_len, splits, wave_keys;
  float c1, c2;
};

__device__ __forceinline__ int length_of(const Args& A, int64_t b) {
  const int64_t n = read_int(A.lengths, A.len_bytes, b), room = A.c.width * A.c.page;
  const int64_t most = room < A.max_len ? room : A.max_len;
  return (int)(n < 0 ? 0 : (n < most ? n : most));
}

// A wave's lanes have written what they read next.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// N neighbouring cells of a row as they lie in memory.
template <typename T, int N>
struct Raw {
  T x[N];
};
// Features from d on, zeros behind D. VEC: rows are whole groups of N, aligned to them.
template <bool VEC, typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* row, int d, int D) {
  Raw<T, N> r;
  if constexpr (VEC) {
    constexpr int bytes = N * sizeof(T);
    typedef uint32_t words __attribute__((ext_vector_type(bytes >= 4 ? bytes / 4 : 1)));
    if constexpr (bytes >= 4) {
      words w = {};
      if (d < D) w = *reinterpret_cast<const words*>(row + d);
      __builtin_memcpy(&r, &w, bytes);
    } else {
      uint16_t w = 0;
      if (d < D) w = *reinterpret_cast<const uint16_t*>(row + d);
      __builtin_memcpy(&r, &w, bytes);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (d + i < D)
        r.x[i] = row[d + i];
      else
        r.x[i] = T{};
    }
  }
  return r;
}
template <int N>
__device__ __forceinline__ void floats(const Raw<float, N>& r, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = r.x[i];
}
template <int N>
__device__ __forceinline__ void floats(const Raw<__bf16, N>& r, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)r.x[i];
}
template <int N>
__device__ __forceinline__ void floats(const Raw<uint8_t, N>& r, float (&x)[N]) {
  uint32_t w[(N + 3) / 4] = {};
  __builtin_memcpy(w, &r, N);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const auto p = (i & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], true)
                           : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], false);
    x[i] = p[0], x[i + 1] = p[1];
  }
}

// 2^(e - 127), e the biased exponent a row was written with
__device__ __forceinline__ float power(uint32_t e) { return __builtin_ldexpf(1.0f, (int)e - 127); }

// Slots of a wave's keys (a page lookup each), -1 where there is no token; for 8-bit cells also
// the powers of two of their means and variances.
template <typename Cell>
__device__ __forceinline__ void wave_slots(const Args& A, int64_t b, int g, int from, int to, int lane, int first_scale,
                                           int64_t* slot, float* pm, float* pS) {
  for (int i = lane; i < A.wave_keys; i += 64) {
    const int64_t row = from + i < to ? cache_row(A.c, b, from + i, g) : -1;
    slot[i] = row;
    if constexpr (sizeof(typename Cell::type) == 1) {
      const uint32_t e = row < 0 ? 0x7f7f7f7fu : reinterpret_cast<const uint32_t*>(A.c.scales)[row];
      pm[i] = power((e >> (8 * first_scale)) & 255), pS[i] = power((e >> (8 * first_scale + 8)) & 255);
    }
  }
  wave_sync();
}

// First of the eight features that lane group k8 brings to step s. Where 64 features are 64
// bytes, two steps share a lane's 16 bytes.
template <typename Cell, int DP>
__device__ __forceinline__ int feature(int s, int k8) {
  if constexpr (sizeof(typename Cell::type) == 1 && DP >= 64) return 64 * (s >> 1) + 16 * k8 + 8 * (s & 1);
  return 32 * s + 8 * k8;
}

// Blocks of a CU: the operands of long heads in several parts, or gathered cell by cell, take a
// SIMD's registers for one wave.
template <typename Cell, int DP, bool VEC>
constexpr int blocks_of() {
  return DP == 128 && !(VEC && sizeof(typename Cell::type) == 1) ? 1 : 2;
}

// HT query heads at a time: 4 of the 16 columns where a key head has no more (a wave's tables in
// LDS are a quarter, so a CU holds two blocks).
template <typename Cell, int DP, bool VEC, int HT>
__global__ void __launch_bounds__(kThreads, (blocks_of<Cell, DP, VEC>())) scores_kernel(const Args A) {
  typedef typename Cell::type T;
  constexpr int S = DP / 32, P1 = CellParts<Cell>::one, P2 = CellParts<Cell>::two;
  constexpr bool scaled_rows = sizeof(T) == 1;
  constexpr int kRow = 64 + 4;  // floats of a head's 64 scores, banks apart
  __shared__ int64_t slots[kWaves][kWaveKeys];
  __shared__ float powers[kWaves][scaled_rows ? 2 * kWaveKeys : 1];
  __shared__ __align__(16) float tile[kWaves][2][HT * kRow];
  const int64_t b = blockIdx.z;
  const int g = blockIdx.y, D = A.c.D, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, k8 = lane >> 4;
  const int len = length_of(A, b), from = ((int)blockIdx.x * kWaves + wave) * A.wave_keys;
  const int to = from + A.wave_keys < len ? from + A.wave_keys : len;
  int64_t* slot = slots[wave];
  float *pm = powers[wave], *pS = pm + (scaled_rows ? kWaveKeys : 0);
  if (from < to) wave_slots<Cell>(A, b, g, from, to, lane, 0, slot, pm, pS);
  for (int r0 = 0; r0 < A.R; r0 += HT) {
    const int n = A.R - r0 < HT ? A.R - r0 : HT;
    const int64_t h = b * A.H + g * A.R + r0;
    float mt[HT] = {}, vt[HT] = {};
    if (from < to) {
      Parts<3> q[S], Q[S], P[S];  // q, Sq, Sq + q^2, scaled
      const int64_t qa = b * A.lq.sb + (int64_t)(g * A.R + r0 + (col < n ? col : n - 1)) * A.lq.sh;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float x[8], X[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = feature<Cell, DP>(s, k8) + i;
          x[i] = d < D ? A.mq[qa + d] * A.c1 : 0.f, X[i] = d < D ? A.Sq[qa + d] * A.c2 : 0.f;
          y[i] = fmaf(x[i], x[i], X[i]);
        }
        q[s] = split<3>(x), Q[s] = split<3>(X), P[s] = split<3>(y);
      }
      const int tiles = (to - from + 15) / 16;
      Raw<T, 8> km[S], kS[S];
      auto fetch = [&](int t) {
        const int64_t row = slot[16 * t + col], at = (row < 0 ? 0 : row) * D;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const int d = feature<Cell, DP>(s, k8);
          km[s] = load_raw<VEC, T, 8>(static_cast<const T*>(A.c.km) + at, d, D);
          kS[s] = load_raw<VEC, T, 8>(static_cast<const T*>(A.c.kS) + at, d, D);
        }
      };
      fetch(0);
      for (int t = 0; t < tiles; ++t) {
        acc4 m = {0, 0, 0, 0}, v = m, w = m;
        Raw<T, 8> am[S], aS[S];
#pragma unroll
        for (int s = 0; s < S; ++s) am[s] = km[s], aS[s] = kS[s];
        if (t + 1 < tiles) fetch(t + 1);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          float x[8], y[8];
          floats(am[s], x);
          m = mma(split<P1>(x), q[s], m);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= x[i];
          floats(aS[s], y);
          if constexpr (scaled_rows) {
            v = mma(split<P2>(x), Q[s], v);
            w = mma(split<P1>(y), P[s], w);
          } else {
            v = mma(split<P2>(x), Q[s], v);
            v = mma(split<P1>(y), P[s], v);
          }
        }
        const int at = 16 * (t & 3) + 4 * k8;  // of the 64 keys under way
        if constexpr (scaled_rows) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float a = pm[16 * t + 4 * k8 + r], s = pS[16 * t + 4 * k8 + r];
            m[r] *= a;
            v[r] = fmaf(v[r] * a, a, w[r] * s);
          }
        }
        if (col < n) {
          *reinterpret_cast<acc4*>(&tile[wave][0][col * kRow + at]) = m;
          *reinterpret_cast<acc4*>(&tile[wave][1][col * kRow + at]) = v;
        }
        if ((t & 3) != 3 && t + 1 < tiles) continue;
        // 64 keys: a lane to a key, the heads one after another
        wave_sync();
        const int key = (t & ~3) * 16 + lane;
        const bool on = from + key < to, there = on && slot[key < A.wave_keys ? key : 0] >= 0;
#pragma unroll
        for (int r = 0; r < HT; ++r) {
          if (r >= n) continue;
          Rectified z = rectify(tile[wave][0][r * kRow + lane], tile[wave][1][r * kRow + lane]);
          if (!there) z.mm = z.vm = 0.f;
          if (on) A.scores[(h + r) * A.max_len + from + key] = make_float2(z.mm, z.vm);
          mt[r] += z.mm, vt[r] += z.vm;
        }
        wave_sync();
      }
    }
#pragma unroll
    for (int r = 0; r < HT; ++r) {
      if (r >= n) continue;
      const float x = wave_sum(mt[r]), y = wave_sum(vt[r]);
      if (lane == 0) {
        float* o = A.sums + ((h + r) * A.splits * kWaves + (int)blockIdx.x * kWaves + wave) * 2;
        o[0] = x, o[1] = y;
      }
    }
  }
}

// Lane (r, k8) of a wave brings the features ND r .. ND r + ND - 1 (ND = DP / 16) of keys 8 k8 ..
// 8 k8 + 7 of every 32: the j-th of them, over the eight keys, is its share of a product whose rows
// are the features ND r + j. So a load covers whole rows and no value moves between lanes.
template <typename Cell, int DP, bool VEC, int HT>
__global__ void __launch_bounds__(kThreads, (HT == 16 ? 1 : blocks_of<Cell, DP, VEC>())) values_kernel(const Args A) {
  typedef typename Cell::type T;
  constexpr int ND = DP / 16, P1 = CellParts<Cell>::one, P2 = CellParts<Cell>::two;
  constexpr bool scaled_rows = sizeof(T) == 1;
  constexpr int kRow = 64 + 8;  // keys of a head's weights, banks apart
  constexpr int kPart = HT * kRow;
  __shared__ int64_t slots[kWaves][kWaveKeys];
  __shared__ float powers[kWaves][scaled_rows ? 2 * kWaveKeys : 1];
  __shared__ __align__(16) __bf16 weights[kWaves][9 * kPart];  // [w, kw, kw + w^2][part][head][key]
  __shared__ RowSums row[HT];
  __shared__ float totals[kWaves][HT];
  const int64_t b = blockIdx.z;
  const int g = blockIdx.y, D = A.c.D, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, k8 = lane >> 4;
  const int len = length_of(A, b), block_from = (int)blockIdx.x * kWaves * A.wave_keys;
  if (block_from >= len && blockIdx.x > 0) return;  // the join adds what the length reaches
  const int from = block_from + wave * A.wave_keys;
  const int to = from + A.wave_keys < len ? from + A.wave_keys : len;
  int64_t* slot = slots[wave];
  float *pm = powers[wave], *pS = pm + (scaled_rows ? kWaveKeys : 0);
  if (from < to) wave_slots<Cell>(A, b, g, from, to, lane, 2, slot, pm, pS);
  for (int r0 = 0; r0 < A.R; r0 += HT) {
    const int n = A.R - r0 < HT ? A.R - r0 : HT;
    const int64_t h = b * A.H + g * A.R + r0;
    __syncthreads();  // the heads before are done with the sums and weights
    for (int r = wave; r < n; r += kWaves) {
      const float* p = A.sums + (h + r) * A.splits * kWaves * 2;
      float mt = 0.f, vt = 0.f;
      for (int i = lane; i < A.splits * kWaves; i += 64) mt += p[2 * i], vt += p[2 * i + 1];
      mt = wave_sum(mt), vt = wave_sum(vt);
      if (lane == 0) row[r] = row_sums(mt, vt);
    }
    __syncthreads();
    acc4 om[ND], oS[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) om[j] = oS[j] = acc4{0, 0, 0, 0};
    float total[HT] = {};
    __bf16* W = weights[wave];
    for (int key0 = from; key0 < to; key0 += 64) {
      const int i0 = key0 - from;
      {
        // a lane to a key
        const bool on = key0 + lane < to;
        float a = 1.f, s = 1.f;
        if constexpr (scaled_rows) a = pm[i0 + lane], s = pS[i0 + lane];
#pragma unroll
        for (int r = 0; r < HT; ++r) {
          if (r >= n) continue;
          float w = 0.f, k = 0.f;
          const float2 x = on ? A.scores[(h + r) * A.max_len + key0 + lane] : make_float2(0.f, 0.f);
          if (x.x > 0.f) {
            const Weight o = weigh(Rectified{x.x, x.y, 0.f, 0.f}, row[r]);
            w = o.w, k = o.k;
          }
          total[r] += w;
          // the powers of two of the rows go into their weights
          const float w2 = w * w, kw = k * w2;
          const float y[3] = {w * a, kw * a * a, (kw + w2) * s};
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            float rest = y[q];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
              const __bf16 part = (__bf16)rest;
              W[(3 * q + p) * kPart + r * kRow + lane] = part;
              rest -= (float)part;
            }
          }
        }
      }
      wave_sync();
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        if (key0 + 32 * half >= to) break;
        Raw<T, ND> am[8], aS[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t at = slot[i0 + 32 * half + 8 * k8 + i], o = (at < 0 ? 0 : at) * D;
          am[i] = load_raw<VEC, T, ND>(static_cast<const T*>(A.c.vm) + o, ND * col, D);
          aS[i] = load_raw<VEC, T, ND>(static_cast<const T*>(A.c.vS) + o, ND * col, D);
        }
        Parts<3> w[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            w[q].p[p] = *reinterpret_cast<const bf8*>(W + (3 * q + p) * kPart + (col < n ? col : n - 1) * kRow + 32 * half + 8 * k8);
        float x[8][ND], y[8][ND];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          floats(am[i], x[i]), floats(aS[i], y[i]);
          // what is not there weighs nothing, whatever its slot holds
          if (slot[i0 + 32 * half + 8 * k8 + i] < 0) {
#pragma unroll
            for (int j = 0; j < ND; ++j) x[i][j] = y[i][j] = 0.f;
          }
        }
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          float e[8], f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = x[i][j], f[i] = y[i][j];
          om[j] = mma(split<P1>(e), w[0], om[j]);
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] *= e[i];
          oS[j] = mma(split<P2>(e), w[1], oS[j]);
          oS[j] = mma(split<P1>(f), w[2], oS[j]);
        }
      }
      wave_sync();
    }
#pragma unroll
    for (int r = 0; r < HT; ++r) {
      if (r >= n) continue;
      const float x = wave_sum(total[r]);
      if (lane == 0) totals[wave][r] = x;
    }
    // the waves' sums in order, means and variances in turn, through the weights' LDS
    float* part = A.parts + (h * A.splits + blockIdx.x) * (2 * D + 1);
    const int64_t step = (int64_t)A.splits * (2 * D + 1);
    float* red = reinterpret_cast<float*>(&weights[0][0]);  // [wave][feature][head]
    static_assert(sizeof(weights) >= sizeof(float) * kWaves * HT * DP, "the sums fit the weights' LDS");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col < HT) red[(wave * DP + ND * (4 * k8 + r) + j) * HT + col] = k == 0 ? om[j][r] : oS[j][r];
      __syncthreads();
      for (int i = threadIdx.x; i < n * D; i += kThreads) {
        const int r = i / D, f = i - r * D;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += red[(w * DP + f) * HT + r];
        part[r * step + k * D + f] = x;
      }
    }
    if ((int)threadIdx.x < n) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x += totals[w][threadIdx.x];
      part[threadIdx.x * step + 2 * D] = x;
    }
  }
}

// A wave to a query head: the splits that its sequence's length reaches, in order.
__global__ void __launch_bounds__(kThreads) join_kernel(const Args A) {
  const int64_t h = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (h >= A.B * A.H) return;
  const int D = A.c.D, step = 2 * D + 1, block_keys = kWaves * A.wave_keys;
  const int len = length_of(A, h / A.H), n = len <= block_keys ? 1 : (len + block_keys - 1) / block_keys;
  const float* p = A.parts + h * A.splits * step;
  float sum = 0.f;
  for (int k = 0; k < n; ++k) sum += p[k * step + 2 * D];
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor)), inv2 = inv * inv;
  for (int f = threadIdx.x & 63; f < D; f += 64) {
    float x = 0.f, y = 0.f;
    for (int k = 0; k < n; ++k) x += p[k * step + f], y += p[k * step + D + f];
    A.mo[h * D + f] = x * inv, A.So[h * D + f] = y * inv2;
  }
}

// Keys of a wave: as many as leave a few blocks for each of the 256 CUs.
int wave_keys_of(int64_t B, int64_t G, int64_t max_len) {
  int keys = kWaveKeys;
  while (keys > 64 && B * G * cdiv(max_len, kWaves * keys) < 1024) keys /= 2;
  return keys;
}
int64_t splits_of(int64_t B, int64_t G, int64_t max_len) {
  const int64_t s = cdiv(max_len, kWaves * wave_keys_of(B, G, max_len));
  return s < 1 ? 1 : s;
}
int64_t score_floats(int64_t B, int64_t H, int64_t max_len) { return 2 * B * H * max_len; }

template <typename Cell, int DP, bool VEC, int HT>
void launch(const Args& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((scores_kernel<Cell, DP, VEC, HT>), grid, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((values_kernel<Cell, DP, VEC, HT>), grid, dim3(kThreads), 0, s, a);
}
template <typename Cell, int DP>
void launch_heads(const Args& a, bool vec, dim3 grid, hipStream_t s) {
  if (a.R <= 4)
    vec ? launch<Cell, DP, true, 4>(a, grid, s) : launch<Cell, DP, false, 4>(a, grid, s);
  else
    vec ? launch<Cell, DP, true, 16>(a, grid, s) : launch<Cell, DP, false, 16>(a, grid, s);
}
template <typename Cell>
void launch_dim(const Args& a, bool vec, dim3 grid, hipStream_t s) {
  if (a.c.D <= 32)
    launch_heads<Cell, 32>(a, vec, grid, s);
  else if (a.c.D <= 64)
    launch_heads<Cell, 64>(a, vec, grid, s);
  else
    launch_heads<Cell, 128>(a, vec, grid, s);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_remax_attention_step_ws_bytes(int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_len) {
  if (B <= 0 || H <= 0 || G <= 0 || D <= 0 || max_len < 0) return 0;
  return 4 * (score_floats(B, H, max_len) + B * H * splits_of(B, G, max_len) * (2 * kWaves + 2 * D + 1));
}

extern "C" int tagi_remax_attention_step(const float* mq, const float* Sq, const tagi_heads* lq,
                                         const tagi_kv_cache* cache, const int32_t* table, int64_t width,
                                         const void* lengths, int len_bytes, float* mo, float* So, int64_t B, int64_t H,
                                         int64_t max_len, double scale, void* ws, int64_t ws_bytes,
                                         tagi_stream_t stream) {
  const char* what = "tagi_remax_attention_step";
  Args a{};
  if (int rc = cache_view(what, &a.c, cache, table, width, B)) return rc;
  const int64_t G = a.c.G, D = a.c.D;
  TAGI_REQUIRE(H > 0 && H % G == 0 && max_len >= 0, "%s: bad sizes", what);
  TAGI_REQUIRE(B < 65536 && G < 65536 && H < (1 << 20) && max_len < (1 << 30), "%s: too large", what);
  if (B == 0) return TAGI_OK;
  TAGI_REQUIRE(mq && Sq && lq && mo && So, "%s: null pointer", what);
  TAGI_REQUIRE(lengths && (len_bytes == 4 || len_bytes == 8), "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(ws && ws_bytes >= tagi_remax_attention_step_ws_bytes(B, H, G, D, max_len), "%s: workspace too small",
               what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 12.0 * B * H * max_len * D, 4.0 * cell_bytes(cache->type) * B * G * max_len * D);
  a.mq = mq, a.Sq = Sq, a.lq = *lq, a.lengths = lengths, a.len_bytes = len_bytes, a.mo = mo, a.So = So;
  a.B = B, a.H = (int)H, a.R = (int)(H / G), a.max_len = (int)(cache->pages ? max_len : 0);
  a.wave_keys = wave_keys_of(B, G, max_len), a.splits = (int)splits_of(B, G, max_len);
  a.c1 = (float)scale, a.c2 = (float)(scale * scale);
  a.scores = static_cast<float2*>(ws);
  a.sums = static_cast<float*>(ws) + score_floats(B, H, max_len), a.parts = a.sums + 2 * kWaves * B * H * a.splits;
  // a lane's cells in whole words: eight features (fewer in the values of short heads), 16-byte rows
  const int size = cell_bytes((int)cache->type), group = size == 1 && D > 32 ? 16 : 8;
  const uintptr_t all = (uintptr_t)a.c.km | (uintptr_t)a.c.kS | (uintptr_t)a.c.vm | (uintptr_t)a.c.vS;
  const bool vec = D % group == 0 && all % 16 == 0;
  const dim3 grid((unsigned)a.splits, (unsigned)G, (unsigned)B);
  if (cache->type == CELL_F32)
    launch_dim<F32Cell>(a, vec, grid, s);
  else if (cache->type == CELL_BF16)
    launch_dim<Bf16Cell>(a, vec, grid, s);
  else
    launch_dim<Fp8Cell>(a, vec, grid, s);
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)cdiv(B * H, kWaves)), dim3(kThreads), 0, s, a);
  return check_launch(what);
}
