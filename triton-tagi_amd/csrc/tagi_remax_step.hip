// Remax attention of one query of every sequence over the pages of its cache.
//
// The formulas of tagi_remax_attention.hip with one row per head. A sequence's tokens are split
// over blocks; a weight needs the sums over all of them first, so there are three launches (one where
// a block holds a sequence and every block a CU):
//   scores: the keys' pages once; moments of the rectified scores (mm, vm) to the workspace, and
//           each wave's sums of them
//   values: those sums added in order, weights, the values' pages once; each split's sums
//   join:   the splits' sums added in order and normalised
// HBM bound: the cache is read once, straight into the registers that feed the matrix cores, and
// the scores between the launches are 16 bytes a token and head beside 4 D cells a token and key
// head. Cells of 8 and 16 bits are one bf16 part (tagi_split_bf16.h; their squares one and two),
// so only the queries and weights are split. The query heads that share a key head are the columns
// of the products. Up to four of them take all 16 columns with their three parts, four for each (the
// last four are zeros), and a product of all parts is one MFMA instead of three; more than four take
// 16 columns at a time, part after part (16 sequences of 16384 tokens, 8 key heads of 128 in e4m3,
// four query heads to each: 288 us, 395 as 16 columns; five: 404, 441 as four and one).
//
// Measured: the same in bf16, one query head to a key head, 407 us for 2.15 GB, 5.3 TB/s; in e4m3
// 265 us for 1.08 GB, 4.1 TB/s: there a cell's way to bf16, its square and the scores' moments (800
// vector instructions for a wave's 64 keys) are as long as its way from HBM. Loads are counted:
// behind a branch each tile waited for all of them (611 us of 16 x 28672 tokens, 492 without).
#include "tagi_kv_cache.h"
#include "tagi_remax.h"
#include "tagi_split_bf16.h"

namespace tagi {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
// Most keys of a wave: their slots and scales stay in LDS. A block's way to its first tile (lengths,
// pages, queries) is shared by more of them: 16 x 28672 tokens 511 us at 256, 492 at 512.
constexpr int kWaveKeys = 512;

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
  static constexpr int words = (N * (int)sizeof(T) + 3) / 4;
  uint32_t w[words];
};
// A GPU's memory, said so: of two pointers to choose from the compiler would not know it.
template <typename T>
__device__ __forceinline__ T load_global(const void* p) {
  return *(const __attribute__((address_space(1))) T*)(p);
}
// Features from d on. VEC: rows are whole groups of N, aligned to them, and behind D the row's first
// stand: they meet a query's zeros (a row with a NaN there has NaN scores as it is) or go to sums
// that nobody reads. Else zeros.
template <bool VEC, typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* row, int d, int D) {
  Raw<T, N> r;
  if constexpr (VEC && N * sizeof(T) >= 4) {
    typedef uint32_t words __attribute__((ext_vector_type(Raw<T, N>::words)));
    const words w = load_global<words>(row + (d < D ? d : 0));
#pragma unroll
    for (int i = 0; i < Raw<T, N>::words; ++i) r.w[i] = w[i];
  } else if constexpr (VEC) {
    r.w[0] = load_global<uint16_t>(row + (d < D ? d : 0));
  } else {
#pragma unroll
    for (int i = 0; i < Raw<T, N>::words; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t x = 0;
      if (d + i < D) {
        if constexpr (sizeof(T) == 4) x = load_global<uint32_t>(row + d + i);
        if constexpr (sizeof(T) == 2) x = load_global<uint16_t>(row + d + i);
        if constexpr (sizeof(T) == 1) x = load_global<uint8_t>(row + d + i);
      }
      constexpr int per = 4 / sizeof(T);
      r.w[i / per] |= x << (32 / per * (i % per));
    }
  }
  return r;
}
// Eight of them.
template <typename T, int N>
__device__ __forceinline__ Raw<T, 8> eight(const Raw<T, N>& r, int first) {
  Raw<T, 8> o;
#pragma unroll
  for (int i = 0; i < Raw<T, 8>::words; ++i) o.w[i] = r.w[first * (int)sizeof(T) / 4 + i];
  return o;
}

// Eight cells as bf16 parts, and their squares.
__device__ __forceinline__ Parts<3> parts_of(const Raw<float, 8>& r) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i]);
  return split<3>(x);
}
__device__ __forceinline__ Parts<3> squares_of(const Raw<float, 8>& r) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i]) * __uint_as_float(r.w[i]);
  return split<3>(x);
}
__device__ __forceinline__ Parts<1> parts_of(const Raw<__bf16, 8>& r) {
  Parts<1> o;
  __builtin_memcpy(&o.p[0], r.w, 16);
  return o;
}
__device__ __forceinline__ Parts<2> squares_of(const Raw<__bf16, 8>& r) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float(r.w[i] << 16), hi = __uint_as_float(r.w[i] & 0xffff0000u);
    x[2 * i] = lo * lo, x[2 * i + 1] = hi * hi;
  }
  return split<2>(x);
}
__device__ __forceinline__ Parts<1> parts_of(const Raw<uint8_t, 8>& r) {
  bf2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[i / 2], 1.0f, true)
                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[i / 2], 1.0f, false);
  Parts<1> o;
  __builtin_memcpy(&o.p[0], x, 16);
  return o;
}
__device__ __forceinline__ Parts<1> squares_of(const Raw<uint8_t, 8>& r) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto p = (i & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[i / 2], true)
                           : __builtin_amdgcn_cvt_pk_f32_fp8((int)r.w[i / 2], false);
    x[2 * i] = p[0] * p[0], x[2 * i + 1] = p[1] * p[1];
  }
  return split<1>(x);
}

// Eight rows of N cells as N columns of eight.
template <int N>
__device__ __forceinline__ void turn(const Raw<float, N> (&a)[8], Raw<float, 8> (&o)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[j].w[i] = a[i].w[j];
}
template <int N>
__device__ __forceinline__ void turn(const Raw<__bf16, N> (&a)[8], Raw<__bf16, 8> (&o)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t x = a[i].w[j / 2], y = a[i + 1].w[j / 2];
      o[j].w[i / 2] = __builtin_amdgcn_perm(y, x, 0x05040100u);
      o[j + 1].w[i / 2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    }
}
template <int N>
__device__ __forceinline__ void turn(const Raw<uint8_t, N> (&a)[8], Raw<uint8_t, 8> (&o)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 4)
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const uint32_t x0 = a[i].w[j / 4], x1 = a[i + 1].w[j / 4], x2 = a[i + 2].w[j / 4], x3 = a[i + 3].w[j / 4];
      const uint32_t l0 = __builtin_amdgcn_perm(x1, x0, 0x05010400u), l1 = __builtin_amdgcn_perm(x3, x2, 0x05010400u);
      o[j].w[i / 4] = __builtin_amdgcn_perm(l1, l0, 0x05040100u);
      o[j + 1].w[i / 4] = __builtin_amdgcn_perm(l1, l0, 0x07060302u);
      if (j + 2 < N) {
        const uint32_t h0 = __builtin_amdgcn_perm(x1, x0, 0x07030602u), h1 = __builtin_amdgcn_perm(x3, x2, 0x07030602u);
        o[j + 2].w[i / 4] = __builtin_amdgcn_perm(h1, h0, 0x05040100u);
        o[j + 3].w[i / 4] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
      }
    }
}

// The right operand of HT heads: column 4 p + r is part p of head r, or column r of each part.
template <int HT>
struct Right {
  bf8 p[HT == 4 ? 1 : 3];
};
template <int HT, int PA>
__device__ __forceinline__ acc4 mul(const Parts<PA>& a, const Right<HT>& b, acc4 c) {
  if constexpr (HT == 4) {
#pragma unroll
    for (int i = PA - 1; i >= 0; --i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[0], c, 0, 0, 0);
    return c;
  } else {
    Parts<3> x;
#pragma unroll
    for (int i = 0; i < 3; ++i) x.p[i] = b.p[i];
    return mma(a, x, c);
  }
}
// This lane's column of it.
template <int HT>
__device__ __forceinline__ Right<HT> right_of(const float (&x)[8], int col) {
  const Parts<3> s = split<3>(x);
  Right<HT> o;
  if constexpr (HT == 4)
    o.p[0] = col < 4 ? s.p[0] : (col < 8 ? s.p[1] : (col < 12 ? s.p[2] : bf8{}));
  else
    o.p[0] = s.p[0], o.p[1] = s.p[1], o.p[2] = s.p[2];
  return o;
}
// A row's sum over the columns of a head's parts, in every one of them.
template <int HT>
__device__ __forceinline__ float over_parts(float x) {
  if constexpr (HT == 4) {
    // row_ror: 8 columns on, then 4
    x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x124, 0xf, 0xf, true));
  }
  return x;
}

// Eight features of a query from d on, any behind D. Loads without a branch between them: all are in
// flight at once.
__device__ __forceinline__ void load_query(const float* p, int d, int D, float (&x)[8]) {
  const bool whole = D % 8 == 0;
  if (whole) {
    const f4u a = load4(p + (d < D ? d : 0)), b = load4(p + (d < D ? d : 0) + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < 4 ? a[i & 3] : b[i & 3];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[d + i < D ? d + i : 0];
  }
}

// What a row holds that is not there.
__device__ const uint4 kNothing[32] = {};

// 2^(e - 127), e the biased exponent a row was written with
__device__ __forceinline__ float power(uint32_t e) { return __builtin_ldexpf(1.0f, (int)e - 127); }

// Where a wave's keys begin in the pools (a page lookup each), -1 where there is no token; for 8-bit cells also
// the powers of two of their means and variances.
template <typename Cell>
__device__ __forceinline__ void wave_slots(const Args& A, int64_t b, int g, int from, int to, int lane, int first_scale,
                                           int64_t* slot, float* pm, float* pS) {
  for (int i = lane; i < A.wave_keys; i += 64) {
    const int64_t row = from + i < to ? cache_row(A.c, b, from + i, g) : -1;
    slot[i] = row < 0 ? -1 : row * A.c.D;
    if constexpr (sizeof(typename Cell::type) == 1) {
      const uint32_t e = row < 0 ? 0x7f7f7f7fu : reinterpret_cast<const uint32_t*>(A.c.scales)[row];
      pm[i] = power((e >> (8 * first_scale)) & 255), pS[i] = power((e >> (8 * first_scale + 8)) & 255);
    }
  }
  wave_sync();
}

// Eight features of every 32 to a lane group; where 64 features are 64 bytes, two steps share a
// lane's 16 bytes.
template <typename T, int DP>
constexpr int group_of() {
  return sizeof(T) == 1 && DP >= 64 ? 16 : 8;
}
template <typename T, int DP>
__device__ __forceinline__ int feature(int s, int k8) {
  constexpr int N = group_of<T, DP>(), per = N / 8;
  return 4 * N * (s / per) + N * k8 + 8 * (s % per);
}

// Blocks of a CU: fp32 cells of long heads, and 16 columns of three parts, take a SIMD's registers
// for one wave; so do cells gathered one by one.
template <typename Cell, int DP, bool VEC, int HT>
constexpr int blocks_of() {
  if (DP < 128) return VEC || HT == 4 ? 2 : 1;
  return VEC && HT == 4 && sizeof(typename Cell::type) < 4 ? 2 : 1;
}

// HT query heads at a time.
template <typename Cell, int DP, bool VEC, int HT>
__device__ __forceinline__ void scores_of(const Args& A) {
  typedef typename Cell::type T;
  constexpr int S = DP / 32, N = group_of<T, DP>(), L = DP / (4 * N);  // L loads of N features
  constexpr int F = VEC && HT == 4 ? 4 / sizeof(T) : 1;                // tiles in flight
  constexpr bool scaled_rows = sizeof(T) == 1;
  constexpr int kRow = 64 + 4;  // floats of a head's 64 scores, banks apart
  __shared__ int64_t slots[kWaves][kWaveKeys];
  __shared__ float powers[kWaves][scaled_rows ? 2 * kWaveKeys : 1];
  __shared__ __align__(16) float tile[kWaves][2][HT * kRow];
  const int64_t b = blockIdx.z;
  const int g = blockIdx.y, D = A.c.D, wave = threadIdx.x >> 6;
  const int len = length_of(A, b), from = ((int)blockIdx.x * kWaves + wave) * A.wave_keys;
  const int to = from + A.wave_keys < len ? from + A.wave_keys : len;
  int64_t* slot = slots[wave];
  float *pm = powers[wave], *pS = pm + (scaled_rows ? kWaveKeys : 0);
  for (int r0 = 0; r0 < A.R; r0 += HT) {
    int lane = threadIdx.x & 63;
    // addresses are formed for each turn: where one turn takes the registers they would wait in scratch memory
    if constexpr (HT > 4) asm volatile("" : "+v"(lane));
    const int col = lane & 15, k8 = lane >> 4, head = HT == 4 ? col & 3 : col;
    const int n = A.R - r0 < HT ? A.R - r0 : HT;
    const int64_t h = b * A.H + g * A.R + r0;
    float mt[HT] = {}, vt[HT] = {};
    if (from < to) {
      Right<HT> q[S], Q[S], P[S];  // q, Sq, Sq + q^2, scaled
      const int64_t qa = b * A.lq.sb + (int64_t)(g * A.R + r0 + (head < n ? head : n - 1)) * A.lq.sh;
      float x[S][8], X[S][8];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        load_query(A.mq + qa, feature<T, DP>(s, k8), D, x[s]);
        load_query(A.Sq + qa, feature<T, DP>(s, k8), D, X[s]);
      }
      // while the queries are on their way
      if (r0 == 0) wave_slots<Cell>(A, b, g, from, to, lane, 0, slot, pm, pS);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool on = feature<T, DP>(s, k8) + i < D;
          x[s][i] = on ? x[s][i] * A.c1 : 0.f, X[s][i] = on ? X[s][i] * A.c2 : 0.f;
          y[i] = fmaf(x[s][i], x[s][i], X[s][i]);
        }
        q[s] = right_of<HT>(x[s], col), Q[s] = right_of<HT>(X[s], col), P[s] = right_of<HT>(y, col);
      }
      // whole groups of four tiles, and every fetch is made (the last ones again): what waits for a
      // load counts those behind it, and behind a branch it would have to wait for all
      const int tiles = (to - from + 63) / 64 * 4;
      Raw<T, N> km[F][L], kS[F][L];
      auto fetch = [&](int t, int f) {
        const int64_t row = slot[16 * t + col], at = row < 0 ? 0 : row;
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const int d = 4 * N * l + N * k8;
          km[f][l] = load_raw<VEC, T, N>(static_cast<const T*>(A.c.km) + at, d, D);
          kS[f][l] = load_raw<VEC, T, N>(static_cast<const T*>(A.c.kS) + at, d, D);
        }
      };
#pragma unroll
      for (int f = 0; f < F; ++f) {
        fetch(f, f);
        __builtin_amdgcn_sched_barrier(0);  // in this order: it is what the waits count
      }
      for (int t0 = 0; t0 < tiles; t0 += 4) {  // 64 keys
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t = t0 + u, f = u % F;
          acc4 m = {0, 0, 0, 0}, v = m, w = m;
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const Raw<T, 8> x = eight(km[f][8 * s / N], 8 * s % N), y = eight(kS[f][8 * s / N], 8 * s % N);
            m = mul<HT>(parts_of(x), q[s], m);
            v = mul<HT>(squares_of(x), Q[s], v);
            if constexpr (scaled_rows)
              w = mul<HT>(parts_of(y), P[s], w);
            else
              v = mul<HT>(parts_of(y), P[s], v);
          }
          fetch(t + F < tiles ? t + F : t, f);
          if constexpr (scaled_rows) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float a = pm[16 * t + 4 * k8 + r], s = pS[16 * t + 4 * k8 + r];
              m[r] *= a;
              v[r] = fmaf(v[r] * a, a, w[r] * s);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) m[r] = over_parts<HT>(m[r]), v[r] = over_parts<HT>(v[r]);
          if (col < n) {
            *reinterpret_cast<acc4*>(&tile[wave][0][col * kRow + 16 * u + 4 * k8]) = m;
            *reinterpret_cast<acc4*>(&tile[wave][1][col * kRow + 16 * u + 4 * k8]) = v;
          }
        }
        // a lane to a key, the heads one after another
        wave_sync();
        const int key = 16 * t0 + lane;
        const bool on = from + key < to, there = on && slot[key] >= 0;
#pragma unroll
        for (int r = 0; r < HT; ++r) {
          if (HT > 4 && r >= n) continue;
          Rectified z = rectify(tile[wave][0][r * kRow + lane], tile[wave][1][r * kRow + lane]);
          z.mm = there ? z.mm : 0.f, z.vm = there ? z.vm : 0.f;
          if (on && r < n) A.scores[(h + r) * A.max_len + from + key] = make_float2(z.mm, z.vm);
          mt[r] += z.mm, vt[r] += z.vm;
        }
        wave_sync();
      }
    }
#pragma unroll
    for (int r = 0; r < HT; ++r) {
      if (HT > 4 && r >= n) continue;
      const float x = wave_sum(mt[r]), y = wave_sum(vt[r]);
      if (lane == 0 && r < n) {
        float* o = A.sums + ((h + r) * A.splits * kWaves + (int)blockIdx.x * kWaves + wave) * 2;
        o[0] = x, o[1] = y;
      }
    }
  }
}

template <typename Cell, int DP, bool VEC, int HT>
__global__ void __launch_bounds__(kThreads, (blocks_of<Cell, DP, VEC, HT>())) scores_kernel(const Args A) {
  scores_of<Cell, DP, VEC, HT>(A);
}

// Lane (r, k8) of a wave brings the features ND r .. ND r + ND - 1 (ND = DP / 16) of keys 8 k8 ..
// 8 k8 + 7 of every 32: the j-th of them, over the eight keys, is its share of a product whose rows
// are the features ND r + j. So a load covers whole rows and no value moves between lanes.
// WHOLE: the block has all of its sequence's tokens and writes the outputs.
template <typename Cell, int DP, bool VEC, int HT, bool WHOLE>
__device__ __forceinline__ void values_of(const Args& A) {
  typedef typename Cell::type T;
  constexpr int ND = DP / 16;
  constexpr bool scaled_rows = sizeof(T) == 1, ahead = DP * sizeof(T) <= 128;  // the next 32 keys' cells are in flight
  constexpr int kRow = 64 + 8;                // keys of a column's weights, banks apart
  constexpr int kCols = HT == 4 ? 16 : 3 * HT;  // columns: part p of head r is HT p + r
  __shared__ int64_t slots[kWaves][kWaveKeys];
  __shared__ float powers[kWaves][scaled_rows ? 2 * kWaveKeys : 1];
  __shared__ __align__(16) __bf16 weights[kWaves][3 * kCols * kRow];  // [w, kw, kw + w^2][column][key]
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
  __bf16* W = weights[wave];
  Raw<T, ND> am[8], aS[8];
  const T* none = reinterpret_cast<const T*>(kNothing);
  asm volatile("" : "+v"(none));  // its address is kept, not formed again
  auto fetch = [&](int i0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // what is not there weighs nothing, whatever its slot holds
      const int64_t at = slot[i0 + 8 * k8 + i];
      const T *m = static_cast<const T*>(A.c.vm) + at, *S = static_cast<const T*>(A.c.vS) + at;
      asm("" : "+v"(m), "+v"(S));  // formed before the choice, which then is no branch
      am[i] = load_raw<VEC, T, ND>(at < 0 ? none : m, ND * col, D);
      aS[i] = load_raw<VEC, T, ND>(at < 0 ? none : S, ND * col, D);
    }
  };
  for (int r0 = 0; r0 < A.R; r0 += HT) {
    const int n = A.R - r0 < HT ? A.R - r0 : HT;
    const int64_t h = b * A.H + g * A.R + r0;
    __syncthreads();  // the heads before are done with the sums and weights
    if (ahead && from < to) fetch(0);
    for (int r = wave; r < n; r += kWaves) {
      const float* p = A.sums + (h + r) * A.splits * kWaves * 2;
      float mt = 0.f, vt = 0.f;
      for (int i = lane; i < A.splits * kWaves; i += 64) mt += p[2 * i], vt += p[2 * i + 1];
      mt = wave_sum(mt), vt = wave_sum(vt);
      if (lane == 0) row[r] = row_sums(mt, vt);
    }
    // columns that no head writes
    for (int i = lane; i < 3 * kCols * kRow / 8; i += 64) reinterpret_cast<bf8*>(W)[i] = bf8{};
    __syncthreads();
    acc4 om[ND], oS[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) om[j] = oS[j] = acc4{0, 0, 0, 0};
    float total[HT] = {};
    float2 z[HT];
    auto fetch_scores = [&](int key0) {
      const int key = key0 + lane < to ? key0 + lane : from;
#pragma unroll
      for (int r = 0; r < HT; ++r) z[r] = A.scores[(h + (r < n ? r : 0)) * A.max_len + key];
    };
    if (from < to) fetch_scores(from);
    for (int key0 = from; key0 < to; key0 += 64) {
      const int i0 = key0 - from;
      {
        // a lane to a key
        float a = 1.f, s = 1.f;
        if constexpr (scaled_rows) a = pm[i0 + lane], s = pS[i0 + lane];
#pragma unroll
        for (int r = 0; r < HT; ++r) {
          if (HT > 4 && r >= n) continue;
          const Weight o = weigh(Rectified{z[r].x, z[r].y, 0.f, 0.f}, row[r]);
          const bool there = key0 + lane < to && r < n && z[r].x != 0.f;
          const float w = there ? o.w : 0.f, k = there ? o.k : 0.f;
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
              W[(kCols * q + HT * p + r) * kRow + lane] = part;
              rest -= (float)part;
            }
          }
        }
      }
      wave_sync();
      fetch_scores(key0 + 64 < to ? key0 + 64 : key0);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!ahead) fetch(i0 + 32 * half);
        Raw<T, 8> x[ND], y[ND];
        turn(am, x), turn(aS, y);
        if (ahead) fetch(half == 0 || key0 + 64 < to ? i0 + 32 * half + 32 : i0);
        Right<HT> w[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int p = 0; p < (HT == 4 ? 1 : 3); ++p)
            w[q].p[p] = *reinterpret_cast<const bf8*>(W + (kCols * q + HT * p + col) * kRow + 32 * half + 8 * k8);
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          om[j] = mul<HT>(parts_of(x[j]), w[0], om[j]);
          oS[j] = mul<HT>(squares_of(x[j]), w[1], oS[j]);
          oS[j] = mul<HT>(parts_of(y[j]), w[2], oS[j]);
        }
      }
      wave_sync();
    }
#pragma unroll
    for (int r = 0; r < HT; ++r) {
      if (HT > 4 && r >= n) continue;
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
        for (int r = 0; r < 4; ++r) {
          const float x = over_parts<HT>(k == 0 ? om[j][r] : oS[j][r]);
          if (col < HT) red[(wave * DP + ND * (4 * k8 + r) + j) * HT + col] = x;
        }
      __syncthreads();
      for (int i = threadIdx.x; i < n * D; i += kThreads) {
        const int r = i / D, f = i - r * D;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += red[(w * DP + f) * HT + r];
        if constexpr (WHOLE) {
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) sum += totals[w][r];
          const float inv = fast_rcp(fmaxf(sum, kRemaxFloor));
          if (k == 0)
            A.mo[(h + r) * D + f] = x * inv;
          else
            A.So[(h + r) * D + f] = x * inv * inv;
        } else {
          part[r * step + k * D + f] = x;
        }
      }
    }
    if (!WHOLE && (int)threadIdx.x < n) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x += totals[w][threadIdx.x];
      part[threadIdx.x * step + 2 * D] = x;
    }
  }
}

template <typename Cell, int DP, bool VEC, int HT>
__global__ void __launch_bounds__(kThreads, (HT == 16 ? 1 : blocks_of<Cell, DP, VEC, HT>())) values_kernel(const Args A) {
  values_of<Cell, DP, VEC, HT, false>(A);
}
// Sequences that one block holds: no launch waits for another. A lane reads the scores that it wrote
// itself.
template <typename Cell, int DP>
__global__ void __launch_bounds__(kThreads, 1) whole_kernel(const Args A) {
  scores_of<Cell, DP, true, 4>(A);
  __syncthreads();  // the waves' sums
  values_of<Cell, DP, true, 4, true>(A);
}

// A block to a query head, a thread to a sum: the splits that its sequence's length reaches, in order.
__global__ void __launch_bounds__(kThreads) join_kernel(const Args A) {
  __shared__ float totals[kWaves];
  const int64_t h = blockIdx.x;
  const int D = A.c.D, step = 2 * D + 1, block_keys = kWaves * A.wave_keys;
  const int len = length_of(A, h / A.H), n = len <= block_keys ? 1 : (len + block_keys - 1) / block_keys;
  const float* p = A.parts + h * A.splits * step;
  float sum = 0.f, x = 0.f;
  for (int k = threadIdx.x; k < n; k += kThreads) sum += p[(int64_t)k * step + 2 * D];
  const int f = threadIdx.x;  // 2 D <= kThreads
  if (f < 2 * D) {
#pragma unroll 8
    for (int k = 0; k < n; ++k) x += p[(int64_t)k * step + f];
  }
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) totals[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = (totals[0] + totals[1]) + (totals[2] + totals[3]);
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor));
  if (f < D) A.mo[h * D + f] = x * inv;
  else if (f < 2 * D) A.So[h * D + f - D] = x * inv * inv;
}

// Keys of a wave: as many as leave four blocks for each of the 256 CUs.
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
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)(a.B * a.H)), dim3(kThreads), 0, s, a);
}
template <typename Cell, int DP>
void launch_heads(const Args& a, bool vec, dim3 grid, hipStream_t s) {
  // One launch where no CU has two blocks (8 sequences of 256 tokens, 8 key heads of 32 in fp32: 16.4
  // us, 21.6 as three; 64 of 128 in bf16: 42.8, 39.3, since a CU holds one block of it and two of theirs).
  if (vec && a.R <= 4 && a.splits == 1 && a.B * a.c.G <= 256) {
    hipLaunchKernelGGL((whole_kernel<Cell, DP>), grid, dim3(kThreads), 0, s, a);
    return;
  }
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
  return check_launch(what);
}
