// Remax attention of one query of every sequence over the pages of its cache.
//
// The formulas of tagi_remax_attention.hip with one row per head. A sequence's tokens are split
// over blocks; a weight needs the sums over all of them first, so there are three launches:
//   scores: the keys' pages once; moments of the rectified scores (mm, vm) to the workspace, and
//           each split's sums of them
//   values: the splits' sums added in order, weights, the values' pages once; each split's sums
//   join:   the splits' sums added in order and normalised
// A block reads a key head's tokens once for all of the query heads that share it.
#include "tagi_kv_cache.h"
#include "tagi_remax.h"

namespace tagi {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // query heads at a time
constexpr int kKeys = 64;  // keys whose weights are formed at a time

struct Args {
  const float *mq, *Sq;
  tagi_heads lq;
  CacheView c;
  const void* lengths;
  int len_bytes;
  float *mo, *So;
  float2* scores;  // (B, H, max_len): (mm, vm), mm = 0 where there is no token
  float* sums;     // (B, H, splits, 2)
  float* parts;    // (B, H, splits, 2 D + 1)
  int64_t B;
  int H, R, max_len, splits, chunk;
  float c1, c2;
};

__device__ __forceinline__ int length_of(const Args& A, int64_t b) {
  const int64_t n = read_int(A.lengths, A.len_bytes, b), room = A.c.width * A.c.page;
  const int64_t most = room < A.max_len ? room : A.max_len;
  return (int)(n < 0 ? 0 : (n < most ? n : most));
}

__device__ __forceinline__ float block_sum(float x, float* red) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// A thread to a key.
template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) scores_kernel(const Args A) {
  typedef typename Cell::type T;
  __shared__ float red[4];
  const int64_t b = blockIdx.z;
  const int g = blockIdx.y, D = A.c.D, len = length_of(A, b);
  const int from = blockIdx.x * A.chunk, to = from + A.chunk < len ? from + A.chunk : len;
  for (int r0 = 0; r0 < A.R; r0 += kHeads) {
    const int n = A.R - r0 < kHeads ? A.R - r0 : kHeads;
    float mt[kHeads] = {}, vt[kHeads] = {};
    const float* q = A.mq + b * A.lq.sb + (int64_t)(g * A.R + r0) * A.lq.sh;
    const float* Q = A.Sq + b * A.lq.sb + (int64_t)(g * A.R + r0) * A.lq.sh;
    for (int key = from + (int)threadIdx.x; key < to; key += kThreads) {
      const int64_t row = cache_row(A.c, b, key, g);
      float m[kHeads] = {}, v[kHeads] = {};
      if (row >= 0) {
        const T *km = static_cast<const T*>(A.c.km) + row * D, *kS = static_cast<const T*>(A.c.kS) + row * D;
        for (int d = 0; d < D; d += 4) {
          float a[4], s[4];
          if constexpr (VEC) {
            const f4u x = load4(km + d), y = load4(kS + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = x[j], s[j] = y[j];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = d + j < D ? load1(km + d + j) : 0.f, s[j] = d + j < D ? load1(kS + d + j) : 0.f;
          }
          if constexpr (sizeof(T) == 1) {
            const int em = A.c.scales[row * 4], eS = A.c.scales[row * 4 + 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = scaled(a[j], em), s[j] = scaled(s[j], eS);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float k2 = fmaf(a[j], a[j], s[j]);
#pragma unroll
            for (int r = 0; r < kHeads; ++r) {
              const int64_t at = r < n && d + j < D ? r * A.lq.sh + d + j : 0;
              const float x = q[at], X = Q[at];
              m[r] = fmaf(a[j], x, m[r]);
              v[r] = fmaf(k2, X, fmaf(s[j], x * x, v[r]));
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kHeads; ++r) {
        if (r >= n) continue;
        float mm, vm, cdf;
        rectify(m[r] * A.c1, v[r] * A.c2, mm, vm, cdf);
        if (row < 0) mm = vm = 0.f;
        A.scores[(b * A.H + g * A.R + r0 + r) * A.max_len + key] = make_float2(mm, vm);
        mt[r] += mm, vt[r] += vm;
      }
    }
#pragma unroll
    for (int r = 0; r < kHeads; ++r) {
      if (r >= n) continue;
      const float x = block_sum(mt[r], red), y = block_sum(vt[r], red);
      if (threadIdx.x == 0) {
        float* o = A.sums + ((b * A.H + g * A.R + r0 + r) * A.splits + blockIdx.x) * 2;
        o[0] = x, o[1] = y;
      }
    }
  }
}

// L lanes to a key, four features each; the keys' shares are added through LDS in order.
template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) values_kernel(const Args A, int L) {
  typedef typename Cell::type T;
  __shared__ float4 weights[kHeads][kKeys];
  __shared__ int64_t slot[kKeys];
  __shared__ float acc[kThreads][9];
  const int64_t b = blockIdx.z;
  const int g = blockIdx.y, D = A.c.D, len = length_of(A, b);
  const int from = blockIdx.x * A.chunk, to = from + A.chunk < len ? from + A.chunk : len;
  const int lane = threadIdx.x & (L - 1), share = threadIdx.x / L, shares = kThreads / L, d = 4 * lane;
  for (int r0 = 0; r0 < A.R; r0 += kHeads) {
    const int n = A.R - r0 < kHeads ? A.R - r0 : kHeads;
    const int64_t h = b * A.H + g * A.R + r0;
    // thread (head, key) forms weights: head = tid / 64
    const int wr = threadIdx.x / kKeys, wk = threadIdx.x % kKeys;
    float mt = 0.f, vt = 0.f, sum = 0.f;
    if (wr < n) {
      const float* p = A.sums + (h + wr) * A.splits * 2;
      for (int i = 0; i < A.splits; ++i) mt += p[2 * i], vt += p[2 * i + 1];
    }
    const RowSums rs = row_sums(mt, vt);
    float om[kHeads][4] = {}, oS[kHeads][4] = {};
    for (int key0 = from; key0 < to; key0 += kKeys) {
      __syncthreads();
      if (wr < n) {
        float w = 0.f, k = 0.f, xw, rw;
        if (key0 + wk < to) {
          const float2 x = A.scores[(h + wr) * A.max_len + key0 + wk];
          if (x.x > 0.f) weigh(x.x, x.y, rs, w, k, xw, rw);
        }
        sum += w;
        weights[wr][wk] = make_float4(w, w * w, k * w * w, 0.f);
      }
      if (threadIdx.x < kKeys) slot[threadIdx.x] = key0 + (int)threadIdx.x < to ? cache_row(A.c, b, key0 + threadIdx.x, g) : -1;
      __syncthreads();
      for (int i = share; i < kKeys; i += shares) {
        const int64_t row = slot[i];
        if (row < 0 || d >= D) continue;
        const T *vm = static_cast<const T*>(A.c.vm) + row * D + d, *vS = static_cast<const T*>(A.c.vS) + row * D + d;
        float a[4], s[4];
        if constexpr (VEC) {
          const f4u x = load4(vm), y = load4(vS);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = x[j], s[j] = y[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = d + j < D ? load1(vm + j) : 0.f, s[j] = d + j < D ? load1(vS + j) : 0.f;
        }
        if constexpr (sizeof(T) == 1) {
          const int em = A.c.scales[row * 4 + 2], eS = A.c.scales[row * 4 + 3];
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = scaled(a[j], em), s[j] = scaled(s[j], eS);
        }
#pragma unroll
        for (int r = 0; r < kHeads; ++r) {
          if (r >= n) continue;
          const float4 w = weights[r][i];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            om[r][j] = fmaf(w.x, a[j], om[r][j]);
            oS[r][j] = fmaf(w.z, fmaf(a[j], a[j], s[j]), fmaf(w.y, s[j], oS[r][j]));
          }
        }
      }
    }
    float* part = A.parts + (h * A.splits + blockIdx.x) * (2 * D + 1);
    const int64_t step = (int64_t)A.splits * (2 * D + 1);
    sum = wave_sum(sum);  // kKeys = 64: a wave to a head
    if (wr < n && wk == 0) part[wr * step + 2 * D] = sum;
#pragma unroll
    for (int r = 0; r < kHeads; ++r) {
      if (r >= n) continue;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[threadIdx.x][j] = om[r][j], acc[threadIdx.x][4 + j] = oS[r][j];
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
        const int f = i < D ? i : i - D, q = (i < D ? 0 : 4) + (f & 3);
        float x = 0.f;
        for (int k = 0; k < shares; ++k) x += acc[k * L + (f >> 2)][q];
        part[r * step + i] = x;
      }
    }
  }
}

// A wave to a query head.
__global__ void __launch_bounds__(kThreads) join_kernel(const Args A) {
  const int64_t h = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (h >= A.B * A.H) return;
  const int D = A.c.D, step = 2 * D + 1;
  const float* p = A.parts + h * A.splits * step;
  float sum = 0.f;
  for (int k = 0; k < A.splits; ++k) sum += p[k * step + 2 * D];
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor)), inv2 = inv * inv;
  for (int f = threadIdx.x & 63; f < D; f += 64) {
    float x = 0.f, y = 0.f;
    for (int k = 0; k < A.splits; ++k) x += p[k * step + f], y += p[k * step + D + f];
    A.mo[h * D + f] = x * inv, A.So[h * D + f] = y * inv2;
  }
}

int splits_of(int64_t B, int64_t G, int64_t max_len) {
  int64_t s = cdiv(2048, B * G);
  if (s > cdiv(max_len, 256)) s = cdiv(max_len, 256);
  return (int)(s < 1 ? 1 : s);
}
int64_t score_floats(int64_t B, int64_t H, int64_t max_len) { return 2 * B * H * max_len; }

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_remax_attention_step_ws_bytes(int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_len) {
  if (B <= 0 || H <= 0 || G <= 0 || D <= 0 || max_len < 0) return 0;
  return 4 * (score_floats(B, H, max_len) + B * H * splits_of(B, G, max_len) * (2 * D + 3));
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
  a.B = B, a.H = (int)H, a.R = (int)(H / G), a.max_len = (int)max_len;
  a.splits = splits_of(B, G, max_len), a.chunk = (int)(cdiv(cdiv(max_len, a.splits), kKeys) * kKeys);
  a.c1 = (float)scale, a.c2 = (float)(scale * scale);
  a.scores = static_cast<float2*>(ws);
  a.sums = static_cast<float*>(ws) + score_floats(B, H, max_len), a.parts = a.sums + 2 * B * H * a.splits;
  int L = 1;
  while (4 * L < D) L *= 2;
  const int n = cache->type == CELL_F32 ? 4 : 4 * cell_bytes((int)cache->type);
  const bool vec = D % 4 == 0 && ((uintptr_t)a.c.km | (uintptr_t)a.c.kS | (uintptr_t)a.c.vm | (uintptr_t)a.c.vS) % n == 0;
  const dim3 grid((unsigned)a.splits, (unsigned)G, (unsigned)B), threads(kThreads);
#define STEP(Cell)                                                                                    \
  do {                                                                                                \
    hipLaunchKernelGGL((vec ? scores_kernel<Cell, true> : scores_kernel<Cell, false>), grid, threads, 0, s, a);    \
    hipLaunchKernelGGL((vec ? values_kernel<Cell, true> : values_kernel<Cell, false>), grid, threads, 0, s, a, L); \
  } while (0)
  if (cache->type == CELL_F32)
    STEP(F32Cell);
  else if (cache->type == CELL_BF16)
    STEP(Bf16Cell);
  else
    STEP(Fp8Cell);
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)cdiv(B * H, 4)), threads, 0, s, a);
  return check_launch(what);
}
