// Keys and values of tokens into the pages of a cache, rounded to its type, and back.
//
// A token's entry for one key head is four rows of D cells: means and variances of the key and
// of the value. Types: fp32; bf16 (nearest, ties to even); e4m3 with one power of two a row,
//   e = the least exponent with max|x| <= 448 * 2^e, e in [-126, 127]
//   code = e4m3(x 2^-e) (nearest, ties to even; exact below the rounding, as 2^e is)
// A power of two costs nothing in precision against max|x| / 448 (e4m3 is a floating type: half
// a step is 2^-4 of the value either way) and makes codes, scales and what is read back the
// same on every machine. Infinities and NaN are stored as NaN and leave the scale to the rest.
//
// HBM bound, one pass: L lanes hold a row, four cells each; reads of 16 bytes a lane.
#include "tagi_kv_cache.h"

namespace tagi {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 128;

struct Args {
  const float *mk, *Sk, *mv, *Sv;
  tagi_heads lk, lv;
  float *omk, *oSk, *omv, *oSv;
  const void *starts, *counts;
  int start_bytes, count_bytes;
  CacheView c;
  int64_t B, T, rows;  // rows: B T G, four arrays each
  int L;
};

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ uint32_t fp8x4(f4u x, float r) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = finite(x[j]) ? x[j] * r : __uint_as_float(0x7fc00000u);
  int o = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], o, true);
}

// Items: (row, array), array fastest, so that neighbouring lanes write the four pools.
template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const Args A) {
  typedef typename Cell::type T;
  const int lane = threadIdx.x & (A.L - 1);
  const int64_t item = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / A.L) + threadIdx.x / A.L;
  const int i = (int)(item & 3);
  const int64_t row = item >> 2;
  int64_t slot = -1, at = 0;
  if (row < A.rows) {
    const int g = (int)(row % A.c.G);
    const int64_t bt = row / A.c.G, b = bt / A.T, t = bt - b * A.T;
    if (!A.counts || t < read_int(A.counts, A.count_bytes, b))
      slot = cache_row(A.c, b, (A.starts ? read_int(A.starts, A.start_bytes, b) : 0) + t, g);
    const tagi_heads& l = i < 2 ? A.lk : A.lv;
    at = b * l.sb + t * l.st + g * l.sh;
  }
  const float* src = (i == 0 ? A.mk : (i == 1 ? A.Sk : (i == 2 ? A.mv : A.Sv))) + at;
  T* dst = static_cast<T*>(i == 0 ? A.c.km : (i == 1 ? A.c.kS : (i == 2 ? A.c.vm : A.c.vS))) + slot * A.c.D;
  const int d = 4 * lane;
  f4u x = {0, 0, 0, 0};
  if (slot >= 0 && d < A.c.D) {
    if constexpr (VEC) {
      x = *reinterpret_cast<const f4u*>(src + d);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = d + j < A.c.D ? src[d + j] : 0.f;
    }
  }
  if constexpr (sizeof(T) == 1) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, finite(x[j]) ? fabsf(x[j]) : 0.f);
    for (int w = A.L >> 1; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w));
    if (slot < 0) return;
    // m = f 2^e with f in [1/2, 1): 448 = 0.875 * 2^9
    int e;
    const float f = frexpf(m, &e);
    e = m == 0.f ? -126 : e - (f > 0.875f ? 8 : 9);
    e = e < -126 ? -126 : (e > 127 ? 127 : e);
    if (lane == 0) A.c.scales[slot * 4 + i] = (uint8_t)(e + 127);
    if (d >= A.c.D) return;
    // 2^-e as a float: e = 127 would be subnormal, but a row reaches 448 * 2^120 at most
    const uint32_t codes = fp8x4(x, __uint_as_float((uint32_t)(127 - e) << 23));
    if constexpr (VEC) {
      *reinterpret_cast<uint32_t*>(dst + d) = codes;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < A.c.D) dst[d + j] = (uint8_t)(codes >> (8 * j));
    }
  } else {
    if (slot < 0 || d >= A.c.D) return;
    if constexpr (VEC && sizeof(T) == 4) {
      *reinterpret_cast<f4u*>(dst + d) = x;
    } else if constexpr (VEC) {
      typedef __bf16 b4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<b4*>(dst + d) = b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < A.c.D) dst[d + j] = (T)x[j];
    }
  }
}

// Items as above; starts holds the sequences' lengths.
template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const Args A) {
  typedef typename Cell::type T;
  const int lane = threadIdx.x & (A.L - 1);
  const int64_t item = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / A.L) + threadIdx.x / A.L;
  const int i = (int)(item & 3);
  const int64_t row = item >> 2;
  const int d = 4 * lane;
  if (row >= A.rows || d >= A.c.D) return;
  const int g = (int)(row % A.c.G);
  const int64_t bt = row / A.c.G, b = bt / A.T, t = bt - b * A.T;
  const int64_t slot = t < read_int(A.starts, A.start_bytes, b) ? cache_row(A.c, b, t, g) : -1;
  const T* src = static_cast<const T*>(i == 0 ? A.c.km : (i == 1 ? A.c.kS : (i == 2 ? A.c.vm : A.c.vS))) + slot * A.c.D;
  float* dst = (i == 0 ? A.omk : (i == 1 ? A.oSk : (i == 2 ? A.omv : A.oSv))) + row * A.c.D;
  f4u x = {0, 0, 0, 0};
  if (slot >= 0) {
    if constexpr (VEC) {
      x = load4(src + d);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = d + j < A.c.D ? load1(src + d + j) : 0.f;
    }
    if constexpr (sizeof(T) == 1) {
      const int e = A.c.scales[slot * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = scaled(x[j], e);
    }
  }
  if constexpr (VEC) {
    *reinterpret_cast<f4u*>(dst + d) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < A.c.D) dst[d + j] = x[j];
  }
}

int lanes_of(int D) {
  int L = 1;
  while (4 * L < D) L *= 2;
  return L;
}

int sizes(const char* what, Args& a, int64_t B, int64_t T) {
  TAGI_REQUIRE(T >= 0 && T < (1ll << 31), "%s: bad sizes", what);
  a.B = B, a.T = T, a.L = lanes_of(a.c.D);
  TAGI_REQUIRE(B == 0 || T == 0 || B < (1ll << 40) / T / a.c.G, "%s: too large", what);
  a.rows = B * T * a.c.G;
  return TAGI_OK;
}
dim3 grid_of(const Args& a) {  // fewer than 2^32 threads in one dimension
  const int64_t blocks = cdiv(4 * a.rows, kThreads / a.L), x = blocks < (1 << 20) ? blocks : (1 << 20);
  return dim3((unsigned)x, (unsigned)cdiv(blocks, x));
}
bool al(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }
// rows of four-cell groups, each aligned in the pools
bool vec(const Args& a, int type) {
  const int n = type == CELL_F32 ? 4 : 4 * cell_bytes(type);
  return a.c.D % 4 == 0 && al(a.c.km, n) && al(a.c.kS, n) && al(a.c.vm, n) && al(a.c.vS, n);
}

}  // namespace

int cache_view(const char* what, CacheView* c, const tagi_kv_cache* k, const int32_t* table, int64_t width, int64_t B) {
  TAGI_REQUIRE(k, "%s: null pointer", what);
  TAGI_REQUIRE(k->type >= CELL_F32 && k->type <= CELL_FP8, "%s: unknown cache type", what);
  TAGI_REQUIRE(k->pages >= 0 && k->heads > 0 && k->page_size > 0 && k->head_dim > 0 && width >= 0 && B >= 0,
               "%s: bad sizes", what);
  if (k->head_dim > kMaxDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxDim);
  TAGI_REQUIRE(k->pages < (1ll << 31) && k->heads < (1 << 20) && k->page_size < (1 << 30) && B < (1 << 30), "%s: too large",
               what);
  TAGI_REQUIRE(k->pages == 0 || (k->km && k->kS && k->vm && k->vS && (k->type != CELL_FP8 || k->scales)),
               "%s: null pointer", what);
  TAGI_REQUIRE(B == 0 || width == 0 || table, "%s: null pointer", what);
  c->km = k->km, c->kS = k->kS, c->vm = k->vm, c->vS = k->vS, c->scales = static_cast<uint8_t*>(k->scales);
  c->table = table, c->pages = k->pages, c->width = width;
  c->G = (int)k->heads, c->D = (int)k->head_dim, c->page = (int)k->page_size;
  return TAGI_OK;
}

}  // namespace tagi

using namespace tagi;

#define CACHE_LAUNCH(kernel)                                                                     \
  do {                                                                                           \
    const bool v = vec(a, cache->type);                                                          \
    if (cache->type == CELL_F32)                                                                 \
      hipLaunchKernelGGL((v ? kernel<F32Cell, true> : kernel<F32Cell, false>), grid_of(a), dim3(kThreads), 0, s, a);   \
    else if (cache->type == CELL_BF16)                                                           \
      hipLaunchKernelGGL((v ? kernel<Bf16Cell, true> : kernel<Bf16Cell, false>), grid_of(a), dim3(kThreads), 0, s, a); \
    else                                                                                         \
      hipLaunchKernelGGL((v ? kernel<Fp8Cell, true> : kernel<Fp8Cell, false>), grid_of(a), dim3(kThreads), 0, s, a);   \
  } while (0)

extern "C" int tagi_kv_cache_write(const tagi_kv_cache* cache, const float* mk, const float* Sk, const tagi_heads* lk,
                                   const float* mv, const float* Sv, const tagi_heads* lv, const int32_t* table,
                                   int64_t width, const void* starts, int start_bytes, const void* counts,
                                   int count_bytes, int64_t B, int64_t T, tagi_stream_t stream) {
  const char* what = "tagi_kv_cache_write";
  Args a{};
  if (int rc = cache_view(what, &a.c, cache, table, width, B)) return rc;
  if (int rc = sizes(what, a, B, T)) return rc;
  TAGI_REQUIRE(!starts || start_bytes == 4 || start_bytes == 8, "%s: starts are int32 or int64", what);
  TAGI_REQUIRE(!counts || count_bytes == 4 || count_bytes == 8, "%s: counts are int32 or int64", what);
  if (a.rows == 0 || cache->pages == 0 || width == 0) return TAGI_OK;
  TAGI_REQUIRE(mk && Sk && lk && mv && Sv && lv, "%s: null pointer", what);
  a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv, a.lk = *lk, a.lv = *lv;
  a.starts = starts, a.start_bytes = start_bytes, a.counts = counts, a.count_bytes = count_bytes;
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 0.0, (16.0 + 4.0 * cell_bytes(cache->type)) * a.rows * a.c.D);
  CACHE_LAUNCH(cache_write_kernel);
  return check_launch(what);
}

extern "C" int tagi_kv_cache_read(const tagi_kv_cache* cache, const int32_t* table, int64_t width, const void* lengths,
                                  int len_bytes, float* mk, float* Sk, float* mv, float* Sv, int64_t B, int64_t T,
                                  tagi_stream_t stream) {
  const char* what = "tagi_kv_cache_read";
  Args a{};
  if (int rc = cache_view(what, &a.c, cache, table, width, B)) return rc;
  if (int rc = sizes(what, a, B, T)) return rc;
  if (a.rows == 0) return TAGI_OK;
  TAGI_REQUIRE(lengths && (len_bytes == 4 || len_bytes == 8), "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(mk && Sk && mv && Sv, "%s: null pointer", what);
  a.omk = mk, a.oSk = Sk, a.omv = mv, a.oSv = Sv, a.starts = lengths, a.start_bytes = len_bytes;
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 0.0, (16.0 + 4.0 * cell_bytes(cache->type)) * a.rows * a.c.D);
  CACHE_LAUNCH(cache_read_kernel);
  return check_launch(what);
}
