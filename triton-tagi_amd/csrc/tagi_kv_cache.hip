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
// HBM bound, one pass: L lanes hold the four rows of a token and key head, four cells of each, so
// that four loads of 16 bytes a lane are in flight and the slot is looked up once. Measured: 16 x 2048
// tokens of 8 heads of 128 into e4m3 128 us, 5.3 TB/s of 672 MB, where a copy has 5.4 (a row of one
// array to the lanes, with divisions of 64 bits: 256 us); 5 x 6001 out of bf16 126 us, 5.1 TB/s.
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
  int64_t B, rows;  // rows: T G of a sequence, four arrays each
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

// Blocks of a row's lanes: x over a sequence's rows (token, key head), y over sequences.
struct Row {
  uint32_t t, g;
  bool on;
};
__device__ __forceinline__ Row row_of(const Args& A) {
  const uint32_t i = blockIdx.x * (kThreads / A.L) + threadIdx.x / A.L, t = i / (uint32_t)A.c.G;
  return {t, i - t * (uint32_t)A.c.G, i < A.rows};
}

template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const Args A) {
  typedef typename Cell::type T;
  const int lane = threadIdx.x & (A.L - 1), d = 4 * lane;
  const Row r = row_of(A);
  const float* const src[4] = {A.mk, A.Sk, A.mv, A.Sv};
  T* const dst[4] = {static_cast<T*>(A.c.km), static_cast<T*>(A.c.kS), static_cast<T*>(A.c.vm), static_cast<T*>(A.c.vS)};
  for (int64_t b = blockIdx.y; b < A.B; b += gridDim.y) {
    int64_t slot = -1;
    if (r.on && (!A.counts || r.t < read_int(A.counts, A.count_bytes, b)))
      slot = cache_row(A.c, b, (A.starts ? read_int(A.starts, A.start_bytes, b) : 0) + r.t, r.g);
    const bool on = slot >= 0 && d < A.c.D;
    f4u x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const tagi_heads& l = i < 2 ? A.lk : A.lv;
      const float* const p = src[i] + b * l.sb + (int64_t)r.t * l.st + (int64_t)r.g * l.sh + d;
      x[i] = f4u{0, 0, 0, 0};
      if constexpr (VEC) {
        if (on) x[i] = *reinterpret_cast<const f4u*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = on && d + j < A.c.D ? p[j] : 0.f;
      }
    }
    uint32_t exponents = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T* const o = dst[i] + slot * A.c.D + d;
      if constexpr (sizeof(T) == 1) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, finite(x[i][j]) ? fabsf(x[i][j]) : 0.f);
        for (int w = A.L >> 1; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w));
        // m = f 2^e with f in [1/2, 1): 448 = 0.875 * 2^9
        int e;
        const float f = frexpf(m, &e);
        e = m == 0.f ? -126 : e - (f > 0.875f ? 8 : 9);
        e = e < -126 ? -126 : (e > 127 ? 127 : e);
        exponents |= (uint32_t)(e + 127) << (8 * i);
        // 2^-e as a float: e = 127 would be subnormal, but a row reaches 448 * 2^120 at most
        const uint32_t codes = fp8x4(x[i], __uint_as_float((uint32_t)(127 - e) << 23));
        if constexpr (VEC) {
          if (on) *reinterpret_cast<uint32_t*>(o) = codes;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (on && d + j < A.c.D) o[j] = (uint8_t)(codes >> (8 * j));
        }
      } else if constexpr (VEC && sizeof(T) == 4) {
        if (on) *reinterpret_cast<f4u*>(o) = x[i];
      } else if constexpr (VEC) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        if (on) *reinterpret_cast<b4*>(o) = b4{(__bf16)x[i][0], (__bf16)x[i][1], (__bf16)x[i][2], (__bf16)x[i][3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (on && d + j < A.c.D) o[j] = (T)x[i][j];
      }
    }
    if (sizeof(T) == 1 && lane == 0 && on) reinterpret_cast<uint32_t*>(A.c.scales)[slot] = exponents;
  }
}

// starts holds the sequences' lengths.
template <typename Cell, bool VEC>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const Args A) {
  typedef typename Cell::type T;
  const int d = 4 * (threadIdx.x & (A.L - 1));
  const Row r = row_of(A);
  if (!r.on || d >= A.c.D) return;
  const T* const src[4] = {static_cast<const T*>(A.c.km), static_cast<const T*>(A.c.kS), static_cast<const T*>(A.c.vm),
                           static_cast<const T*>(A.c.vS)};
  float* const dst[4] = {A.omk, A.oSk, A.omv, A.oSv};
  for (int64_t b = blockIdx.y; b < A.B; b += gridDim.y) {
    const int64_t slot = r.t < read_int(A.starts, A.start_bytes, b) ? cache_row(A.c, b, r.t, r.g) : -1;
    const int64_t to = (b * A.rows + (int64_t)r.t * A.c.G + r.g) * A.c.D + d;
    f4u x[4];
    uint32_t exponents = 0;
    if (sizeof(T) == 1 && slot >= 0) exponents = reinterpret_cast<const uint32_t*>(A.c.scales)[slot];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* const p = src[i] + slot * A.c.D + d;
      x[i] = f4u{0, 0, 0, 0};
      if constexpr (VEC) {
        if (slot >= 0) x[i] = load4(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = slot >= 0 && d + j < A.c.D ? load1(p + j) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = scaled(x[i][j], (exponents >> (8 * i)) & 255);
      }
      if constexpr (VEC) {
        *reinterpret_cast<f4u*>(dst[i] + to) = x[i];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < A.c.D) dst[i][to + j] = x[i][j];
      }
    }
  }
}

int lanes_of(int D) {
  int L = 1;
  while (4 * L < D) L *= 2;
  return L;
}

int sizes(const char* what, Args& a, int64_t B, int64_t T) {
  TAGI_REQUIRE(T >= 0 && T < (1ll << 31), "%s: bad sizes", what);
  a.B = B, a.rows = T * a.c.G, a.L = lanes_of(a.c.D);
  // fewer than 2^32 threads in one dimension
  TAGI_REQUIRE(a.rows < (1ll << 32) / a.L && cdiv(a.rows, kThreads / a.L) * kThreads < (1ll << 32), "%s: too large", what);
  return TAGI_OK;
}
dim3 grid_of(const Args& a) {
  const int64_t y = a.B < 65535 ? a.B : 65535;
  return dim3((unsigned)cdiv(a.rows, kThreads / a.L), (unsigned)y);
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
  TAGI_REQUIRE(k->type != CELL_FP8 || (uintptr_t)k->scales % 4 == 0, "%s: scales are not aligned to a row's four", what);
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
  if (a.rows == 0 || B == 0 || cache->pages == 0 || width == 0) return TAGI_OK;
  TAGI_REQUIRE(mk && Sk && lk && mv && Sv && lv, "%s: null pointer", what);
  a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv, a.lk = *lk, a.lv = *lv;
  a.starts = starts, a.start_bytes = start_bytes, a.counts = counts, a.count_bytes = count_bytes;
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 0.0, (16.0 + 4.0 * cell_bytes(cache->type)) * a.B * a.rows * a.c.D);
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
  if (a.rows == 0 || B == 0) return TAGI_OK;
  TAGI_REQUIRE(lengths && (len_bytes == 4 || len_bytes == 8), "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(mk && Sk && mv && Sv, "%s: null pointer", what);
  a.omk = mk, a.oSk = Sk, a.omv = mv, a.oSv = Sv, a.starts = lengths, a.start_bytes = len_bytes;
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 0.0, (16.0 + 4.0 * cell_bytes(cache->type)) * a.B * a.rows * a.c.D);
  CACHE_LAUNCH(cache_read_kernel);
  return check_launch(what);
}
