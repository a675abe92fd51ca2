// The paged key and value cache as its kernels see it (layout in include/tagi_hip.h).
#pragma once
#include "tagi_common.h"

namespace tagi {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// Element types of the pools.
struct F32Cell {
  typedef float type;
};
struct Bf16Cell {
  typedef __bf16 type;
};
struct Fp8Cell {  // e4m3: four exponent bits, three mantissa bits, no infinities, largest 448
  typedef uint8_t type;
};

struct CacheView {
  void *km, *kS, *vm, *vS;  // (pages, G, page, D)
  uint8_t* scales;          // (pages, G, page, 4): biased exponents of a row's km, kS, vm, vS
  const int32_t* table;     // (B, width): pages of each sequence in order
  int64_t pages, width;
  int G, D, page;
};

// Row (page slot) of token `at` of sequence b for key head g: -1 where the table or the pool
// has no such page.
__device__ __forceinline__ int64_t cache_row(const CacheView& c, int64_t b, int64_t at, int g) {
  if (at < 0) return -1;
  // a division of 64 bits takes the time of the row's loads
  const int64_t i = at >> 31 ? at / c.page : (int64_t)((uint32_t)at / (uint32_t)c.page);
  if (i >= c.width) return -1;
  const int64_t p = c.table[b * c.width + i];
  if (p < 0 || p >= c.pages) return -1;
  return (p * c.G + g) * c.page + (at - i * c.page);
}

__device__ __forceinline__ int64_t read_int(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// code * 2^(e - 127): exact
__device__ __forceinline__ float scaled(float code, int e) { return __builtin_ldexpf(code, e - 127); }

// Four neighbouring cells as floats (codes unscaled), from an address aligned to four cells.
__device__ __forceinline__ f4u load4(const float* p) { return *reinterpret_cast<const f4u*>(p); }
__device__ __forceinline__ f4u load4(const __bf16* p) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  return f4u{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
             __uint_as_float(x.y & 0xffff0000u)};
}
__device__ __forceinline__ f4u load4(const uint8_t* p) {
  const int x = *reinterpret_cast<const int*>(p);
  return f4u{__builtin_amdgcn_cvt_f32_fp8(x, 0), __builtin_amdgcn_cvt_f32_fp8(x, 1),
             __builtin_amdgcn_cvt_f32_fp8(x, 2), __builtin_amdgcn_cvt_f32_fp8(x, 3)};
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ float load1(const uint8_t* p) { return __builtin_amdgcn_cvt_f32_fp8((int)*p, 0); }

enum CellType { CELL_F32 = 0, CELL_BF16 = 1, CELL_FP8 = 2 };
inline int cell_bytes(int type) { return type == CELL_F32 ? 4 : (type == CELL_BF16 ? 2 : 1); }

// Checks of a cache's description; fills the view. `what` names the entry point.
int cache_view(const char* what, CacheView* c, const tagi_kv_cache* cache, const int32_t* table, int64_t width,
               int64_t B);

}  // namespace tagi
