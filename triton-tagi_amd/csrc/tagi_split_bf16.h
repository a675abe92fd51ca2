// Products of fp32 values on the bf16 matrix cores: a value as up to three bf16 parts.
//
// x = p0 + p1 + p2 with p0 = bf16(x), p1 = bf16(x - p0), p2 = bf16(x - p0 - p1): 24 bits in three
// parts of 8, exact for normal values above 2^-109. A product of two split values keeps the part
// pairs (i, j) with i + j <= 2: what is dropped is 2^-24 of the product and less, the size of an
// fp32 rounding. Values that are bf16 (or e4m3) already have one part, their squares two (one):
// products of 8 (4) bits.
#pragma once
#include "tagi_common.h"

namespace tagi {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float acc4 __attribute__((ext_vector_type(4)));

template <int P>
struct Parts {
  bf8 p[P];
};

template <int P>
__device__ __forceinline__ Parts<P> split(const float (&x)[8]) {
  Parts<P> out;
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int k = 0; k < P; ++k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out.p[k][i] = (__bf16)rest[i];
    if (k + 1 < P) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] -= (float)out.p[k][i];
    }
  }
  return out;
}

// c += a b over 32 terms of a 16 x 16 tile: lane l holds row (column) l % 16 of a (b), terms
// 8 (l / 16) + 0..7, and of c column l % 16, rows 4 (l / 16) + 0..3. Small parts first.
template <int PA, int PB>
__device__ __forceinline__ acc4 mma(const Parts<PA>& a, const Parts<PB>& b, acc4 c) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < PA; ++i) {
      const int j = s - i;
      if (j >= 0 && j < PB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    }
  return c;
}

}  // namespace tagi
