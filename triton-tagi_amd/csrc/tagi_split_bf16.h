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

// What a part leaves: x0 - p.x and x1 - p.y, each one product-sum of the packed pair with (-1, 0) or
// (0, -1) that takes no unpacking (exact: the difference is a float). The two constants come from
// scalar registers: written out, (-1, 0) becomes the inline constant -1.0, which the hardware reads
// as (0, -1).
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void rest_of(bf2 p, float& x0, float& x1) {
  uint32_t c0 = 0x0000bf80u, c1 = 0xbf800000u;
  asm("" : "+s"(c0));
  asm("" : "+s"(c1));
  x0 = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(bf2, c0), x0, false);
  x1 = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(bf2, c1), x1, false);
}

template <int P>
__device__ __forceinline__ Parts<P> split(const float (&x)[8]) {
  Parts<P> out;
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int k = 0; k < P; ++k)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const bf2 p = {(__bf16)rest[i], (__bf16)rest[i + 1]};
      out.p[k][i] = p.x, out.p[k][i + 1] = p.y;
      if (k + 1 < P) rest_of(p, rest[i], rest[i + 1]);
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
