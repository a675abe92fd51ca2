// Scaled embedding lookup, and the parameter deltas of its table by sorted tokens.
//
//   mz[t] = c mw[id_t],  Sz[t] = c^2 Sw[id_t]
//   dmw[v] = c Sw[v] sum_{t: id_t = v} dmz[t],  dSw[v] = (c Sw[v])^2 sum_{t: id_t = v} dSz[t]
//
// Ids equal to padding_idx or outside [0, V) look up zeros and add nothing. The deltas sort
// the tokens by category (stable, so a category's tokens keep their order), cut the sorted
// list into pieces of 16 to 64 tokens and let one wavefront sum each piece's runs of equal
// ids: O(N) whatever the table holds, and a category that half of the batch asks for is
// spread over as many wavefronts as it has pieces. A run that crosses a piece's border
// leaves partial sums, which a second kernel adds in piece order. Every order is fixed by
// the ids alone: results are deterministic, with no float atomics.
#include "tagi_common.h"
#include "tagi_moments.h"

namespace tagi {
namespace {

constexpr int kSortThreads = 256;
constexpr int kMaxRadixBits = 10;

inline bool al16e(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// The category of token t, or V (sorted behind every category) for padding and ids outside
// the table. Float ids are cast toward zero; a NaN is outside.
__device__ __forceinline__ uint32_t category(const void* ids, int type, int64_t t, int64_t V, int64_t pad) {
  int64_t id = -1;
  if (type == TAGI_IDS_F32) {
    const float f = static_cast<const float*>(ids)[t];
    if (f > -1.f && f < (float)V) id = (int64_t)f;
  } else if (type == TAGI_IDS_I32) {
    id = static_cast<const int32_t*>(ids)[t];
  } else {
    id = static_cast<const int64_t*>(ids)[t];
  }
  return (id >= 0 && id < V && id != pad) ? (uint32_t)id : (uint32_t)V;
}

// ------------------------------------------------------------------------------ lookup
// One float4 (or one value) per thread and moment; a block takes whole tokens.
template <int VEC>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const void* __restrict__ ids, int type,
                                                               const float* __restrict__ mw,
                                                               const float* __restrict__ Sw, float* __restrict__ mz,
                                                               float* __restrict__ Sz, int64_t n, int64_t V, int DV,
                                                               int tok_per_block, int64_t pad, float c, float c2) {
  const int t0 = (int)threadIdx.x / DV, q0 = (int)threadIdx.x - t0 * DV;
  const int64_t t = (int64_t)blockIdx.x * tok_per_block + t0;
  if (t0 >= tok_per_block || t >= n) return;
  const uint32_t cat = category(ids, type, t, V, pad);
  const bool ok = cat < V;
  for (int q = q0; q < DV; q += 256) {
    const int64_t src = ((int64_t)cat * DV + q) * VEC, dst = (t * DV + q) * VEC;
    if constexpr (VEC == 4) {
      float4 m = make_float4(0.f, 0.f, 0.f, 0.f), s = m;
      if (ok) {
        m = *reinterpret_cast<const float4*>(mw + src);
        s = *reinterpret_cast<const float4*>(Sw + src);
      }
      *reinterpret_cast<float4*>(mz + dst) = make_float4(m.x * c, m.y * c, m.z * c, m.w * c);
      *reinterpret_cast<float4*>(Sz + dst) = make_float4(s.x * c2, s.y * c2, s.z * c2, s.w * c2);
    } else {
      mz[dst] = ok ? mw[src] * c : 0.f;
      Sz[dst] = ok ? Sw[src] * c2 : 0.f;
    }
  }
}

// -------------------------------------------------------------------------------- sort
// Least-significant-digit radix sort of (category, token index). Per digit: every block
// counts its tile's digits; a wave per digit turns the blocks' counts into places; every
// block writes its tile's pairs to them in order. Latency bound: 65536 tokens of 131071
// categories take 2 digits of 9 bits, about KSORT us a digit. Up to kSmall tokens one block
// does all of it in LDS (a launch instead of three per digit).
constexpr int kSmall = 4096, kSmallBits = 8;

struct SortPlan {
  int64_t nblk;
  int bits, passes, items;  // items: tokens of a tile for each thread
};
int key_bits(int64_t V) {  // keys are 0..V
  int b = 1;
  while ((V >> b) != 0) ++b;
  return b;
}
SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  const int total = key_bits(V);
  p.passes = (int)cdiv(total, kMaxRadixBits);
  p.bits = (int)cdiv(total, p.passes);
  p.items = n > (1 << 20) ? 16 : 4;
  p.nblk = cdiv(n, kSortThreads * p.items);
  return p;
}

struct SortArgs {
  const void* ids;
  int type, first;
  const uint32_t* kin;
  const uint32_t* vin;
  uint32_t* kout;
  uint32_t* vout;
  uint32_t* hist;   // [digit][block]: counts, then places within the digit
  uint32_t* total;  // [digit]
  int64_t n, V, pad;
  int nblk, shift, bits;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t i) {
  return a.first ? category(a.ids, a.type, i, a.V, a.pad) : a.kin[i];
}

// Lanes of the wave whose `bits`-bit digit equals this lane's (among those with `on`).
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool on, int bits) {
  uint64_t same = __ballot(on);
  for (int bit = 0; bit < bits; ++bit) {
    const uint64_t m = __ballot((d >> bit) & 1);
    same &= ((d >> bit) & 1) ? m : ~m;
  }
  return same;
}

template <int IT>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  __shared__ uint32_t cnt[1 << kMaxRadixBits];
  const int radix = 1 << a.bits;
  for (int d = threadIdx.x; d < radix; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * (kSortThreads * IT) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int64_t i = i0 + k * kSortThreads;
    if (i < a.n) atomicAdd(&cnt[(sort_key(a, i) >> a.shift) & (radix - 1)], 1u);  // whole numbers: any order
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) a.hist[(int64_t)d * a.nblk + blockIdx.x] = cnt[d];
}

// One wave per digit: the blocks' counts become places within the digit.
__global__ void __launch_bounds__(256) sort_places_kernel(SortArgs a) {
  const int d = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (d >= 1 << a.bits) return;
  uint32_t* h = a.hist + (int64_t)d * a.nblk;
  uint32_t run = 0;
  for (int b0 = 0; b0 < a.nblk; b0 += 64) {
    const uint32_t c = b0 + lane < a.nblk ? h[b0 + lane] : 0u;
    uint32_t x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (b0 + lane < a.nblk) h[b0 + lane] = run + x - c;
    run += __shfl(x, 63);
  }
  if (lane == 0) a.total[d] = run;
}

// Each wave owns a contiguous strip of the tile, in order: a pair's place is its digit's
// first place, the block's within the digit, the earlier strips' counts, and the digits met
// before it in this strip (a counter per wave and digit, and a ballot match within 64 pairs).
template <int IT>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortArgs a) {
  constexpr int W = kSortThreads / 64;
  __shared__ uint32_t cnt[W][1 << kMaxRadixBits];
  __shared__ uint32_t wsum[W];
  const int radix = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)blockIdx.x * (kSortThreads * IT) + wave * 64 * IT + lane;
  uint32_t key[IT], val[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int64_t i = i0 + 64 * k;
    key[k] = i < a.n ? sort_key(a, i) : 0u;
    val[k] = i < a.n && !a.first ? a.vin[i] : (uint32_t)i;
  }
  for (int i = threadIdx.x; i < W * radix; i += kSortThreads) (&cnt[0][0])[(i / radix) * (1 << kMaxRadixBits) + i % radix] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < IT; ++k)
    if (i0 + 64 * k < a.n) atomicAdd(&cnt[wave][(key[k] >> a.shift) & (radix - 1)], 1u);
  // digits' first places: a running sum over the digits, 256 at a time
  uint32_t first[(1 << kMaxRadixBits) / kSortThreads];
  uint32_t run = 0;
#pragma unroll
  for (int r = 0; r < (1 << kMaxRadixBits) / kSortThreads; ++r) {
    const int d = r * kSortThreads + (int)threadIdx.x;
    const uint32_t c = d < radix ? a.total[d] : 0u;
    uint32_t x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    uint32_t before = run, all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < wave) before += wsum[w];
      all += wsum[w];
    }
    first[r] = before + x - c;
    run += all;
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < (1 << kMaxRadixBits) / kSortThreads; ++r) {
    const int d = r * kSortThreads + (int)threadIdx.x;
    if (d >= radix) continue;
    uint32_t at = first[r] + a.hist[(int64_t)d * a.nblk + blockIdx.x];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t c = cnt[w][d];
      cnt[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
  volatile uint32_t* mine = cnt[wave];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const bool on = i0 + 64 * k < a.n;
    const uint32_t d = (key[k] >> a.shift) & (radix - 1);
    const uint64_t same = same_digit(d, on, a.bits);
    if (on) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const uint32_t at = mine[d] + rank;
      a.kout[at] = key[k];
      a.vout[at] = val[k];
      if (rank == 0) mine[d] = at + __popcll(same);  // after this round's reads: one wave, in order
    }
  }
}

// The whole sort of up to kSmall tokens: 16 waves, strips of 256 tokens, digits of 8 bits.
__global__ void __launch_bounds__(1024) sort_small_kernel(SortArgs a, int passes) {
  constexpr int W = 16, IT = kSmall / 1024, R = 1 << kSmallBits;
  __shared__ uint32_t cnt[W][R];
  __shared__ uint32_t ks[kSmall], vs[kSmall];
  __shared__ uint32_t wsum[R / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = wave * 64 * IT + lane, n = (int)a.n;
  uint32_t key[IT], val[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int i = i0 + 64 * k;
    key[k] = i < n ? sort_key(a, i) : 0u;
    val[k] = (uint32_t)i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * kSmallBits;
    for (int i = threadIdx.x; i < W * R; i += 1024) (&cnt[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < IT; ++k)
      if (i0 + 64 * k < n) atomicAdd(&cnt[wave][(key[k] >> shift) & (R - 1)], 1u);
    __syncthreads();
    const int d0 = threadIdx.x;
    uint32_t c = 0, x = 0;
    if (d0 < R) {  // whole waves: a digit's count over the strips, then the digits' running sum
      for (int w = 0; w < W; ++w) c += cnt[w][d0];
      x = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (lane == 63) wsum[wave] = x;
    }
    __syncthreads();
    if (d0 < R) {
      uint32_t at = x - c;
      for (int w = 0; w < wave; ++w) at += wsum[w];
      for (int w = 0; w < W; ++w) {
        const uint32_t q = cnt[w][d0];
        cnt[w][d0] = at;
        at += q;
      }
    }
    __syncthreads();
    volatile uint32_t* mine = cnt[wave];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const bool on = i0 + 64 * k < n;
      const uint32_t d = (key[k] >> shift) & (R - 1);
      const uint64_t same = same_digit(d, on, kSmallBits);
      if (on) {
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const uint32_t at = mine[d] + rank;
        ks[at] = key[k];
        vs[at] = val[k];
        if (rank == 0) mine[d] = at + __popcll(same);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = i0 + 64 * k;
      if (i < n) key[k] = ks[i], val[k] = vs[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int i = i0 + 64 * k;
    if (i < n) a.kout[i] = key[k], a.vout[i] = val[k];
  }
}

// -------------------------------------------------------------------------------- sums
struct SumArgs {
  const uint32_t* key;
  const uint32_t* val;
  const float* dmz;
  const float* dSz;
  float* part;  // [piece][slot: 0 first run, 1 last run][moment][D]
  float* mw;    // with the update: the parameters, in place
  float* Sw;
  float* dmw;  // may be null with the update
  float* dSw;
  int64_t n, V;
  int D, pieces, piece;
  float c, c2, cap;
};

// Four consecutive floats at any 4-byte alignment: one 16-byte access on gfx950.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ f4 ld4(const float* p, int left) {
  if (left >= 4) return *reinterpret_cast<const f4*>(p);
  f4 v = {p[0], 0.f, 0.f, 0.f};
  if (left > 1) v.y = p[1];
  if (left > 2) v.z = p[2];
  return v;
}
__device__ __forceinline__ void st4(float* p, f4 v, int left) {
  if (left >= 4) {
    *reinterpret_cast<f4*>(p) = v;
    return;
  }
  p[0] = v.x;
  if (left > 1) p[1] = v.y;
  if (left > 2) p[2] = v.z;
}

// The finished sums of up to 4 columns of a category: weighted, stored, applied.
template <bool UPD>
__device__ __forceinline__ void finish(const SumArgs& a, uint32_t cat, int col, f4 sm, f4 ss) {
  const int64_t o = (int64_t)cat * a.D + col;
  const int left = a.D - col;
  f4 S = ld4(a.Sw + o, left);
  const f4 dm = (sm * a.c) * S, dS = (ss * a.c2) * (S * S);
  if (!UPD || a.dmw) {
    st4(a.dmw + o, dm, left);
    st4(a.dSw + o, dS, left);
  }
  if constexpr (UPD) {
    f4 m = ld4(a.mw + o, left);
    float mm[4] = {m.x, m.y, m.z, m.w}, vv[4] = {S.x, S.y, S.z, S.w};
    const float d[4] = {dm.x, dm.y, dm.z, dm.w}, e[4] = {dS.x, dS.y, dS.z, dS.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) capped(mm[i], vv[i], d[i], e[i], a.cap);
    st4(a.mw + o, f4{mm[0], mm[1], mm[2], mm[3]}, left);
    st4(a.Sw + o, f4{vv[0], vv[1], vv[2], vv[3]}, left);
  }
}

// One wave per piece and 256 columns; the rows of kAhead tokens are loaded before they are
// added, in order.
constexpr int kAhead = 8;
template <bool UPD>
__global__ void __launch_bounds__(64) embedding_sum_kernel(SumArgs a) {
  const int lane = threadIdx.x, col = ((int)blockIdx.y * 64 + lane) * 4, P = a.piece, left = a.D - col;
  const int64_t p0 = (int64_t)blockIdx.x * P;
  const int cnt = (int)min((int64_t)P, a.n - p0);
  const uint32_t mykey = lane < cnt ? a.key[p0 + lane] : 0u, myval = lane < cnt ? a.val[p0 + lane] : 0u;
  const uint32_t before = p0 > 0 ? a.key[p0 - 1] : 0xffffffffu;
  const uint32_t after = p0 + cnt < a.n ? a.key[p0 + cnt] : 0xffffffffu;
  const f4 z = {0.f, 0.f, 0.f, 0.f};
  f4 sm = z, ss = z;
  int start = 0;  // first entry of the run being summed
  const uint64_t padding = __ballot(lane < cnt && mykey >= a.V);
  const int real = padding ? __ffsll((long long)padding) - 1 : cnt;  // padding sorts last
  for (int j0 = 0; j0 < real; j0 += kAhead) {
    f4 xm[kAhead], xs[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      xm[u] = xs[u] = z;
      if (j0 + u < real && left > 0) {
        const int64_t at = (int64_t)(uint32_t)__builtin_amdgcn_readlane(myval, j0 + u) * a.D + col;
        xm[u] = ld4(a.dmz + at, left);
        xs[u] = ld4(a.dSz + at, left);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = j0 + u;
      if (j >= real) break;
      sm += xm[u];
      ss += xs[u];
      const uint32_t cat = __builtin_amdgcn_readlane(mykey, j);
      const bool last = j + 1 == cnt;
      const uint32_t next = last ? after : (uint32_t)__builtin_amdgcn_readlane(mykey, j + 1);
      const bool open_right = last && next == cat;
      if (next != cat || open_right) {
        const bool open_left = start == 0 && before == cat;
        if (left > 0) {
          if (open_left || open_right) {
            float* p = a.part + (((int64_t)blockIdx.x * 2 + (open_left ? 0 : 1)) * 2) * a.D + col;
            st4(p, sm, left);
            st4(p + a.D, ss, left);
          } else {
            finish<UPD>(a, cat, col, sm, ss);
          }
        }
        sm = ss = z;
        start = j + 1;
      }
    }
  }
}

// Runs over several pieces: the block of the piece where the run starts adds the partial
// sums, each of its waves a stretch of them in order and then the waves in order, in float64
// (up to n / piece of them).
constexpr int kJoinWaves = 4;
template <bool UPD>
__global__ void __launch_bounds__(64 * kJoinWaves) embedding_join_kernel(SumArgs a) {
  __shared__ double red[kJoinWaves][8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = ((int)blockIdx.y * 64 + lane) * 4, left = a.D - col;
  const int64_t p = blockIdx.x, P = a.piece, last = (p + 1) * P - 1;
  if (last + 1 >= a.n) return;  // the last piece's runs end in it
  const uint32_t cat = a.key[last];
  if (cat >= a.V || a.key[last + 1] != cat) return;
  if (p > 0 && a.key[p * P] == cat && a.key[p * P - 1] == cat) return;  // started in an earlier piece
  // pieces p + 1 .. p + more hold the run's further partial sums
  int64_t more = 0;
  while (true) {
    const int64_t r = p + 1 + more + lane;
    const uint64_t off = ~__ballot(r < a.pieces && a.key[r * P] == cat);
    if (off) {
      more += __ffsll((long long)off) - 1;
      break;
    }
    more += 64;
  }
  double s[8] = {};
  if (left > 0) {
    const int64_t q0 = (more + 1) * wave / kJoinWaves, q1 = (more + 1) * (wave + 1) / kJoinWaves;
#pragma unroll 4
    for (int64_t q = q0; q < q1; ++q) {
      const float* x = a.part + ((p + q) * 2 + (q == 0 ? 1 : 0)) * 2 * a.D + col;
      const f4 m = ld4(x, left), v = ld4(x + a.D, left);
      s[0] += m.x, s[1] += m.y, s[2] += m.z, s[3] += m.w;
      s[4] += v.x, s[5] += v.y, s[6] += v.z, s[7] += v.w;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[wave][e][lane] = s[e];
  __syncthreads();
  if (wave || left <= 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += red[w][e][lane];
  finish<UPD>(a, cat, col, f4{(float)s[0], (float)s[1], (float)s[2], (float)s[3]},
              f4{(float)s[4], (float)s[5], (float)s[6], (float)s[7]});
}

__global__ void __launch_bounds__(256) zero2_kernel(float* __restrict__ x, float* __restrict__ y, int64_t n) {
  const f4 z = {0.f, 0.f, 0.f, 0.f};
  const int64_t step = (int64_t)gridDim.x * 1024;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += step) {
    st4(x + i, z, n - i < 4 ? (int)(n - i) : 4);
    st4(y + i, z, n - i < 4 ? (int)(n - i) : 4);
  }
}

// Tokens of a piece: as many as keep 2048 waves busy, 16 to 64. Shorter pieces leave more
// partial sums (PIECE).
int piece_len(int64_t n, int64_t D) {
  const int64_t cols = cdiv(D, 256);
  int p = 64;
  while (p > 16 && cdiv(n, p) * cols < 2048) p /= 2;
  return p;
}

int64_t pad16(int64_t x) { return (x + 15) & ~int64_t(15); }

struct Layout {
  int64_t keys, hist, total, part, bytes;  // byte offsets: keys: 4 arrays of n
};
Layout layout(int64_t n, int64_t V, int64_t D) {
  const SortPlan p = sort_plan(n, V);
  Layout l;
  l.keys = 0;
  l.hist = pad16(4 * n) * 4;
  l.total = l.hist + pad16(4 * (p.nblk << p.bits));
  l.part = l.total + (4 << kMaxRadixBits);
  l.bytes = l.part + cdiv(n, piece_len(n, D)) * 4 * D * 4;
  return l;
}

template <bool UPD>
void launch_sums(const SumArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.pieces, (unsigned)cdiv(a.D, 256));
  hipLaunchKernelGGL((embedding_sum_kernel<UPD>), grid, dim3(64), 0, s, a);
  if (a.pieces > 1) hipLaunchKernelGGL((embedding_join_kernel<UPD>), grid, dim3(64 * kJoinWaves), 0, s, a);
}

int sorted_impl(const char* what, const void* ids, int type, const float* dmz, const float* dSz, float* mw, float* Sw,
                float* dmw, float* dSw, bool upd, float cap, int64_t n, int64_t V, int64_t D, int64_t pad, double c,
                void* ws, int64_t ws_bytes, hipStream_t s) {
  TAGI_REQUIRE(type >= TAGI_IDS_F32 && type <= TAGI_IDS_I64, "%s: unknown id type %d", what, type);
  TAGI_REQUIRE(n >= 0 && V > 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(n < (1ll << 31) && V < (1ll << 31) && D < (1ll << 21) && V * D < (1ll << 40), "%s: too large", what);
  TAGI_REQUIRE(Sw && (n == 0 || (ids && dmz && dSz)), "%s: null pointer", what);
  TAGI_REQUIRE((dmw == nullptr) == (dSw == nullptr) && (upd || dmw), "%s: null pointer", what);
  const Layout l = layout(n, V, D);
  TAGI_REQUIRE(n == 0 || (ws && ws_bytes >= l.bytes), "%s: workspace too small", what);
  ProfScope ps(FAM_EMBEDDING, s, 0.0, 4.0 * n + 8.0 * n * D + (dmw ? 8.0 * V * D : 0.0));
  if (dmw) hipLaunchKernelGGL(zero2_kernel, dim3(ew_blocks(cdiv(V * D, 4), 256)), dim3(256), 0, s, dmw, dSw, V * D);
  if (n == 0) return check_launch(what);
  const SortPlan p = sort_plan(n, V);
  char* base = static_cast<char*>(ws);
  const int64_t na = pad16(4 * n);
  uint32_t* buf[4];
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(base + l.keys + i * na);
  SortArgs a{};
  a.ids = ids, a.type = type, a.n = n, a.V = V, a.pad = pad, a.nblk = (int)p.nblk, a.bits = p.bits;
  a.hist = reinterpret_cast<uint32_t*>(base + l.hist);
  a.total = reinterpret_cast<uint32_t*>(base + l.total);
  if (n <= kSmall) {
    a.first = 1, a.kout = buf[0], a.vout = buf[1];
    hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(1024), 0, s, a, (int)cdiv(key_bits(V), kSmallBits));
  } else {
    for (int k = 0; k < p.passes; ++k) {
      a.first = k == 0;
      a.kin = buf[2 * ((k + 1) & 1)], a.vin = buf[2 * ((k + 1) & 1) + 1];
      a.kout = buf[2 * (k & 1)], a.vout = buf[2 * (k & 1) + 1];
      a.shift = k * p.bits;
      const dim3 grid((unsigned)p.nblk), block(kSortThreads), digits((unsigned)cdiv(1 << p.bits, 4));
      if (p.items == 4)
        hipLaunchKernelGGL(sort_count_kernel<4>, grid, block, 0, s, a);
      else
        hipLaunchKernelGGL(sort_count_kernel<16>, grid, block, 0, s, a);
      hipLaunchKernelGGL(sort_places_kernel, digits, dim3(256), 0, s, a);
      if (p.items == 4)
        hipLaunchKernelGGL(sort_scatter_kernel<4>, grid, block, 0, s, a);
      else
        hipLaunchKernelGGL(sort_scatter_kernel<16>, grid, block, 0, s, a);
    }
  }
  SumArgs q{};
  q.key = a.kout, q.val = a.vout, q.dmz = dmz, q.dSz = dSz;
  q.part = reinterpret_cast<float*>(base + l.part);
  q.mw = mw, q.Sw = Sw, q.dmw = dmw, q.dSw = dSw, q.n = n, q.V = V, q.D = (int)D;
  q.piece = piece_len(n, D), q.pieces = (int)cdiv(n, q.piece), q.c = (float)c, q.c2 = (float)(c * c), q.cap = cap;
  upd ? launch_sums<true>(q, s) : launch_sums<false>(q, s);
  return check_launch(what);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int tagi_embedding_scaled_fwd(const void* ids, int id_type, const float* mw, const float* Sw, float* mz,
                                         float* Sz, int64_t n, int64_t V, int64_t D, int64_t padding_idx, double scale,
                                         tagi_stream_t stream) {
  const char* what = "tagi_embedding_scaled_fwd";
  TAGI_REQUIRE(id_type >= TAGI_IDS_F32 && id_type <= TAGI_IDS_I64, "%s: unknown id type %d", what, id_type);
  TAGI_REQUIRE(n >= 0 && V > 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(n < (1ll << 31) && V < (1ll << 31) && D < (1ll << 21), "%s: too large", what);
  if (n == 0) return TAGI_OK;
  TAGI_REQUIRE(ids && mw && Sw && mz && Sz, "%s: null pointer", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_EMBEDDING, s, 0.0, 4.0 * n + 16.0 * n * D);
  const bool vec = D % 4 == 0 && al16e(mw) && al16e(Sw) && al16e(mz) && al16e(Sz);
  const int DV = (int)(vec ? D / 4 : D), tpb = DV < 256 ? 256 / DV : 1;
  const dim3 grid((unsigned)cdiv(n, tpb));
  const float c = (float)scale, c2 = (float)(scale * scale);
  if (vec)
    hipLaunchKernelGGL(embedding_lookup_kernel<4>, grid, dim3(256), 0, s, ids, id_type, mw, Sw, mz, Sz, n, V, DV, tpb,
                       padding_idx, c, c2);
  else
    hipLaunchKernelGGL(embedding_lookup_kernel<1>, grid, dim3(256), 0, s, ids, id_type, mw, Sw, mz, Sz, n, V, DV, tpb,
                       padding_idx, c, c2);
  return check_launch(what);
}

extern "C" int64_t tagi_embedding_sorted_ws_bytes(int64_t n, int64_t V, int64_t D) {
  if (n <= 0 || V <= 0 || D <= 0) return 0;
  return layout(n, V, D).bytes;
}

extern "C" int tagi_embedding_sorted_bwd(const void* ids, int id_type, const float* dmz, const float* dSz,
                                         const float* Sw, float* dmw, float* dSw, int64_t n, int64_t V, int64_t D,
                                         int64_t padding_idx, double scale, void* ws, int64_t ws_bytes,
                                         tagi_stream_t stream) {
  return sorted_impl("tagi_embedding_sorted_bwd", ids, id_type, dmz, dSz, nullptr, const_cast<float*>(Sw), dmw, dSw,
                     false, 0.f, n, V, D, padding_idx, scale, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int tagi_embedding_sorted_bwd_update(const void* ids, int id_type, const float* dmz, const float* dSz,
                                                float* mw, float* Sw, float* dmw, float* dSw, float cap_factor,
                                                int64_t n, int64_t V, int64_t D, int64_t padding_idx, double scale,
                                                void* ws, int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_embedding_sorted_bwd_update";
  TAGI_REQUIRE(mw, "%s: null pointer", what);
  TAGI_REQUIRE(cap_factor > 0.f && cap_factor <= 3.4e38f, "%s: cap_factor must be positive and finite", what);
  return sorted_impl(what, ids, id_type, dmz, dSz, mw, Sw, dmw, dSw, true, cap_factor, n, V, D, padding_idx, scale, ws,
                     ws_bytes, (hipStream_t)stream);
}
