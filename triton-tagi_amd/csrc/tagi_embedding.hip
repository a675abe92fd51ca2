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
constexpr int kMaxRadixBits = 11;

// Four consecutive floats at any 4-byte alignment: one 16-byte access on gfx950.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ f4 ld4(const float* p) { return *reinterpret_cast<const f4*>(p); }
__device__ __forceinline__ void st4(float* p, f4 v) { *reinterpret_cast<f4*>(p) = v; }

// A lane's columns of rows of D. The last lane of rows with D % 4 != 0 takes the row's last
// four, so that every lane's loads are one access with no branch between them; only the
// columns no other lane has (from `skip` on) are its own to store. Lanes past the row load its
// first columns and store none: every lane of the wave stays active, as reading another
// lane's register asks for. Rows shorter than four load a column at a time. (Rows of 390 with
// a branch on the row's end instead: 101 us a pass against 70.)
struct Cols {
  int at, skip;  // first column; columns of it that are not the lane's own
};
__device__ __forceinline__ Cols columns(int chunk, int D) {
  Cols c{4 * chunk, 0};
  if (c.at >= D)
    c.at = 0, c.skip = 4;
  else if (c.at + 4 > D && D >= 4)
    c.skip = c.at + 4 - D, c.at = D - 4;
  return c;
}
template <bool WIDE>  // D >= 4
__device__ __forceinline__ f4 ldc(const float* p, int D) {
  if constexpr (WIDE) return ld4(p);
  f4 v = {p[0], 0.f, 0.f, 0.f};
  if (D > 1) v.y = p[1];
  if (D > 2) v.z = p[2];
  return v;
}
template <bool WIDE>
__device__ __forceinline__ void stc(float* p, f4 v, int D, int skip) {
  if (WIDE && skip == 0) {
    st4(p, v);
    return;
  }
  const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e >= skip && e < D) p[e] = x[e];
}

// The category of token t, or V (sorted behind every category) for padding and ids outside
// the table. Float ids are cast toward zero; a NaN is outside.
__device__ __forceinline__ uint32_t category(const void* ids, int type, int64_t t, int64_t V, int64_t pad) {
  int64_t id = -1;
  if (type == TAGI_IDS_F32) {
    const float f = static_cast<const float*>(ids)[t];
    if (f > -1.f && f < 9.2e18f) id = (int64_t)f;
  } else if (type == TAGI_IDS_I32) {
    id = static_cast<const int32_t*>(ids)[t];
  } else {
    id = static_cast<const int64_t*>(ids)[t];
  }
  return (id >= 0 && id < V && id != pad) ? (uint32_t)id : (uint32_t)V;
}

// ------------------------------------------------------------------------------ lookup
// Four columns per thread and moment; a block takes whole tokens. HBM bound: 51949 rows of 391
// from a table that the caches hold take 48 us (163 MB written; a long copy's rate gives 33, and
// four tokens to a thread took the same 48).
template <bool WIDE>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const void* __restrict__ ids, int type,
                                                               const float* __restrict__ mw,
                                                               const float* __restrict__ Sw, float* __restrict__ mz,
                                                               float* __restrict__ Sz, int64_t n, int64_t V, int D,
                                                               int chunks, int tok_per_block, int64_t pad, float c,
                                                               float c2) {
  const int t0 = (int)threadIdx.x / chunks, q0 = (int)threadIdx.x - t0 * chunks;
  if (t0 >= tok_per_block) return;
  for (int64_t t = (int64_t)blockIdx.x * tok_per_block + t0; t < n; t += (int64_t)gridDim.x * tok_per_block) {
    const uint32_t cat = category(ids, type, t, V, pad);
    for (int q = q0; q < chunks; q += 256) {
      const int at = columns(q, D).at;  // columns of two threads get the same values from both
      f4 m = {0.f, 0.f, 0.f, 0.f}, s = m;
      if (cat < V) {
        const int64_t src = (int64_t)cat * D + at;
        m = ldc<WIDE>(mw + src, D) * c, s = ldc<WIDE>(Sw + src, D) * c2;
      }
      stc<WIDE>(mz + t * D + at, m, D, 0);
      stc<WIDE>(Sz + t * D + at, s, D, 0);
    }
  }
}

// -------------------------------------------------------------------------------- sort
// Least-significant-digit radix sort of (category, token index). Per digit: every block
// counts its tile's digits; a wave per digit turns the blocks' counts into places (few blocks
// add them up themselves); every block writes its tile's pairs to them in order. Latency bound:
// 65536 tokens of 131071 categories take 2 digits of 9 bits, 18 us a digit. Up to kSmall tokens
// one block does all of it in LDS: a launch instead of three per digit (4096 tokens x 64 over
// 50000 rows: 25 us a call against 40, 16 tokens 16 against 30; 16384 tokens in one block took
// 24 us against 15 for one digit).
constexpr int kSmall = 4096, kSmallBits = 8;
// Up to this many blocks and counts in all, every block adds the counts up itself, a launch less
// per digit (us a call: 16 blocks of 7 bits 25 -> 23, 20 of 8 bits 69 -> 65; 32 of 10 bits
// 43 -> 45, 64 of 9 67 -> 71).
constexpr int kFewBlocks = 32, kFewCounts = 16384;

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
  uint32_t* hist;   // [digit][block]: counts, then places within the digit; few blocks: [block][digit], counts
  uint32_t* total;  // [digit]
  int64_t n, V, pad;
  int nblk, shift, bits;
  // Zeros for the deltas of the rows that do not occur: the sort waits on latency, the fill on
  // bandwidth, so each launch of the sort takes a share of it in blocks after its own `work`.
  float* z0;
  float* z1;
  int64_t f0, f1;
  int work;
};

__device__ __forceinline__ bool fills(const SortArgs& a) {
  if ((int)blockIdx.x < a.work) return false;
  const f4 z = {0.f, 0.f, 0.f, 0.f};
  const int64_t threads = blockDim.x, step = (int64_t)(gridDim.x - a.work) * threads * 4;
  for (int64_t i = a.f0 + ((int64_t)(blockIdx.x - a.work) * threads + threadIdx.x) * 4; i < a.f1; i += step) {
    if (i + 4 <= a.f1) {
      st4(a.z0 + i, z);
      st4(a.z1 + i, z);
    } else {
      for (int64_t j = i; j < a.f1; ++j) a.z0[j] = a.z1[j] = 0.f;
    }
  }
  return true;
}

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

template <int IT, bool FEW>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  if (fills(a)) return;
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
  for (int d = threadIdx.x; d < radix; d += kSortThreads)
    a.hist[FEW ? (int64_t)blockIdx.x * radix + d : (int64_t)d * a.nblk + blockIdx.x] = cnt[d];
}

// One wave per digit: the blocks' counts become places within the digit.
__global__ void __launch_bounds__(256) sort_places_kernel(SortArgs a) {
  if (fills(a)) return;
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
template <int IT, bool FEW>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortArgs a) {
  if (fills(a)) return;
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
  uint32_t inside[(1 << kMaxRadixBits) / kSortThreads];  // the block's first place within the digit
  uint32_t run = 0;
#pragma unroll
  for (int r = 0; r < (1 << kMaxRadixBits) / kSortThreads; ++r) {
    if (r * kSortThreads >= radix) break;
    const int d = r * kSortThreads + (int)threadIdx.x;
    uint32_t c = 0, in = 0;
    if (d < radix) {
      if constexpr (FEW) {
#pragma unroll 8
        for (int b = 0; b < a.nblk; ++b) {
          const uint32_t h = a.hist[(int64_t)b * radix + d];
          c += h;
          in += b < (int)blockIdx.x ? h : 0u;
        }
      } else {
        c = a.total[d], in = a.hist[(int64_t)d * a.nblk + blockIdx.x];
      }
    }
    inside[r] = in;
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
    uint32_t at = first[r] + inside[r];
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
      if (rank == 0) mine[d] = at + __popcll(same);  // after these reads: one wave, in order
    }
  }
}

// The whole sort of up to kSmall tokens: 16 waves, strips of 256 tokens, digits of 8 bits.
__global__ void __launch_bounds__(1024) sort_small_kernel(SortArgs a, int passes) {
  if (fills(a)) return;
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

// The finished sums of a lane's columns of a category: weighted, stored, applied.
template <bool UPD, bool WIDE>
__device__ __forceinline__ void finish(const SumArgs& a, uint32_t cat, const Cols& c, f4 sm, f4 ss, f4 m, f4 S) {
  const int64_t o = (int64_t)cat * a.D + c.at;
  const f4 dm = (sm * a.c) * S, dS = (ss * a.c2) * (S * S);
  if (!UPD || a.dmw) {
    stc<WIDE>(a.dmw + o, dm, a.D, c.skip);
    stc<WIDE>(a.dSw + o, dS, a.D, c.skip);
  }
  if constexpr (UPD) {
    float mm[4] = {m.x, m.y, m.z, m.w}, vv[4] = {S.x, S.y, S.z, S.w};
    const float d[4] = {dm.x, dm.y, dm.z, dm.w}, e[4] = {dS.x, dS.y, dS.z, dS.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) capped(mm[i], vv[i], d[i], e[i], a.cap);
    stc<WIDE>(a.mw + o, f4{mm[0], mm[1], mm[2], mm[3]}, a.D, c.skip);
    stc<WIDE>(a.Sw + o, f4{vv[0], vv[1], vv[2], vv[3]}, a.D, c.skip);
  }
}

// One wave per piece and 256 columns; the rows of AHEAD tokens, and the table's rows of the
// runs that end among them, are loaded before the tokens are added in order. Most categories
// of a large table have one token: without that each would wait for its own row.
template <bool UPD, bool WIDE, int AHEAD>
__global__ void __launch_bounds__(64) embedding_sum_kernel(SumArgs a) {
  const int lane = threadIdx.x, P = a.piece;
  const Cols c = columns((int)blockIdx.y * 64 + lane, a.D);
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
  const auto category_at = [&](int j) -> uint32_t {
    return j < cnt ? (uint32_t)__builtin_amdgcn_readlane(mykey, j) : after;
  };
  for (int j0 = 0; j0 < real; j0 += AHEAD) {
    f4 xm[AHEAD], xs[AHEAD], rm[UPD ? AHEAD : 1], rS[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = j0 + u;
      xm[u] = xs[u] = rS[u] = z;
      if constexpr (UPD) rm[u] = z;
      if (j < real) {
        const int64_t at = (int64_t)(uint32_t)__builtin_amdgcn_readlane(myval, j) * a.D + c.at;
        xm[u] = ldc<WIDE>(a.dmz + at, a.D);
        xs[u] = ldc<WIDE>(a.dSz + at, a.D);
        const uint32_t cat = category_at(j);
        if (category_at(j + 1) != cat) {
          const int64_t o = (int64_t)cat * a.D + c.at;
          rS[u] = ldc<WIDE>(a.Sw + o, a.D);
          if constexpr (UPD) rm[u] = ldc<WIDE>(a.mw + o, a.D);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = j0 + u;
      if (j >= real) break;
      sm += xm[u];
      ss += xs[u];
      const uint32_t cat = category_at(j), next = category_at(j + 1);
      const bool open_right = j + 1 == cnt && next == cat;
      if (next != cat || open_right) {
        const bool open_left = start == 0 && before == cat;
        if (open_left || open_right) {
          float* p = a.part + (((int64_t)blockIdx.x * 2 + (open_left ? 0 : 1)) * 2) * a.D + c.at;
          stc<WIDE>(p, sm, a.D, c.skip);
          stc<WIDE>(p + a.D, ss, a.D, c.skip);
        } else {
          finish<UPD, WIDE>(a, cat, c, sm, ss, rm[UPD ? u : 0], rS[u]);
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
template <bool UPD, bool WIDE>
__global__ void __launch_bounds__(64 * kJoinWaves) embedding_join_kernel(SumArgs a) {
  __shared__ double red[kJoinWaves][8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Cols c = columns((int)blockIdx.y * 64 + lane, a.D);
  const int64_t p = blockIdx.x, P = a.piece, last = (p + 1) * P - 1;
  if (last + 1 >= a.n) return;  // the last piece's runs end in it
  // the keys that decide, and those of the next 64 pieces, in one round trip
  const auto first_key = [&](int64_t r) { return r < a.pieces ? a.key[r * P] : 0xffffffffu; };
  const uint32_t cat = a.key[last], after = a.key[last + 1], head = a.key[p * P];
  const uint32_t before = p > 0 ? a.key[p * P - 1] : 0xffffffffu;
  uint32_t ahead = first_key(p + 1 + lane);
  if (cat >= a.V || after != cat) return;
  if (head == cat && before == cat) return;  // started in an earlier piece
  const int64_t o = (int64_t)cat * a.D + c.at;
  f4 S = {0.f, 0.f, 0.f, 0.f}, m = S;
  if (wave == 0) {
    S = ldc<WIDE>(a.Sw + o, a.D);
    if constexpr (UPD) m = ldc<WIDE>(a.mw + o, a.D);
  }
  // pieces p + 1 .. p + more hold the run's further partial sums
  int64_t more = 0;
  while (true) {
    const uint64_t off = ~__ballot(ahead == cat);
    if (off) {
      more += __ffsll((long long)off) - 1;
      break;
    }
    more += 64;
    ahead = first_key(p + 1 + more + lane);
  }
  double s[8] = {};
  const int64_t q0 = (more + 1) * wave / kJoinWaves, q1 = (more + 1) * (wave + 1) / kJoinWaves;
#pragma unroll 8
  for (int64_t q = q0; q < q1; ++q) {
    const float* x = a.part + ((p + q) * 2 + (q == 0 ? 1 : 0)) * 2 * a.D + c.at;
    const f4 y = ldc<WIDE>(x, a.D), v = ldc<WIDE>(x + a.D, a.D);
    s[0] += y.x, s[1] += y.y, s[2] += y.z, s[3] += y.w;
    s[4] += v.x, s[5] += v.y, s[6] += v.z, s[7] += v.w;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[wave][e][lane] = s[e];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += red[w][e][lane];
  finish<UPD, WIDE>(a, cat, c, f4{(float)s[0], (float)s[1], (float)s[2], (float)s[3]},
              f4{(float)s[4], (float)s[5], (float)s[6], (float)s[7]}, m, S);
}

// Tokens of a piece: as many as keep 2048 waves busy, 16 to 64. Shorter pieces leave more
// partial sums. (16384 tokens x 256: pieces of 64 25 us for the sums, of 16 7.)
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

// A launch has fewer than 2^32 threads: the joins' blocks for pieces of 64 tokens, which more
// tokens than 2^17 always have.
constexpr int64_t kMaxSorted = (1ll << 30) - 64;
static_assert(kMaxSorted / 64 * 64 * kJoinWaves < (1ll << 32), "blocks of the joins");

constexpr int kAhead = 4;
template <bool UPD, bool WIDE>
void launch_sums(const SumArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.pieces, (unsigned)cdiv(a.D, 256));
  hipLaunchKernelGGL((embedding_sum_kernel<UPD, WIDE, kAhead>), grid, dim3(64), 0, s, a);
  if (a.pieces > 1) hipLaunchKernelGGL((embedding_join_kernel<UPD, WIDE>), grid, dim3(64 * kJoinWaves), 0, s, a);
}

int sorted_impl(const char* what, const void* ids, int type, const float* dmz, const float* dSz, float* mw, float* Sw,
                float* dmw, float* dSw, bool upd, float cap, int64_t n, int64_t V, int64_t D, int64_t pad, double c,
                void* ws, int64_t ws_bytes, hipStream_t s) {
  TAGI_REQUIRE(type >= TAGI_IDS_F32 && type <= TAGI_IDS_I64, "%s: unknown id type %d", what, type);
  TAGI_REQUIRE(n >= 0 && V > 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(n <= kMaxSorted && V < (1ll << 31) && D < (1ll << 21) && V * D < (1ll << 40), "%s: too large", what);
  TAGI_REQUIRE(Sw && (n == 0 || (ids && dmz && dSz)), "%s: null pointer", what);
  TAGI_REQUIRE((dmw == nullptr) == (dSw == nullptr) && (upd || dmw), "%s: null pointer", what);
  const Layout l = layout(n, V, D);
  TAGI_REQUIRE(n == 0 || (ws && ws_bytes >= l.bytes), "%s: workspace too small", what);
  ProfScope ps(FAM_EMBEDDING, s, 0.0, 4.0 * n + 8.0 * n * D + (dmw ? 8.0 * V * D : 0.0));
  const SortPlan p = sort_plan(n, V);
  char* base = static_cast<char*>(ws);
  const int64_t na = pad16(4 * n);
  uint32_t* buf[4];
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(base + l.keys + i * na);
  SortArgs a{};
  a.ids = ids, a.type = type, a.n = n, a.V = V, a.pad = pad, a.nblk = (int)p.nblk, a.bits = p.bits;
  a.hist = reinterpret_cast<uint32_t*>(base + l.hist);
  a.total = reinterpret_cast<uint32_t*>(base + l.total);
  a.z0 = dmw, a.z1 = dSw;
  const bool small = n <= kSmall;
  const bool few = p.nblk <= kFewBlocks && p.nblk << p.bits <= kFewCounts;
  const int launches = small ? 1 : (few ? 2 : 3) * p.passes;
  const int64_t share = dmw ? cdiv(cdiv(V * D, launches), 4) * 4 : 0;
  int done = 0;
  // the next launch's grid: `work` blocks, and those for its share of the zeros
  const auto grid = [&](int64_t work, int threads) {
    a.work = (int)work;
    a.f0 = done * share, a.f1 = dmw ? (a.f0 + share < V * D ? a.f0 + share : V * D) : 0;
    ++done;
    int64_t fill = a.f1 > a.f0 ? cdiv(cdiv(a.f1 - a.f0, 4), threads) : 0;
    if (fill > 1024) fill = 1024;
    return dim3((unsigned)(work + fill));
  };
  if (small) {
    a.first = 1, a.kout = buf[0], a.vout = buf[1];
    const dim3 g = grid(n > 0 ? 1 : 0, 1024);
    if (g.x) hipLaunchKernelGGL(sort_small_kernel, g, dim3(1024), 0, s, a, (int)cdiv(key_bits(V), kSmallBits));
    if (n == 0) return check_launch(what);
  } else {
    for (int k = 0; k < p.passes; ++k) {
      a.first = k == 0;
      a.kin = buf[2 * ((k + 1) & 1)], a.vin = buf[2 * ((k + 1) & 1) + 1];
      a.kout = buf[2 * (k & 1)], a.vout = buf[2 * (k & 1) + 1];
      a.shift = k * p.bits;
      const dim3 block(kSortThreads);
      dim3 g = grid(p.nblk, kSortThreads);
      if (few)
        hipLaunchKernelGGL((sort_count_kernel<4, true>), g, block, 0, s, a);
      else if (p.items == 4)
        hipLaunchKernelGGL((sort_count_kernel<4, false>), g, block, 0, s, a);
      else
        hipLaunchKernelGGL((sort_count_kernel<16, false>), g, block, 0, s, a);
      if (!few) {
        g = grid(cdiv(1 << p.bits, 4), kSortThreads);
        hipLaunchKernelGGL(sort_places_kernel, g, block, 0, s, a);
      }
      g = grid(p.nblk, kSortThreads);
      if (few)
        hipLaunchKernelGGL((sort_scatter_kernel<4, true>), g, block, 0, s, a);
      else if (p.items == 4)
        hipLaunchKernelGGL((sort_scatter_kernel<4, false>), g, block, 0, s, a);
      else
        hipLaunchKernelGGL((sort_scatter_kernel<16, false>), g, block, 0, s, a);
    }
  }
  SumArgs q{};
  q.key = a.kout, q.val = a.vout, q.dmz = dmz, q.dSz = dSz;
  q.part = reinterpret_cast<float*>(base + l.part);
  q.mw = mw, q.Sw = Sw, q.dmw = dmw, q.dSw = dSw, q.n = n, q.V = V, q.D = (int)D;
  q.piece = piece_len(n, D), q.pieces = (int)cdiv(n, q.piece), q.c = (float)c, q.c2 = (float)(c * c), q.cap = cap;
  if (D >= 4)
    upd ? launch_sums<true, true>(q, s) : launch_sums<false, true>(q, s);
  else
    upd ? launch_sums<true, false>(q, s) : launch_sums<false, false>(q, s);
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
  TAGI_REQUIRE(n < (1ll << 30) && V < (1ll << 31) && D < (1ll << 21), "%s: too large", what);
  if (n == 0) return TAGI_OK;
  TAGI_REQUIRE(ids && mw && Sw && mz && Sz, "%s: null pointer", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_EMBEDDING, s, 0.0, 4.0 * n + 16.0 * n * D);
  const int chunks = (int)cdiv(D, 4), tpb = chunks < 256 ? 256 / chunks : 1;
  const int64_t blocks = cdiv(n, tpb);  // a launch has fewer than 2^32 threads
  const dim3 grid((unsigned)(blocks < (1 << 23) ? blocks : (1 << 23)));
  const float c = (float)scale, c2 = (float)(scale * scale);
  const auto kernel = D < 4 ? embedding_lookup_kernel<false> : embedding_lookup_kernel<true>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, ids, id_type, mw, Sw, mz, Sz, n, V, (int)D, chunks, tpb,
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
