// Scaled embedding lookup, and the parameter deltas of its table by sorted tokens.
//
//   mz[t] = c mw[id_t],  Sz[t] = c^2 Sw[id_t]
//   dmw[v] = c Sw[v] sum_{t: id_t = v} dmz[t],  dSw[v] = (c Sw[v])^2 sum_{t: id_t = v} dSz[t]
//
// Ids equal to padding_idx or outside [0, V) look up zeros and add nothing. The deltas sort
// the tokens by category (stable, so a category's tokens keep their order), cut the sorted
// list into pieces of kPiece tokens and let one wavefront sum each piece's runs of equal
// ids: O(N) whatever the table holds, and a category that half of the batch asks for is
// spread over as many wavefronts as it has pieces. A run that crosses a piece's border
// leaves partial sums, which a second kernel adds in piece order. Every order is fixed by
// the ids alone: results are deterministic, with no float atomics.
#include "tagi_common.h"
#include "tagi_moments.h"

namespace tagi {
namespace {

constexpr int kPiece = 64;       // sorted tokens per wavefront of the sums
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
// counts its tile's digits, one block turns the counts into places, every block writes its
// tile's pairs to them in order.
struct SortPlan {
  int64_t tile, nblk;
  int bits, passes;
};
SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  int total = 1;
  while ((V >> total) != 0) ++total;  // keys are 0..V
  p.passes = (int)cdiv(total, kMaxRadixBits);
  p.bits = (int)cdiv(total, p.passes);
  p.tile = cdiv(cdiv(n, 256), kSortThreads) * kSortThreads;
  if (p.tile < 1024) p.tile = 1024;
  p.nblk = cdiv(n, p.tile);
  return p;
}

struct SortArgs {
  const void* ids;
  int type, first;
  const uint32_t* kin;
  const uint32_t* vin;
  uint32_t* kout;
  uint32_t* vout;
  uint32_t* hist;  // [digit][block]
  int64_t n, V, pad, tile;
  int nblk, shift, bits;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t i) {
  return a.first ? category(a.ids, a.type, i, a.V, a.pad) : a.kin[i];
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  __shared__ uint32_t cnt[1 << kMaxRadixBits];
  const int radix = 1 << a.bits;
  for (int d = threadIdx.x; d < radix; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads)
    atomicAdd(&cnt[(sort_key(a, i) >> a.shift) & (radix - 1)], 1u);  // whole numbers: any order
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) a.hist[(int64_t)d * a.nblk + blockIdx.x] = cnt[d];
}

__global__ void __launch_bounds__(1024) sort_places_kernel(uint32_t* __restrict__ hist, int total) {
  __shared__ uint32_t sums[1024];
  const int per = (total + 1023) / 1024, i0 = min(total, (int)threadIdx.x * per), i1 = min(total, i0 + per);
  uint32_t s = 0;
  for (int i = i0; i < i1; ++i) s += hist[i];
  sums[threadIdx.x] = s;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const uint32_t x = threadIdx.x >= (unsigned)o ? sums[threadIdx.x - o] : 0u;
    __syncthreads();
    sums[threadIdx.x] += x;
    __syncthreads();
  }
  uint32_t run = sums[threadIdx.x] - s;
  for (int i = i0; i < i1; ++i) {
    const uint32_t c = hist[i];
    hist[i] = run;
    run += c;
  }
}

// Each wave owns a contiguous strip of the tile, in order: a pair's place is its digit's
// place for the block, plus the earlier strips' counts, plus the digits met before it in
// this strip (a counter per wave and digit, and a ballot match within 64 pairs).
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortArgs a) {
  constexpr int W = kSortThreads / 64;
  __shared__ uint32_t cnt[W][1 << kMaxRadixBits];
  const int radix = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < W * radix; i += kSortThreads) cnt[i / radix][i % radix] = 0;
  __syncthreads();
  const int64_t strip = a.tile / W, i0 = (int64_t)blockIdx.x * a.tile + wave * strip, i1 = min(a.n, i0 + strip);
  for (int64_t i = i0 + lane; i < i1; i += 64) atomicAdd(&cnt[wave][(sort_key(a, i) >> a.shift) & (radix - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) {
    uint32_t run = a.hist[(int64_t)d * a.nblk + blockIdx.x];
    for (int w = 0; w < W; ++w) {
      const uint32_t c = cnt[w][d];
      cnt[w][d] = run;
      run += c;
    }
  }
  __syncthreads();
  volatile uint32_t* mine = cnt[wave];
  for (int64_t b = i0; b < i1; b += 64) {
    const int64_t i = b + lane;
    const bool on = i < i1;
    const uint32_t key = on ? sort_key(a, i) : 0u;
    const uint32_t d = (key >> a.shift) & (radix - 1);
    uint64_t same = __ballot(on);
    for (int bit = 0; bit < a.bits; ++bit) {
      const uint64_t m = __ballot((d >> bit) & 1);
      same &= ((d >> bit) & 1) ? m : ~m;
    }
    if (on) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const uint32_t at = mine[d] + rank;
      a.kout[at] = key;
      a.vout[at] = a.first ? (uint32_t)i : a.vin[i];
      if (rank == 0) mine[d] = at + __popcll(same);  // after this round's reads: one wave, in order
    }
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
  int D, pieces;
  float c, c2, cap;
};

// The finished sums of 1 or 4 columns of a category: weighted, stored, applied.
template <int VEC, bool UPD>
__device__ __forceinline__ void finish(const SumArgs& a, uint32_t cat, int col, const float* sm, const float* ss) {
  const int64_t o = (int64_t)cat * a.D + col;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float S = a.Sw[o + e];
    const float dm = (sm[e] * a.c) * S, dS = (ss[e] * a.c2) * (S * S);
    if (!UPD || a.dmw) {
      a.dmw[o + e] = dm;
      a.dSw[o + e] = dS;
    }
    if constexpr (UPD) {
      float m = a.mw[o + e];
      capped(m, S, dm, dS, a.cap);
      a.mw[o + e] = m;
      a.Sw[o + e] = S;
    }
  }
}

template <int VEC, bool UPD>
__global__ void __launch_bounds__(64) embedding_sum_kernel(SumArgs a) {
  const int lane = threadIdx.x, col = ((int)blockIdx.y * 64 + lane) * VEC;
  const int64_t p0 = (int64_t)blockIdx.x * kPiece;
  const int cnt = (int)min((int64_t)kPiece, a.n - p0);
  const uint32_t mykey = lane < cnt ? a.key[p0 + lane] : 0u, myval = lane < cnt ? a.val[p0 + lane] : 0u;
  const uint32_t before = p0 > 0 ? a.key[p0 - 1] : 0xffffffffu;
  const uint32_t after = p0 + cnt < a.n ? a.key[p0 + cnt] : 0xffffffffu;
  const bool live = col < a.D;
  float sm[VEC] = {}, ss[VEC] = {};
  int start = 0;  // first entry of the run being summed
  for (int j = 0; j < cnt; ++j) {
    const uint32_t cat = __builtin_amdgcn_readlane(mykey, j);
    if (cat >= a.V) break;  // padding sorts last
    const uint32_t t = __builtin_amdgcn_readlane(myval, j);
    if (live) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        sm[e] += a.dmz[(int64_t)t * a.D + col + e];
        ss[e] += a.dSz[(int64_t)t * a.D + col + e];
      }
    }
    const uint32_t next = j + 1 < cnt ? (uint32_t)__builtin_amdgcn_readlane(mykey, j + 1) : after;
    const bool open_right = j + 1 == cnt && next == cat;
    if (next != cat || open_right) {
      const bool open_left = start == 0 && before == cat;
      if (live) {
        if (open_left || open_right) {
          float* p = a.part + (((int64_t)blockIdx.x * 2 + (open_left ? 0 : 1)) * 2) * a.D + col;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            p[e] = sm[e];
            p[a.D + e] = ss[e];
          }
        } else {
          finish<VEC, UPD>(a, cat, col, sm, ss);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sm[e] = ss[e] = 0.f;
      start = j + 1;
    }
  }
}

// Runs over several pieces: the block of the piece where the run starts adds the partial
// sums in piece order, in float64 (up to N / kPiece of them).
template <int VEC, bool UPD>
__global__ void __launch_bounds__(64) embedding_join_kernel(SumArgs a) {
  const int col = ((int)blockIdx.y * 64 + (int)threadIdx.x) * VEC;
  const int64_t p = blockIdx.x, last = (p + 1) * kPiece - 1;
  if (last + 1 >= a.n) return;  // the last piece's runs end in it
  const uint32_t cat = a.key[last];
  if (cat >= a.V || a.key[last + 1] != cat) return;
  if (p > 0 && a.key[p * kPiece] == cat && a.key[p * kPiece - 1] == cat) return;  // started in an earlier piece
  if (col >= a.D) return;
  double sm[VEC], ss[VEC];
  const float* q = a.part + (p * 2 + 1) * 2 * a.D + col;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sm[e] = q[e], ss[e] = q[a.D + e];
  for (int64_t r = p + 1; r < a.pieces && a.key[r * kPiece] == cat; ++r) {
    const float* x = a.part + (r * 2) * 2 * a.D + col;
#pragma unroll
    for (int e = 0; e < VEC; ++e) sm[e] += x[e], ss[e] += x[a.D + e];
  }
  float fm[VEC], fs[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) fm[e] = (float)sm[e], fs[e] = (float)ss[e];
  finish<VEC, UPD>(a, cat, col, fm, fs);
}

__global__ void __launch_bounds__(256) zero2_kernel(float* __restrict__ x, float* __restrict__ y, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) x[i] = y[i] = 0.f;
}

int64_t pad16(int64_t x) { return (x + 15) & ~int64_t(15); }

struct Layout {
  int64_t keys, hist, part, total;  // byte offsets: keys: 4 arrays of n
};
Layout layout(int64_t n, int64_t V, int64_t D) {
  const SortPlan p = sort_plan(n, V);
  Layout l;
  l.keys = 0;
  l.hist = pad16(4 * n) * 4;
  l.part = l.hist + pad16(4 * (p.nblk << p.bits));
  l.total = l.part + cdiv(n, kPiece) * 4 * D * 4;
  return l;
}

template <int VEC, bool UPD>
void launch_sums(const SumArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.pieces, (unsigned)cdiv(a.D, 64 * VEC));
  hipLaunchKernelGGL((embedding_sum_kernel<VEC, UPD>), grid, dim3(64), 0, s, a);
  if (a.pieces > 1) hipLaunchKernelGGL((embedding_join_kernel<VEC, UPD>), grid, dim3(64), 0, s, a);
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
  TAGI_REQUIRE(n == 0 || (ws && ws_bytes >= l.total), "%s: workspace too small", what);
  ProfScope ps(FAM_EMBEDDING, s, 0.0, 4.0 * n + 8.0 * n * D + (dmw ? 8.0 * V * D : 0.0));
  if (dmw) hipLaunchKernelGGL(zero2_kernel, dim3(ew_blocks(V * D, 256)), dim3(256), 0, s, dmw, dSw, V * D);
  if (n == 0) return check_launch(what);
  const SortPlan p = sort_plan(n, V);
  char* base = static_cast<char*>(ws);
  const int64_t na = pad16(4 * n);
  uint32_t* buf[4];
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(base + l.keys + i * na);
  SortArgs a{};
  a.ids = ids, a.type = type, a.hist = reinterpret_cast<uint32_t*>(base + l.hist);
  a.n = n, a.V = V, a.pad = pad, a.tile = p.tile, a.nblk = (int)p.nblk, a.bits = p.bits;
  for (int k = 0; k < p.passes; ++k) {
    a.first = k == 0;
    a.kin = buf[2 * ((k + 1) & 1)], a.vin = buf[2 * ((k + 1) & 1) + 1];
    a.kout = buf[2 * (k & 1)], a.vout = buf[2 * (k & 1) + 1];
    a.shift = k * p.bits;
    hipLaunchKernelGGL(sort_count_kernel, dim3(a.nblk), dim3(kSortThreads), 0, s, a);
    hipLaunchKernelGGL(sort_places_kernel, dim3(1), dim3(1024), 0, s, a.hist, a.nblk << a.bits);
    hipLaunchKernelGGL(sort_scatter_kernel, dim3(a.nblk), dim3(kSortThreads), 0, s, a);
  }
  SumArgs q{};
  q.key = a.kout, q.val = a.vout, q.dmz = dmz, q.dSz = dSz;
  q.part = reinterpret_cast<float*>(base + l.part);
  q.mw = mw, q.Sw = Sw, q.dmw = dmw, q.dSw = dSw, q.n = n, q.V = V, q.D = (int)D;
  q.pieces = (int)cdiv(n, kPiece), q.c = (float)c, q.c2 = (float)(c * c), q.cap = cap;
  const bool vec = D % 4 == 0;
  if (upd)
    vec ? launch_sums<4, true>(q, s) : launch_sums<1, true>(q, s);
  else
    vec ? launch_sums<4, false>(q, s) : launch_sums<1, false>(q, s);
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
  return layout(n, V, D).total;
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
