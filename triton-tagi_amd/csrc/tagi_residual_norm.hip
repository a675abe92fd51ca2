// Sum of two Gaussian streams and its RMSNorm, forward and backward.
//
//   ms = ma + mr,  Ss = Sa + Sr
//   inv = 1 / sqrt(mean(ms^2 + Ss) + eps)                         (one per row)
//   mz = ms inv g,  Sz = inv^2 (Ss (g^2 + Sg) + Sg ms^2)
// backward, from the deltas at z and (optionally) at the sum:
//   dm = dmz inv g + dms,  dS = dSz (inv g)^2 + dSs               (the same for both inputs)
//   dg = Sg sum_rows dmz inv ms,  dSg = Sg^2 sum_rows dSz (inv ms)^2
#include "tagi_common.h"

namespace tagi {
namespace {

// Four consecutive floats at any 4-byte alignment: one 16-byte access on gfx950.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

template <bool NT>
__device__ __forceinline__ f4 ld(const float* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const f4*>(p));
  return *reinterpret_cast<const f4*>(p);
}
template <bool NT>
__device__ __forceinline__ void st(float* p, f4 v) {
  if constexpr (NT)
    __builtin_nontemporal_store(v, reinterpret_cast<f4*>(p));
  else
    *reinterpret_cast<f4*>(p) = v;
}
// A thread's four columns. The last chunk of a row with D % 4 != 0 is the row's last four, of
// which the first `skip` are the chunk's before as well: every load is one access with no
// branch between them. Threads past the row take its first columns, all skipped. D >= 4.
struct Cols {
  int at, skip;
};
__device__ __forceinline__ Cols columns(int chunk, int D) {
  Cols c{4 * chunk, 0};
  if (c.at >= D)
    c.at = 0, c.skip = 4;
  else if (c.at + 4 > D)
    c.skip = c.at + 4 - D, c.at = D - 4;
  return c;
}
__device__ __forceinline__ f4 own(f4 v, int skip) {  // zeros for the skipped
  return f4{skip > 0 ? 0.f : v.x, skip > 1 ? 0.f : v.y, skip > 2 ? 0.f : v.z, skip > 3 ? 0.f : v.w};
}

// Sum over the TPR threads of a row (a wave, or the whole block).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) x += __shfl_xor(x, w);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) x += red[w];
  }
  return x;
}

// Blocks in two dimensions: a launch has fewer than 2^32 threads in one.
inline dim3 row_grid(int64_t blocks) {
  const int64_t x = blocks < (1 << 20) ? blocks : (1 << 20);
  return dim3((unsigned)x, (unsigned)cdiv(blocks, x));
}
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// One pass: TPR threads hold a row's sums in registers (NV chunks of four each) between the
// statistic and the output, so every input is read and every output written once. HBM bound:
// 16384 x 4096 moves 2.15 GB in 380 us (5.65 TB/s; a copy kernel reaches 6.26 here), 65536 x 256
// 537 MB in 93 us.
template <int TPR, int NV, bool NT>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) add_rms_norm_kernel(
    const float* __restrict__ ma, const float* __restrict__ Sa, const float* __restrict__ mr,
    const float* __restrict__ Sr, const float* __restrict__ mw, const float* __restrict__ Sw, float* __restrict__ mz,
    float* __restrict__ Sz, float* __restrict__ ms, float* __restrict__ Ss, float* __restrict__ inv_rms, int64_t rows,
    int D, float eps) {
  __shared__ float red[TPR / 64];
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;  // rows of a block
  const int t = (int)threadIdx.x % TPR;
  const int64_t row = row_block() * RPB + (int)threadIdx.x / TPR, o = row * D;
  if (row >= rows) return;  // TPR > 64 has one row a block: no thread of it leaves
  f4 m[NV], v[NV];
  float acc = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t at = o + columns(t + j * TPR, D).at;
    const f4 a = ld<NT>(ma + at), b = ld<NT>(mr + at), x = ld<NT>(Sa + at), y = ld<NT>(Sr + at);
    m[j] = a + b, v[j] = x + y;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const f4 q = own(m[j] * m[j] + v[j], columns(t + j * TPR, D).skip);
    acc += (q.x + q.y) + (q.z + q.w);
  }
  const float inv = 1.f / sqrtf(row_sum<TPR>(acc, red) / (float)D + eps);
  if (t == 0) inv_rms[row] = inv;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Cols c = columns(t + j * TPR, D);
    if (c.skip == 4) continue;
    const int64_t at = o + c.at;
    const f4 g = *reinterpret_cast<const f4*>(mw + c.at), sg = *reinterpret_cast<const f4*>(Sw + c.at);
    // columns of two threads get the same values from both
    st<NT>(ms + at, m[j]);
    if (Ss) st<NT>(Ss + at, v[j]);
    st<NT>(mz + at, m[j] * inv * g);
    st<NT>(Sz + at, inv * inv * (v[j] * (g * g + sg) + sg * (m[j] * m[j])));
  }
}

struct FwdArgs {
  const float *ma, *Sa, *mr, *Sr, *mw, *Sw;
  float *mz, *Sz, *ms, *Ss, *inv;
  int64_t rows;
  int D;
  float eps;
};
__device__ __forceinline__ void write_value(const FwdArgs& a, int64_t at, int c, float inv) {
  const float m = a.ma[at] + a.mr[at], v = a.Sa[at] + a.Sr[at], g = a.mw[c], sg = a.Sw[c];
  a.ms[at] = m;
  if (a.Ss) a.Ss[at] = v;
  a.mz[at] = m * inv * g;
  a.Sz[at] = inv * inv * (v * (g * g + sg) + sg * (m * m));
}

// Rows too long for registers: the inputs are read twice.
__global__ void __launch_bounds__(1024) add_rms_norm_long_kernel(FwdArgs a) {
  __shared__ float red[16];
  const int64_t row = row_block(), o = row * a.D;
  if (row >= a.rows) return;
  float acc = 0.f;
  for (int c = threadIdx.x; c < a.D; c += 1024) {
    const float m = a.ma[o + c] + a.mr[o + c], v = a.Sa[o + c] + a.Sr[o + c];
    acc += m * m + v;
  }
  const float inv = 1.f / sqrtf(row_sum<1024>(acc, red) / (float)a.D + a.eps);
  if (threadIdx.x == 0) a.inv[row] = inv;
  for (int c = threadIdx.x; c < a.D; c += 1024) write_value(a, o + c, c, inv);
}

// Rows shorter than four, a thread for each.
__global__ void __launch_bounds__(256) add_rms_norm_short_kernel(FwdArgs a) {
  const int64_t row = row_block() * 256 + threadIdx.x, o = row * a.D;
  if (row >= a.rows) return;
  float acc = 0.f;
  for (int c = 0; c < a.D; ++c) {
    const float m = a.ma[o + c] + a.mr[o + c], v = a.Sa[o + c] + a.Sr[o + c];
    acc += m * m + v;
  }
  const float inv = 1.f / sqrtf(acc / (float)a.D + a.eps);
  a.inv[row] = inv;
  for (int c = 0; c < a.D; ++c) write_value(a, o + c, c, inv);
}

// Blocks own a range of rows and 4 CT columns (CT threads across, 256 / CT rows at a time);
// a thread keeps the weights and sums of its four columns in registers over the range, every
// kFloatRows rows' floats added in float64 (wide rows leave few blocks, and the ranges grow
// with the batch: 512 rows at 65536 x 8192), the threads of a column are joined in float64
// through LDS, and one partial sum per block, column and moment goes to ws[moment][block][D].
// HBM bound: 16384 x 4096 with deltas at the sum moves 1.88 GB in 343 us (5.5 TB/s); all floats
// over the range took the same.
constexpr int kFloatRows = 32;
template <bool NT, bool WIDE>
__global__ void __launch_bounds__(256) add_rms_norm_bwd_kernel(
    const float* __restrict__ dmz, const float* __restrict__ dSz, const float* __restrict__ dms,
    const float* __restrict__ dSs, const float* __restrict__ ms, const float* __restrict__ inv_rms,
    const float* __restrict__ mw, float* __restrict__ dma, float* __restrict__ dSa, float* __restrict__ ws,
    int64_t rows, int D, int CT) {
  __shared__ f4 red[2][256];
  const int RG = 256 / CT, ct = (int)threadIdx.x % CT, rg = (int)threadIdx.x / CT, nblk = (int)gridDim.x;
  const int64_t r0 = rows * blockIdx.x / nblk, r1 = rows * (blockIdx.x + 1) / nblk;
  double tm[4] = {}, ts[4] = {};
  const auto fold = [&](const f4& m, const f4& s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) tm[e] += m[e], ts[e] += s[e];
  };
  int skip = 4;
  if constexpr (WIDE) {
    const Cols c = columns((int)blockIdx.y * CT + ct, D);
    skip = rg < RG ? c.skip : 4;
    if (skip < 4) {
      const f4 g = *reinterpret_cast<const f4*>(mw + c.at);
      for (int64_t p = r0 + rg; p < r1; p += (int64_t)kFloatRows * RG) {
        const int64_t end = min(r1, p + (int64_t)kFloatRows * RG);
        f4 am = {0.f, 0.f, 0.f, 0.f}, as = am;
#pragma unroll 2
        for (int64_t r = p; r < end; r += RG) {
          const int64_t o = r * D + c.at;
          const float inv = inv_rms[r];
          const f4 a = ld<NT>(dmz + o), b = ld<NT>(dSz + o), x = ld<NT>(ms + o) * inv, k = g * inv;
          f4 u = a * k, w = b * (k * k);
          if (dms) u += ld<NT>(dms + o), w += ld<NT>(dSs + o);
          st<NT>(dma + o, u);  // columns of two threads get the same values from both
          st<NT>(dSa + o, w);
          am += a * x;
          as += b * (x * x);
        }
        fold(am, as);
      }
    }
  } else if (rg < RG) {  // rows of one to three values, one thread across
    skip = 0;
    for (int64_t p = r0 + rg; p < r1; p += (int64_t)kFloatRows * RG) {
      const int64_t end = min(r1, p + (int64_t)kFloatRows * RG);
      f4 am = {0.f, 0.f, 0.f, 0.f}, as = am;
      for (int64_t r = p; r < end; r += RG)
        for (int e = 0; e < D; ++e) {
          const int64_t o = r * D + e;
          const float inv = inv_rms[r], x = inv * ms[o], k = inv * mw[e], a = dmz[o], b = dSz[o];
          dma[o] = a * k + (dms ? dms[o] : 0.f);
          dSa[o] = b * (k * k) + (dSs ? dSs[o] : 0.f);
          am[e] += a * x;
          as[e] += b * (x * x);
        }
      fold(am, as);
    }
  }
  f4 am = {(float)tm[0], (float)tm[1], (float)tm[2], (float)tm[3]};
  f4 as = {(float)ts[0], (float)ts[1], (float)ts[2], (float)ts[3]};
  // the thread's own columns first
  if (skip == 1) am = f4{am.y, am.z, am.w, 0.f}, as = f4{as.y, as.z, as.w, 0.f};
  if (skip == 2) am = f4{am.z, am.w, 0.f, 0.f}, as = f4{as.z, as.w, 0.f, 0.f};
  if (skip == 3) am = f4{am.w, 0.f, 0.f, 0.f}, as = f4{as.w, 0.f, 0.f, 0.f};
  red[0][threadIdx.x] = am, red[1][threadIdx.x] = as;
  __syncthreads();
  // value e of column chunk q, moment w: the RG threads' sums in order
  const float* f = reinterpret_cast<const float*>(&red[0][0]);
  for (int i = threadIdx.x; i < 8 * CT; i += 256) {
    const int w = i / (4 * CT), e = i % (4 * CT), col = 4 * (int)blockIdx.y * CT + e;
    if (col >= D) continue;
    double s = 0.0;
    for (int r = 0; r < RG; ++r) s += f[w * 1024 + r * 4 * CT + e];
    ws[((int64_t)w * nblk + blockIdx.x) * D + col] = (float)s;
  }
}

// 32 columns and 8 stretches of the blocks' partial sums at a time, in float64.
__global__ void __launch_bounds__(256) add_rms_norm_finalize_kernel(const float* __restrict__ ws,
                                                                    const float* __restrict__ Sw,
                                                                    float* __restrict__ dmw, float* __restrict__ dSw,
                                                                    int D, int nblk) {
  __shared__ double red[8][32];
  const int cl = threadIdx.x & 31, part = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + cl, w = blockIdx.y;
  const int b0 = nblk * part / 8, b1 = nblk * (part + 1) / 8;
  const float* p = ws + (int64_t)w * nblk * D + c;
  double s = 0.0;
  if (c < D) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) s += p[(int64_t)b * D];
  }
  red[part][cl] = s;
  __syncthreads();
  if (part || c >= D) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) s += red[q][cl];
  const float sg = Sw[c];
  if (w)
    dSw[c] = sg * sg * (float)s;
  else
    dmw[c] = sg * (float)s;
}

// Threads across a block's columns, and row ranges: up to 1024 blocks (16384 x 4096: 512 blocks
// 333 us, 1024 342, 2048 375; 65536 x 256: 94, 90, 96), 4 rows a thread at least.
struct BwdPlan {
  int ct, chunks, nblk;
};
BwdPlan bwd_plan(int64_t rows, int64_t D) {
  BwdPlan p;
  const int64_t q = cdiv(D, 4);
  p.ct = (int)(q < 256 ? q : 256);
  p.chunks = (int)cdiv(q, p.ct);
  const int64_t rg = 256 / p.ct;
  int64_t n = cdiv(rows, rg * 4);
  const int64_t most = p.chunks < 1024 ? 1024 / p.chunks : 1;
  p.nblk = (int)(n > most ? most : n);
  return p;
}

// Above this much traffic nothing a kernel reads or writes is still in the 256 MB last-level
// cache when it is needed next, and the nontemporal policy reaches further
// (16384 x 4096: forward 400 -> 380 us, backward 364 -> 342; 16384 x 1024: 120 -> 109, 105 -> 95).
constexpr double kCacheBytes = 256e6;

template <int TPR, int NV>
void launch_fwd(const FwdArgs& a, bool nt, hipStream_t s) {
  const dim3 grid = row_grid(cdiv(a.rows, TPR < 256 ? 256 / TPR : 1)), block(TPR < 256 ? 256 : TPR);
  // these take few rows only (below 4096 of 1024 values, 512 of 8192), which stay in the cache
  constexpr bool kFew = (TPR == 256 && NV == 1) || (TPR == 1024 && NV <= 2);
  auto kernel = add_rms_norm_kernel<TPR, NV, false>;
  if constexpr (!kFew)
    if (nt) kernel = add_rms_norm_kernel<TPR, NV, true>;
  hipLaunchKernelGGL(kernel, grid, block, 0, s, a.ma, a.Sa, a.mr, a.Sr, a.mw, a.Sw, a.mz, a.Sz, a.ms, a.Ss, a.inv,
                     a.rows, a.D, a.eps);
}
// Chunks of four per thread: rounded up to a kernel that holds them, TPR * 32 values at most
// (a wave's rows are at most 1024 long).
template <int TPR>
void launch_fwd_nv(const FwdArgs& a, bool nt, hipStream_t s) {
  const int64_t nv = cdiv(cdiv(a.D, 4), TPR);
  if (nv <= 1)
    launch_fwd<TPR, 1>(a, nt, s);
  else if (nv <= 2)
    launch_fwd<TPR, 2>(a, nt, s);
  else if (TPR == 64 || nv <= 4)
    launch_fwd<TPR, 4>(a, nt, s);
  else if constexpr (TPR > 64)
    launch_fwd<TPR, 8>(a, nt, s);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int tagi_add_rmsnorm_fwd(const float* ma, const float* Sa, const float* mr, const float* Sr,
                                    const float* mw, const float* Sw, float* mz, float* Sz, float* ms, float* Ss,
                                    float* inv_rms, int64_t rows, int64_t D, float eps, tagi_stream_t stream) {
  const char* what = "tagi_add_rmsnorm_fwd";
  TAGI_REQUIRE(rows >= 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(rows < (1ll << 31) && D < (1ll << 24), "%s: too large", what);
  if (rows == 0) return TAGI_OK;
  TAGI_REQUIRE(ma && Sa && mr && Sr && mw && Sw && mz && Sz && ms && inv_rms, "%s: null pointer", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_RMSNORM, s, 0.0, (Ss ? 32.0 : 28.0) * rows * D + 4.0 * rows);
  const FwdArgs a{ma, Sa, mr, Sr, mw, Sw, mz, Sz, ms, Ss, inv_rms, rows, (int)D, eps};
  const bool nt = 32.0 * rows * D > kCacheBytes;
  // threads of a row: a wave for short rows, or for longer ones when there are rows enough to
  // fill the GPU; more where few rows would wait on each thread's loads
  const int64_t chunks = cdiv(D, 4);
  if (D < 4)
    hipLaunchKernelGGL(add_rms_norm_short_kernel, row_grid(cdiv(rows, 256)), dim3(256), 0, s, a);
  else if (chunks > 8 * 1024)
    hipLaunchKernelGGL(add_rms_norm_long_kernel, row_grid(rows), dim3(1024), 0, s, a);
  else if (chunks <= 64 || (chunks <= 4 * 64 && rows >= 4096))
    launch_fwd_nv<64>(a, nt, s);
  else if (chunks <= 256 || (chunks <= 8 * 256 && rows >= 512))
    launch_fwd_nv<256>(a, nt, s);
  else
    launch_fwd_nv<1024>(a, nt, s);
  return check_launch(what);
}

extern "C" int64_t tagi_add_rmsnorm_bwd_ws_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0) return 0;
  return (int64_t)bwd_plan(rows, D).nblk * 2 * D * (int64_t)sizeof(float);
}

extern "C" int tagi_add_rmsnorm_bwd(const float* dmz, const float* dSz, const float* dms, const float* dSs,
                                    const float* ms, const float* inv_rms, const float* mw, const float* Sw,
                                    float* dma, float* dSa, float* dmw, float* dSw, int64_t rows, int64_t D, void* ws,
                                    int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_add_rmsnorm_bwd";
  TAGI_REQUIRE(rows >= 0 && D > 0, "%s: bad sizes", what);
  TAGI_REQUIRE(rows < (1ll << 31) && D < (1ll << 24), "%s: too large", what);
  TAGI_REQUIRE(mw && Sw && dmw && dSw, "%s: null pointer", what);
  TAGI_REQUIRE((dms == nullptr) == (dSs == nullptr), "%s: dms and dSs must be given together", what);
  TAGI_REQUIRE(rows == 0 || (dmz && dSz && ms && inv_rms && dma && dSa && ws), "%s: null pointer", what);
  TAGI_REQUIRE(ws_bytes >= tagi_add_rmsnorm_bwd_ws_bytes(rows, D), "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_RMSNORM, s, 0.0, (dms ? 28.0 : 20.0) * rows * D);
  const BwdPlan p = bwd_plan(rows, D);
  if (rows > 0) {
    const dim3 grid((unsigned)p.nblk, (unsigned)p.chunks);
    float* part = static_cast<float*>(ws);
    const bool nt = (dms ? 28.0 : 20.0) * rows * D > kCacheBytes;
    const auto kernel = D < 4 ? add_rms_norm_bwd_kernel<false, false>
                              : (nt ? add_rms_norm_bwd_kernel<true, true> : add_rms_norm_bwd_kernel<false, true>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, dmz, dSz, dms, dSs, ms, inv_rms, mw, dma, dSa, part, rows, (int)D,
                       p.ct);
  }
  hipLaunchKernelGGL(add_rms_norm_finalize_kernel, dim3((unsigned)cdiv(D, 32), 2), dim3(256), 0, s,
                     static_cast<const float*>(ws), Sw, dmw, dSw, (int)D, p.nblk);
  return check_launch(what);
}
