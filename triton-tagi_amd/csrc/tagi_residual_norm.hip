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

constexpr int kThreads = 256;

// One block per row.
__global__ void __launch_bounds__(kThreads) add_rms_norm_kernel(
    const float* __restrict__ ma, const float* __restrict__ Sa, const float* __restrict__ mr,
    const float* __restrict__ Sr, const float* __restrict__ mw, const float* __restrict__ Sw, float* __restrict__ mz,
    float* __restrict__ Sz, float* __restrict__ ms, float* __restrict__ Ss, float* __restrict__ inv_rms, int64_t rows,
    int D, float eps) {
  __shared__ float red[kThreads / 64];
  const int64_t row = blockIdx.x, o = row * D;
  float acc = 0.f;
  for (int c = threadIdx.x; c < D; c += kThreads) {
    const float m = ma[o + c] + mr[o + c], v = Sa[o + c] + Sr[o + c];
    ms[o + c] = m;
    if (Ss) Ss[o + c] = v;
    acc += m * m + v;
  }
  for (int w = 32; w > 0; w >>= 1) acc += __shfl_xor(acc, w);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  const float inv = 1.f / sqrtf((red[0] + red[1] + red[2] + red[3]) / (float)D + eps);
  if (threadIdx.x == 0) inv_rms[row] = inv;
  for (int c = threadIdx.x; c < D; c += kThreads) {
    const float m = ma[o + c] + mr[o + c], v = Sa[o + c] + Sr[o + c], g = mw[c], sg = Sw[c];
    mz[o + c] = m * inv * g;
    Sz[o + c] = inv * inv * (v * (g * g + sg) + sg * (m * m));
  }
}

// Blocks own a range of rows and 256 columns; partial column sums go to ws[moment][block][D].
__global__ void __launch_bounds__(kThreads) add_rms_norm_bwd_kernel(
    const float* __restrict__ dmz, const float* __restrict__ dSz, const float* __restrict__ dms,
    const float* __restrict__ dSs, const float* __restrict__ ms, const float* __restrict__ inv_rms,
    const float* __restrict__ mw, float* __restrict__ dma, float* __restrict__ dSa, float* __restrict__ ws,
    int64_t rows, int D) {
  const int c = (int)blockIdx.y * kThreads + (int)threadIdx.x;
  if (c >= D) return;
  const int nblk = (int)gridDim.x;
  const int64_t r0 = rows * blockIdx.x / nblk, r1 = rows * (blockIdx.x + 1) / nblk;
  const float g = mw[c];
  float am = 0.f, as = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const int64_t o = r * D + c;
    const float inv = inv_rms[r], k = inv * g, x = inv * ms[o], a = dmz[o], b = dSz[o];
    dma[o] = a * k + (dms ? dms[o] : 0.f);
    dSa[o] = b * (k * k) + (dSs ? dSs[o] : 0.f);
    am += a * x;
    as += b * (x * x);
  }
  ws[(int64_t)blockIdx.x * D + c] = am;
  ws[((int64_t)nblk + blockIdx.x) * D + c] = as;
}

__global__ void __launch_bounds__(kThreads) add_rms_norm_finalize_kernel(const float* __restrict__ ws,
                                                                         const float* __restrict__ Sw,
                                                                         float* __restrict__ dmw,
                                                                         float* __restrict__ dSw, int D, int nblk) {
  const int c = (int)blockIdx.x * kThreads + (int)threadIdx.x;
  if (c >= D) return;
  double m = 0.0, s = 0.0;
  for (int b = 0; b < nblk; ++b) {
    m += ws[(int64_t)b * D + c];
    s += ws[((int64_t)nblk + b) * D + c];
  }
  const float sg = Sw[c];
  dmw[c] = sg * (float)m;
  dSw[c] = sg * sg * (float)s;
}

int bwd_blocks(int64_t rows) {
  const int64_t b = cdiv(rows, 32);
  return (int)(b > 512 ? 512 : b);
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
  hipLaunchKernelGGL(add_rms_norm_kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, ma, Sa, mr, Sr, mw, Sw, mz, Sz,
                     ms, Ss, inv_rms, rows, (int)D, eps);
  return check_launch(what);
}

extern "C" int64_t tagi_add_rmsnorm_bwd_ws_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0) return 0;
  return (int64_t)bwd_blocks(rows) * 2 * D * (int64_t)sizeof(float);
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
  const int nblk = bwd_blocks(rows);
  if (rows > 0)
    hipLaunchKernelGGL(add_rms_norm_bwd_kernel, dim3((unsigned)nblk, (unsigned)cdiv(D, kThreads)), dim3(kThreads), 0,
                       s, dmz, dSz, dms, dSs, ms, inv_rms, mw, dma, dSa, static_cast<float*>(ws), rows, (int)D);
  hipLaunchKernelGGL(add_rms_norm_finalize_kernel, dim3((unsigned)cdiv(D, kThreads)), dim3(kThreads), 0, s,
                     static_cast<const float*>(ws), Sw, dmw, dSw, (int)D, nblk);
  return check_launch(what);
}
