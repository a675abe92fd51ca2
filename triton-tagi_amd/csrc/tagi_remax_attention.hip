// Attention with Remax scores over sequences of any length, forward and backward, without
// storing a score.
//
// With c the scale, for query i and the keys j it sees (remax.py:33-114 over them):
//   m_ij = c q_i.k_j,  v_ij = c^2 [Sq_i.(k_j^2 + Sk_j) + q_i^2.Sk_j]
//   (mm, vm, Phi)_ij: moments of max(z_ij, 0);  mt_i = sum mm, vt_i = sum vm
//   w_ij, k_ij: weight and its relative variance from (mm, vm)_ij and (mt, vt)_i;  s_i = sum w
//   a = w / s,  mo_i = sum a v_j,  So_i = sum a^2 [k (v_j^2 + Sv_j) + Sv_j]
// The weights need the row's sums first, so a row's keys are walked twice: once for mt and vt,
// once for the outputs, which are linear in w and w^2 and are divided by s at the end.
// Backward, each product's other operand at its mean, with J_ij the Remax Jacobian:
//   e_ij = c J (dm_i.v_j),  E_ij = c^2 J^2 (dS_i.v_j^2)
//   dq = e k, dSq = E k^2;  dk = e^T q, dSk = E^T q^2;  dv = a^T dm, dSv = (a^2)^T dS
// Queries and keys are formed again from (mt, vt, s): one kernel walks keys for each query (dq),
// one walks queries for each key (dk, dv); no atomics, every sum's order is fixed by the sizes.
//
// The queries of the H / G heads that share a key head are one list of rows, token by token. A wave
// holds 16 rows (or keys) as right operands in registers; a block's waves walk tiles of 32 keys (or
// rows) together, split into bf16 parts (tagi_split_bf16.h) as they go from HBM to LDS. The walked
// side is in the rows of every product, so a lane holds the scores of one row (or key) and its sums
// need no exchange until the end; and the registers of two products of 16 are the next product's
// right operand as they are, whose left operand is the tile read transposed from LDS.
//
// What bounds it: instruction issue. The outputs' kernel takes 144 matrix instructions for a wave's
// tile of 16 rows and 32 keys of 64 features (half for the scores' moments, half for the outputs) and 800
// vector instructions, 66 a score for its rectified moments and weight. A matrix instruction of this
// shape holds back a SIMD's vector instructions for most of its 16 cycles (16 of them and 64
// multiply-adds: 221 ns in turn, 117 and 144 alone; two waves, one each: 215), so the two add up: 3200 +
// 510 (reciprocals, roots, exponentials) + 2300 cycles, 6240 measured. Neither more waves, nor the two
// kinds interleaved instruction by instruction, nor priorities between the waves changed that. (The
// shape of 32 rows and columns would run beside vector work, 155 ns, but its right operands and sums of
// 64 features take more than the 256 registers of two waves a SIMD.) Measured: 2 x 4096 tokens, 16
// heads of 64 over 4, causal: statistics 0.74 ms, outputs 1.62, dq 1.65, dk and dv 2.5, joins 0.17: 99
// TFLOP/s of fp32 products; on the fp32 matrix cores, whose peak is 154, the same kernels took twice
// as long.
#include "tagi_remax.h"
#include "tagi_split_bf16.h"

namespace tagi {
namespace {

typedef short h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kTile = 32;           // keys (or rows) walked at a time
constexpr int kMaxDim = 128;
constexpr int kLdsBytes = 160 * 1024;
// Walked by one block at most: the matrix cores cut sums off (they do not round them), and what is
// lost of a sum of positive terms grows with their number (late rows' variances: 1.6e-6 after 2048
// keys, 1e-6 after 1024; the join takes 23 us more of 6.2 ms at 4096 tokens). The gradients' terms have
// both signs: 1e-6 after 2048. What blocks walked is added in fp32.
constexpr int kMostWalked = 1024, kMostWalkedBack = 2048;

struct Args {
  const float *mq, *Sq, *mk, *Sk, *mv, *Sv, *dm, *dS;
  tagi_heads lq, lk, lv, ld, loq, lokv;
  const void *lengths, *starts;
  int len_bytes, start_bytes, causal;
  float *mo, *So, *rows, *dmk, *dSk, *dmv, *dSv;  // mo, So: dmq, dSq in the backward
  float *sums, *parts;  // workspace: [split][2][BG][M], [split][BG][M][2 D + 1] (or [..][N][4 D])
  int64_t B, M;         // M = T R rows of a key head
  int T, N, H, G, R, D;
  // The walked side: launch l's split i has the chunk l splits + i; the statistics' split i, all of one
  // launch, that of stat_chunk. parted: outputs are joined from parts.
  int splits, chunk, launch, parted, stat_chunk;
  float c, c2;
};

__device__ __forceinline__ int64_t int_at(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// A sequence: its keys, and where its first query stands.
struct Seq {
  int64_t start;
  int len;
};
__device__ __forceinline__ Seq sequence(const Args& A, int64_t b) {
  Seq s{0, A.N};
  if (A.lengths) {
    const int64_t n = int_at(A.lengths, A.len_bytes, b);
    s.len = (int)(n < 0 ? 0 : (n < A.N ? n : A.N));
  }
  if (A.starts) {  // positions beyond 2^32 either way see nothing, or everything, alike
    const int64_t p = int_at(A.starts, A.start_bytes, b), far = 1ll << 32;
    s.start = p < -far ? -far : (p > far ? far : p);
  }
  return s;
}
// Keys that row rho of its key head sees: those below this.
__device__ __forceinline__ int row_limit(const Args& A, const Seq& s, int64_t rho) {
  if (rho >= A.M) return 0;
  const int64_t pos = s.start + (int)rho / A.R;
  if (pos < 0 || pos >= s.len) return 0;
  return A.causal ? (int)pos + 1 : s.len;
}
// No row of [rho0, rho0 + n) sees a key from here on.
__device__ __forceinline__ int block_limit(const Args& A, const Seq& s, int64_t rho0, int n) {
  if (rho0 >= A.M) return 0;
  const int64_t last = (rho0 + n < A.M ? rho0 + n : A.M) - 1;
  const int64_t first_pos = s.start + (int)rho0 / A.R, pos = s.start + (int)last / A.R;
  if (first_pos >= s.len || pos < 0) return 0;
  return A.causal ? (int)(pos + 1 < s.len ? pos + 1 : s.len) : s.len;
}

__device__ __forceinline__ int64_t row_at(const Args& A, const tagi_heads& l, int64_t b, int g, int64_t rho) {
  const int t = (int)rho / A.R;
  return b * l.sb + (int64_t)t * l.st + (g * A.R + ((int)rho - t * A.R)) * l.sh;
}
__device__ __forceinline__ int64_t key_at(const tagi_heads& l, int64_t b, int g, int64_t key) {
  return b * l.sb + key * l.st + g * l.sh;
}
__device__ __forceinline__ int64_t stat_at(const Args& A, int64_t b, int g, int64_t rho, int q) {
  const int t = (int)rho / A.R, h = g * A.R + ((int)rho - t * A.R);
  return ((q * A.B + b) * A.H + h) * A.T + t;
}

// Eight neighbouring features from d on, zeros behind D. VEC: D is a multiple of eight.
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int d, int D, bool on, float (&x)[8]) {
  if constexpr (VEC) {
    f4 a = {0, 0, 0, 0}, b = a;
    if (on && d < D) a = *reinterpret_cast<const f4*>(p + d), b = *reinterpret_cast<const f4*>(p + d + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = on && d + i < D ? p[d + i] : 0.f;
  }
}

// The block's wave, in a scalar register.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// x is formed here, and not where it is used: what it is formed from would wait in registers.
__device__ __forceinline__ void formed(float& x) { asm volatile("" : "+v"(x)); }
// x, of which the compiler knows nothing: what a tile's addresses need of it is formed in every
// tile and not kept in registers across them.
__device__ __forceinline__ int hidden(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// ------------------------------------------------------------------------ walked tiles in LDS
// A tile is kTile rows of operands in bf16 parts, [part][16 rows][32 features] in the order in
// which a wave's lanes read a left operand: lane l the row l % 16, features 8 (l / 16) + 0..7.
template <int DP, int PARTS>
struct Tile {
  static constexpr int S = DP / 32;
  static constexpr int halves = PARTS * 2 * S * 512;  // 16-bit values
  static constexpr int bytes = 2 * halves;
};
template <int DP>
__device__ __forceinline__ int piece(int part, int kt, int s) {
  return ((part * 2 + kt) * (DP / 32) + s) * 512;
}
// An operand's place: in the instruction where a tile is within its reach of 64 KB; where it is not
// (heads of 128), formed where it is used, since the sums would wait in registers.
template <int DP>
__device__ __forceinline__ int offset(int x) {
  return DP == 128 ? hidden(x) : x;
}
template <int DP, int P>
__device__ __forceinline__ void put(short* tile, int first, int kt, int s, int lane, const Parts<P>& x) {
#pragma unroll
  for (int p = 0; p < P; ++p) *reinterpret_cast<bf8*>(tile + piece<DP>(first + p, kt, s) + 8 * lane) = x.p[p];
}
// c += a b, a 16 rows of the tile: part by part, so that four registers hold the left operand.
template <int DP>
__device__ __forceinline__ acc4 mma_left(const short* left, int first, int kt, int s, const Parts<3>& b, acc4 c) {
  const short* at = left + offset<DP>(piece<DP>(first, 0, 0));
#pragma unroll
  for (int i = 2; i >= 0; --i) {
    const bf8 a = *reinterpret_cast<const bf8*>(at + piece<DP>(i, kt, s));
#pragma unroll
    for (int j = 2 - i; j >= 0; --j) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b.p[j], c, 0, 0, 0);
  }
  return c;
}
// The tile transposed, 16 features (16 dt + lane % 16) as rows of a left operand: lane group g
// holds the tile's rows 4 g + 0..3 and 16 + 4 g + 0..3, as the registers of two products of 16
// rows hold them. ds_read_b64_tr_b16: of the 64 bits that lane p of a group of 16 reads, lane q
// gets element q % 4 of lanes q / 4 + 4 j, j = 0..3.
__device__ __forceinline__ int turned_at(int lane) {
  const int p = lane & 15, g = lane >> 4;
  return (((p & 3) >> 1) * 16 + 4 * g + (p >> 2)) * 8 + 4 * (p & 1);
}
template <int DP>
__device__ __forceinline__ acc4 mma_transposed(const short* turned, int first, int dt, const Parts<3>& b, acc4 c) {
  typedef __attribute__((address_space(3))) h4 lds_h4;
  const short* at = turned + offset<DP>(piece<DP>(first, 0, 0));
#pragma unroll
  for (int i = 2; i >= 0; --i) {
    union {
      bf8 v;
      h4 h[2];
    } u;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
      u.h[kt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_h4*)(at + piece<DP>(i, kt, dt >> 1) + (dt & 1) * 256));
#pragma unroll
    for (int j = 2 - i; j >= 0; --j) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u.v, b.p[j], c, 0, 0, 0);
  }
  return c;
}

// What a lane brings of the next tile: eight features of a row's mean and variance (or deltas).
struct Unit {
  float m[8], S[8];
};
// A tile takes 2 S units a lane and operand pair; wave w of W holds units w, w + W, ...
template <int DP, int W>
constexpr int units_of(int pairs) {
  return (2 * (DP / 32) * pairs + W - 1) / W;
}

// The right operand of a wave's 16 rows: x in parts, eight features a lane and step.
template <int DP>
struct Right {
  Parts<3> p[DP / 32];
};

// The wave's right operands of its rows of an (m, S) pair, formed by f.
template <int DP, bool VEC, typename F>
__device__ __forceinline__ void load_right(const float* pm, const float* pS, int64_t at, int D, bool on, int k8, F&& f) {
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    float m[8], S[8];
    load8<VEC>(pm + at, 32 * s + 8 * k8, D, on, m);
    load8<VEC>(pS + at, 32 * s + 8 * k8, D, on, S);
    f(s, m, S);
  }
}

// The same in two halves: the products of the first parts, and the others. The matrix cores cut
// sums off: a score's mean, on which its tail's weight depends as exp(-m^2 / 2 v), takes the others
// while the sum is small, and then is cut once a step instead of six times (rows of few keys: 1.6e-6
// of the variances wrong before, 6e-7 so).
template <int DP>
__device__ __forceinline__ acc4 mma_first(const short* left, int first, int kt, int s, const Parts<3>& b, acc4 c) {
  const bf8 a = *reinterpret_cast<const bf8*>(left + offset<DP>(piece<DP>(first, kt, s)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b.p[0], c, 0, 0, 0);
}
template <int DP, bool FIRST>
__device__ __forceinline__ void mma_left(const short* left, int first, int kt, int s, const Parts<3>& b, acc4& c,
                                         acc4& rest) {
  const short* at = left + offset<DP>(piece<DP>(first, 0, 0));
#pragma unroll
  for (int i = 2; i >= 0; --i) {
    const bf8 a = *reinterpret_cast<const bf8*>(at + piece<DP>(i, kt, s));
#pragma unroll
    for (int j = 2 - i; j >= 0; --j) {
      if (i + j > 0)
        rest = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b.p[j], rest, 0, 0, 0);
      else if (FIRST)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b.p[j], c, 0, 0, 0);
    }
  }
}

// Nothing is scheduled across: operands of later products loaded early would take the registers
// of those in use.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// Before a loop of a thousand instructions: from the middle of an instruction cache line they take 2%
// longer (outputs of 64 features 1.46 -> 1.43 ms, dq 1.53 -> 1.49 at 2 x 4096 tokens).
__device__ __forceinline__ void at_line() { asm volatile(".p2align 6"); }

// Moments of the scores of 16 walked rows: m = a0 b0, v = a1 b1 + a2 b2 with a0, a1, a2 the parts
// 0, 3, 6 of the tile.
template <int DP>
__device__ __forceinline__ void scores(const short* left, int kt, const Right<DP>& b0, const Right<DP>& b1,
                                       const Right<DP>& b2, acc4& m, acc4& v) {
  acc4 dm = {0, 0, 0, 0}, dv = dm;
  if constexpr (DP < 128) {
    m = v = dm;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      mma_left<DP, true>(left, 0, kt, s, b0.p[s], m, dm);
      mma_left<DP, true>(left, 3, kt, s, b1.p[s], v, dv);
      mma_left<DP, true>(left, 6, kt, s, b2.p[s], v, dv);
    }
    m += dm, v += dv;
  } else {  // the registers of two more sums are not there: the keys' first parts are read again
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      mma_left<DP, false>(left, 0, kt, s, b0.p[s], m, dm);
      mma_left<DP, false>(left, 3, kt, s, b1.p[s], v, dv);
      mma_left<DP, false>(left, 6, kt, s, b2.p[s], v, dv);
    }
    m = dm, v = dv;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      m = mma_first<DP>(left, 0, kt, s, b0.p[s], m);
      v = mma_first<DP>(left, 3, kt, s, b1.p[s], v);
      v = mma_first<DP>(left, 6, kt, s, b2.p[s], v);
    }
  }
}

// The sum over the four lane groups that share a column.
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The least of a wave's lanes, in a scalar register.
__device__ __forceinline__ int least(int x) {
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) {
    const int y = __shfl_xor(x, w);
    x = x < y ? x : y;
  }
  return __builtin_amdgcn_readfirstlane(x);
}

// Blocks in one dimension: (split, key head, rows), the rows of one key head on one XCD where the
// key heads divide evenly, so that their keys stay in its L2.
struct Place {
  int64_t b, bg, block;
  int g, split;
};
__device__ __forceinline__ Place place(const Args& A, int64_t blocks) {
  const int64_t BG = A.B * A.G;
  int64_t i = blockIdx.x;
  Place p;
  if (BG % 8 == 0) {
    const int64_t x = i & 7, k = i >> 3, per = blocks * A.splits;
    p.bg = x + 8 * (k / per);
    i = k % per;
  } else {
    p.bg = i / (blocks * A.splits);
    i -= p.bg * blocks * A.splits;
  }
  p.split = (int)(i / blocks);
  p.block = i - p.split * blocks;
  p.b = p.bg / A.G;
  p.g = (int)(p.bg - p.b * A.G);
  return p;
}

// ---------------------------------------------------------------------------------- forward
// Unit i of the tile of keys (and values) from key0 on, and the unit's place in the tile. Parts:
// keys k 0, k^2 3, Sk 6; values v 9, v^2 12 (, Sv 15).
template <int DP, bool VEC>
__device__ __forceinline__ void fetch_key(const Args& A, const Place& p, int key0, int to, int i, int lane,
                                          bool value_variances, Unit& u) {
  constexpr int S = DP / 32;
  const bool value = i >= 2 * S;
  const int k = value ? i - 2 * S : i, kt = k / S, s = k % S, key = key0 + 16 * kt + (lane & 15);
  const bool on = key < to;
  const int64_t at = on ? key_at(value ? A.lv : A.lk, p.b, p.g, key) : 0;
  const int d = 32 * s + 8 * (lane >> 4);
  load8<VEC>((value ? A.mv : A.mk) + at, d, A.D, on, u.m);
  if (!value || value_variances) load8<VEC>((value ? A.Sv : A.Sk) + at, d, A.D, on, u.S);
}
template <int DP>
__device__ __forceinline__ void put_key(short* tile, int i, int lane, bool value_variances, const Unit& u) {
  constexpr int S = DP / 32;
  const bool value = i >= 2 * S;
  const int k = value ? i - 2 * S : i, kt = k / S, s = k % S, first = value ? 9 : 0;
  float x[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) x[q] = u.m[q] * u.m[q];
  put<DP>(tile, first, kt, s, lane, split<3>(u.m));
  put<DP>(tile, first + 3, kt, s, lane, split<3>(x));
  if (!value || value_variances) put<DP>(tile, first + 6, kt, s, lane, split<3>(u.S));
}
template <int DP, bool VEC, int W, int U>
__device__ __forceinline__ void fetch_keys(const Args& A, const Place& p, int key0, int to, int pairs, int wave, int lane,
                                           bool value_variances, Unit (&u)[U]) {
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (wave + j * W < 2 * (DP / 32) * pairs)
      fetch_key<DP, VEC>(A, p, key0, to, wave + j * W, lane, value_variances, u[j]);
}
template <int DP, int W, int U>
__device__ __forceinline__ void put_keys(short* tile, int pairs, int wave, int lane, bool value_variances,
                                         const Unit (&u)[U]) {
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (U > 1) fence();
    if (wave + j * W < 2 * (DP / 32) * pairs) put_key<DP>(tile, wave + j * W, lane, value_variances, u[j]);
  }
}
// Unit by unit, where registers do not hold more.
template <int DP, bool VEC, int W>
__device__ __forceinline__ void pass_keys(const Args& A, const Place& p, int key0, int to, short* tile, int pairs, int wave,
                                          int lane, bool value_variances) {
  Unit u;
#pragma unroll 1
  for (int i = wave; i < 2 * (DP / 32) * pairs; i += W) {
    fetch_key<DP, VEC>(A, p, key0, to, i, hidden(lane), value_variances, u);
    put_key<DP>(tile, i, hidden(lane), value_variances, u);
  }
}

// The next tile of keys and values behind the products: a wave's loads are in flight together, across
// the barrier (BARRIER) behind which the tile's place is free. Of 128 features one after the other: two
// at once take 130 registers of the outputs' products to scratch memory (1.69 -> 2.75 ms).
template <int DP, bool VEC, int W, bool BARRIER>
__device__ __forceinline__ void next_keys(const Args& A, const Place& p, int key0, int to, short* tile, int wave, int lane,
                                          bool value_variances) {
  fence();
  if constexpr (DP < 128) {
    Unit u[units_of<DP, W>(2)];
    fetch_keys<DP, VEC, W>(A, p, key0, to, 2, wave, hidden(lane), value_variances, u);
    if (BARRIER) __syncthreads();
    fence();
    put_keys<DP, W>(tile, 2, wave, hidden(lane), value_variances, u);
  } else {
    Unit u;
    fetch_key<DP, VEC>(A, p, key0, to, wave, hidden(lane), value_variances, u);
    if (BARRIER) __syncthreads();
    put_key<DP>(tile, wave, hidden(lane), value_variances, u);
#pragma unroll 1
    for (int i = wave + W; i < 4 * (DP / 32); i += W) {
      fetch_key<DP, VEC>(A, p, key0, to, i, hidden(lane), value_variances, u);
      put_key<DP>(tile, i, hidden(lane), value_variances, u);
    }
  }
}

// Queries on the right: q, Sq, Sq + q^2 (against k, k^2, Sk), scaled.
template <int DP, bool VEC>
__device__ __forceinline__ void load_queries(const Args& A, int64_t at, bool on, int k8, Right<DP>& q, Right<DP>& Q,
                                             Right<DP>& P) {
  load_right<DP, VEC>(A.mq, A.Sq, at, A.D, on, k8, [&](int s, float (&m)[8], float (&S)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] *= A.c, S[i] *= A.c2;
    q.p[s] = split<3>(m), Q.p[s] = split<3>(S);
#pragma unroll
    for (int i = 0; i < 8; ++i) S[i] = fmaf(m[i], m[i], S[i]);
    P.p[s] = split<3>(S);
  });
}

// Sums of the rectified moments. NC x 16 rows a wave: two where the right operands fit (heads of up
// to 64), so that a left operand read from LDS serves both.
template <int DP, bool VEC, int W, int NC>
__global__ void __launch_bounds__(64 * W) stats_kernel(const Args A) {
  constexpr int U = units_of<DP, W>(1), kRows = 16 * W;
  typedef Tile<DP, 9> Keys;
  extern __shared__ __align__(16) short lds[];
  const int64_t blocks = (A.M + NC * kRows - 1) / (NC * kRows);
  Place p = place(A, blocks);
  if (A.causal) p.block = blocks - 1 - p.block;  // the longest rows first
  const Seq s = sequence(A, p.b);
  const int wave = wave_id(), lane = threadIdx.x & 63, k8 = lane >> 4;
  const int64_t block0 = p.block * NC * kRows, wave0 = block0 + wave * NC * 16;
  const int from = p.split * A.stat_chunk;
  auto end = [&](int n) { return n < from + A.stat_chunk ? n : from + A.stat_chunk; };
  const int to = end(block_limit(A, s, block0, NC * kRows)), wave_to = end(block_limit(A, s, wave0, NC * 16));
  if (from >= to) return;
  Right<DP> q[NC], Q[NC], P[NC];
  int lim[NC];
  float mt[NC] = {}, vt[NC] = {};
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t rho = wave0 + 16 * c + (lane & 15);
    lim[c] = row_limit(A, s, rho);
    load_queries<DP, VEC>(A, lim[c] ? row_at(A, A.lq, p.b, p.g, rho) : 0, lim[c] > 0, k8, q[c], Q[c], P[c]);
  }
  int whole = lim[0];  // tiles up to here are seen by all of the wave's rows
#pragma unroll
  for (int c = 1; c < NC; ++c) whole = whole < lim[c] ? whole : lim[c];
  whole = least(whole);
  Unit u[U];
  fetch_keys<DP, VEC, W>(A, p, from, to, 1, wave, lane, false, u);
  put_keys<DP, W>(lds, 1, wave, lane, false, u);
  __syncthreads();
  float mts[NC] = {}, vts[NC] = {};  // sums of every kMostWalked keys: the rounding of many grows with their number
  int buf = 0, stop = from + kMostWalked;
  for (int key0 = from; key0 < to; key0 += kTile, buf ^= 1) {
    if (key0 == stop) {
#pragma unroll
      for (int c = 0; c < NC; ++c) mts[c] += mt[c], vts[c] += vt[c], mt[c] = vt[c] = 0.f;
      stop += kMostWalked;
    }
    const short* left = lds + hidden(buf * Keys::halves + 8 * lane);
    const bool more = key0 + kTile < to;
    if (more) fetch_keys<DP, VEC, W>(A, p, key0 + kTile, to, 1, wave, hidden(lane), false, u);
    if (key0 < wave_to) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        // the sums that scores() makes, in its order to the last bit: where a row has few keys, its weights
        // depend on their differences from the row's sums
        acc4 m[NC], v[NC];
        if constexpr (NC == 1) {
          scores<DP>(left, kt, q[0], Q[0], P[0], m[0], v[0]);
        } else {
          acc4 dm[NC], dv[NC];
#pragma unroll
          for (int c = 0; c < NC; ++c) m[c] = v[c] = dm[c] = dv[c] = acc4{0, 0, 0, 0};
#pragma unroll
          for (int st = 0; st < DP / 32; ++st) {
            const short* at = left + piece<DP>(0, kt, st);
#pragma unroll
            for (int x = 0; x < 3; ++x)  // k q, k^2 Q, Sk P
#pragma unroll
              for (int i = 2; i >= 0; --i) {
                const bf8 k = *reinterpret_cast<const bf8*>(at + piece<DP>(3 * x + i, 0, 0));
#pragma unroll
                for (int j = 2 - i; j >= 0; --j)
#pragma unroll
                  for (int c = 0; c < NC; ++c) {
                    const bf8 b = x == 0 ? q[c].p[st].p[j] : (x == 1 ? Q[c].p[st].p[j] : P[c].p[st].p[j]);
                    acc4& to = x == 0 ? (i + j ? dm[c] : m[c]) : (i + j ? dv[c] : v[c]);
                    to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, b, to, 0, 0, 0);
                  }
              }
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) m[c] += dm[c], v[c] += dv[c];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Rectified z = rectify(m[c][r], v[c][r]);
            m[c][r] = z.mm, v[c][r] = z.vm;
          }
          if (key0 + kTile > whole) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool seen = key0 + 16 * kt + 4 * k8 + r < lim[c];
              m[c][r] = seen ? m[c][r] : 0.f, v[c][r] = seen ? v[c][r] : 0.f;
            }
          }
          mt[c] += (m[c][0] + m[c][1]) + (m[c][2] + m[c][3]);
          vt[c] += (v[c][0] + v[c][1]) + (v[c][2] + v[c][3]);
        }
      }
    }
    if (more) put_keys<DP, W>(lds + (buf ^ 1) * Keys::halves, 1, wave, lane, false, u);
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float x = group_sum(mts[c] + mt[c]), y = group_sum(vts[c] + vt[c]);
    const int64_t rho = wave0 + 16 * c + lane;
    if (k8 == 0 && rho < A.M) {
      float* o = A.sums + ((int64_t)p.split * 2 * A.B * A.G + p.bg) * A.M + rho;
      o[0] = x, o[A.B * A.G * A.M] = y;
    }
  }
}

// The sums of the splits that reach a row, in order.
__device__ __forceinline__ void add_sums(const Args& A, const Place& p, int64_t rho, int lim, float& mt, float& vt) {
  const float* o = A.sums + p.bg * A.M + rho;
  const int64_t step = A.B * A.G * A.M;
  for (int i = 0; i < (lim + A.stat_chunk - 1) / A.stat_chunk; ++i, o += 2 * step) mt += o[0], vt += o[step];
}

template <int DP, bool VEC, int W>
__global__ void __launch_bounds__(64 * W) outputs_kernel(const Args A) {
  constexpr int DT = DP / 16, kRows = 16 * W;
  typedef Tile<DP, 18> KeysValues;
  constexpr int bufs = 2 * KeysValues::bytes <= kLdsBytes ? 2 : 1;
  constexpr bool ahead = units_of<DP, W>(2) == 1;  // the next tile waits in registers where they suffice
  extern __shared__ __align__(16) short lds[];
  const int64_t blocks = (A.M + kRows - 1) / kRows;
  Place p = place(A, blocks);
  if (A.causal) p.block = blocks - 1 - p.block;
  const Seq s = sequence(A, p.b);
  const int wave = wave_id(), lane = threadIdx.x & 63, k8 = lane >> 4;
  const int64_t block0 = p.block * kRows, wave0 = block0 + wave * 16, rho = wave0 + (lane & 15);
  const int lim = row_limit(A, s, rho), from = (A.launch * A.splits + p.split) * A.chunk;
  auto end = [&](int n) { return n < from + A.chunk ? n : from + A.chunk; };
  const int to = end(block_limit(A, s, block0, kRows)), wave_to = end(block_limit(A, s, wave0, 16));
  if (from >= to && from > 0) return;
  float mt = 0.f, vt = 0.f;
  if (lim) add_sums(A, p, rho, lim, mt, vt);
  if (from == 0 && k8 == 0 && rho < A.M)
    A.rows[stat_at(A, p.b, p.g, rho, 0)] = mt, A.rows[stat_at(A, p.b, p.g, rho, 1)] = vt;
  const RowSums rs = row_sums(mt, vt);
  Right<DP> q, Q, P;
  load_queries<DP, VEC>(A, lim ? row_at(A, A.lq, p.b, p.g, rho) : 0, lim > 0, k8, q, Q, P);
  // Heads of 128: two of a query's 36 operands wait in LDS, the registers for them are not there.
  static_assert(DP != 128 || bufs * KeysValues::bytes + 2 * 16 * 64 * W <= kLdsBytes, "they fit beside the tile");
  bf8* const kept = reinterpret_cast<bf8*>(lds + bufs * KeysValues::halves) + threadIdx.x;
  if constexpr (DP == 128) kept[0] = P.p[3].p[1], kept[64 * W] = P.p[3].p[2];
  const int whole = least(lim);
  float sum = 0.f;
  acc4 om[DT], oS[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) om[d] = oS[d] = acc4{0, 0, 0, 0};
  Unit u[1];
  if (from < to) pass_keys<DP, VEC, W>(A, p, from, to, lds, 2, wave, lane, true);
  __syncthreads();
  int buf = 0;
  at_line();
  for (int key0 = from; key0 < to; key0 += kTile) {
    const short *left = lds + hidden(buf * KeysValues::halves + 8 * lane),
                *turned = lds + hidden(buf * KeysValues::halves + turned_at(lane));
    const bool more = key0 + kTile < to;
    if constexpr (ahead) {
      if (more) fetch_keys<DP, VEC, W>(A, p, key0 + kTile, to, 2, wave, hidden(lane), true, u);
    }
    if (key0 < wave_to) {
      float w[8], kw[8];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        fence();
        if constexpr (DP == 128) P.p[3].p[1] = kept[0], P.p[3].p[2] = kept[64 * W];
        acc4 m, v;
        scores<DP>(left, kt, q, Q, P, m, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Weight x = weigh(rectify(m[r], v[r]), rs);
          w[4 * kt + r] = x.w, kw[4 * kt + r] = x.k;
          formed(w[4 * kt + r]), formed(kw[4 * kt + r]);
        }
      }
      if (key0 + kTile > whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = key0 + 16 * (i >> 2) + 4 * k8 + (i & 3) < lim ? w[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) kw[i] *= w[i] * w[i], sum += w[i];
      fence();
      {
        const Parts<3> b = split<3>(w);
#pragma unroll
        for (int d = 0; d < DT; ++d) om[d] = mma_transposed<DP>(turned, 9, d, b, om[d]);
      }
      fence();
      {
        const Parts<3> b = split<3>(kw);
#pragma unroll
        for (int d = 0; d < DT; ++d) oS[d] = mma_transposed<DP>(turned, 12, d, b, oS[d]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) kw[i] = fmaf(w[i], w[i], kw[i]);
      fence();
      {
        const Parts<3> b = split<3>(kw);
#pragma unroll
        for (int d = 0; d < DT; ++d) oS[d] = mma_transposed<DP>(turned, 15, d, b, oS[d]);
      }
    }
    if (bufs == 2) buf ^= 1;
    short* const next = lds + buf * KeysValues::halves;
    if constexpr (ahead) {
      if (bufs == 1) __syncthreads();
      if (more) put_keys<DP, W>(next, 2, wave, lane, true, u);
    } else {
      next_keys<DP, VEC, W, bufs == 1>(A, p, more ? key0 + kTile : to, to, next, wave, lane, true);
    }
    __syncthreads();
  }
  sum = group_sum(sum);
  if (rho >= A.M) return;
  if (A.parted) {
    float* o = A.parts + (((int64_t)p.split * A.B * A.G + p.bg) * A.M + rho) * (2 * A.D + 1);
    if (k8 == 0) o[2 * A.D] = sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * d + 4 * k8 + r;
        if (f < A.D) o[f] = om[d][r], o[A.D + f] = oS[d][r];
      }
    return;
  }
  if (k8 == 0) A.rows[stat_at(A, p.b, p.g, rho, 2)] = sum;
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor)), inv2 = inv * inv;
  const int64_t o = row_at(A, A.loq, p.b, p.g, rho);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * d + 4 * k8 + r;
      if (f < A.D) A.mo[o + f] = om[d][r] * inv, A.So[o + f] = oS[d][r] * inv2;
    }
}

// The parts that reach a row added in order to what earlier launches left of it; a wave to a row. NORM:
// divided by the weights' sum once they are complete.
template <bool NORM>
__global__ void __launch_bounds__(256) join_kernel(const Args A) {
  const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= A.B * A.G * A.M) return;
  const int width = 2 * A.D + (NORM ? 1 : 0);
  const int64_t bg = i / A.M, rho = i - bg * A.M, b = bg / A.G, step = A.B * A.G * A.M * width;
  const int g = (int)(bg - b * A.G), lane = threadIdx.x & 63;
  const int lim = row_limit(A, sequence(A, b), rho), chunks = (lim + A.chunk - 1) / A.chunk - A.launch * A.splits;
  if (chunks <= 0 && A.launch > 0) return;  // complete
  const int n = chunks < A.splits ? chunks : A.splits;
  const float* p = A.parts + i * width;
  float inv = 1.f;
  if constexpr (NORM) {
    float* const to = A.rows + stat_at(A, b, g, rho, 2);
    float sum = A.launch > 0 ? *to : 0.f;
    for (int k = 0; k < n; ++k) sum += p[k * step + 2 * A.D];
    if (lane == 0) *to = sum;
    if (chunks <= A.splits) inv = fast_rcp(fmaxf(sum, kRemaxFloor));
  }
  const int64_t o = row_at(A, A.loq, b, g, rho);
  for (int f = lane; f < A.D; f += 64) {
    float x = A.launch > 0 ? A.mo[o + f] : 0.f, y = A.launch > 0 ? A.So[o + f] : 0.f;
    for (int k = 0; k < n; ++k) x += p[k * step + f], y += p[k * step + A.D + f];
    A.mo[o + f] = x * inv, A.So[o + f] = y * (inv * inv);
  }
}

// --------------------------------------------------------------------------------- backward
// Deltas of the queries.
template <int DP, bool VEC, int W>
__global__ void __launch_bounds__(64 * W) dq_kernel(const Args A) {
  constexpr int DT = DP / 16, kRows = 16 * W;
  typedef Tile<DP, 15> KeysValues;
  constexpr int bufs = 2 * KeysValues::bytes <= kLdsBytes ? 2 : 1;
  constexpr bool ahead = units_of<DP, W>(2) == 1;
  extern __shared__ __align__(16) short lds[];
  const int64_t blocks = (A.M + kRows - 1) / kRows;
  Place p = place(A, blocks);
  if (A.causal) p.block = blocks - 1 - p.block;
  const Seq s = sequence(A, p.b);
  const int wave = wave_id(), lane = threadIdx.x & 63, k8 = lane >> 4;
  const int64_t block0 = p.block * kRows, wave0 = block0 + wave * 16, rho = wave0 + (lane & 15);
  const int lim = row_limit(A, s, rho), from = (A.launch * A.splits + p.split) * A.chunk;
  auto end = [&](int n) { return n < from + A.chunk ? n : from + A.chunk; };
  const int to = end(block_limit(A, s, block0, kRows)), wave_to = end(block_limit(A, s, wave0, 16));
  if (from >= to && from > 0) return;
  float mt = 0.f, vt = 0.f, sum = 0.f;
  if (lim)
    mt = A.rows[stat_at(A, p.b, p.g, rho, 0)], vt = A.rows[stat_at(A, p.b, p.g, rho, 1)],
    sum = A.rows[stat_at(A, p.b, p.g, rho, 2)];
  const RowSums rs = row_sums(mt, vt);
  const float inv = fast_rcp(fmaxf(sum, kRemaxFloor));
  Right<DP> q, Q, P, dm, dS;
  load_queries<DP, VEC>(A, lim ? row_at(A, A.lq, p.b, p.g, rho) : 0, lim > 0, k8, q, Q, P);
  load_right<DP, VEC>(A.dm, A.dS, lim ? row_at(A, A.ld, p.b, p.g, rho) : 0, A.D, lim > 0, k8,
                      [&](int st, float (&m)[8], float (&S)[8]) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) m[i] *= A.c, S[i] *= A.c2;
                        dm.p[st] = split<3>(m), dS.p[st] = split<3>(S);
                      });
  const int whole_tiles = least(lim);
  acc4 om[DT], oS[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) om[d] = oS[d] = acc4{0, 0, 0, 0};
  Unit u[1];
  if (from < to) pass_keys<DP, VEC, W>(A, p, from, to, lds, 2, wave, lane, false);
  __syncthreads();
  int buf = 0;
  at_line();
  for (int key0 = from; key0 < to; key0 += kTile) {
    const short *left = lds + hidden(buf * KeysValues::halves + 8 * lane),
                *turned = lds + hidden(buf * KeysValues::halves + turned_at(lane));
    const bool more = key0 + kTile < to;
    if constexpr (ahead) {
      if (more) fetch_keys<DP, VEC, W>(A, p, key0 + kTile, to, 2, wave, hidden(lane), false, u);
    }
    if (key0 < wave_to) {
      float x[8], X[8];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        fence();
        acc4 m, v;
        scores<DP>(left, kt, q, Q, P, m, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Rectified z = rectify(m[r], v[r]);
          const Weight w = weigh(z, rs);
          float J = remax_jacobian(z, w, w.w * inv);
          formed(J);
          m[r] = J;
        }
        acc4 e = {0, 0, 0, 0}, E = e;
#pragma unroll
        for (int st = 0; st < DP / 32; ++st) {
          e = mma_left<DP>(left, 9, kt, st, dm.p[st], e);
          E = mma_left<DP>(left, 12, kt, st, dS.p[st], E);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) x[4 * kt + r] = e[r] * m[r], X[4 * kt + r] = E[r] * (m[r] * m[r]);
      }
      if (key0 + kTile > whole_tiles) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool seen = key0 + 16 * (i >> 2) + 4 * k8 + (i & 3) < lim;
          x[i] = seen ? x[i] : 0.f, X[i] = seen ? X[i] : 0.f;
        }
      }
      fence();
      {
        const Parts<3> b = split<3>(x);
#pragma unroll
        for (int d = 0; d < DT; ++d) om[d] = mma_transposed<DP>(turned, 0, d, b, om[d]);
      }
      fence();
      {
        const Parts<3> b = split<3>(X);
#pragma unroll
        for (int d = 0; d < DT; ++d) oS[d] = mma_transposed<DP>(turned, 3, d, b, oS[d]);
      }
    }
    if (bufs == 2) buf ^= 1;
    short* const next = lds + buf * KeysValues::halves;
    if constexpr (ahead) {
      if (bufs == 1) __syncthreads();
      if (more) put_keys<DP, W>(next, 2, wave, lane, false, u);
    } else {
      next_keys<DP, VEC, W, bufs == 1>(A, p, more ? key0 + kTile : to, to, next, wave, lane, false);
    }
    __syncthreads();
  }
  if (rho >= A.M) return;
  const bool whole = !A.parted;
  float* const to_m = whole ? A.mo + row_at(A, A.loq, p.b, p.g, rho)
                            : A.parts + (((int64_t)p.split * A.B * A.G + p.bg) * A.M + rho) * (2 * A.D);
  float* const to_S = whole ? A.So + row_at(A, A.loq, p.b, p.g, rho) : to_m + A.D;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * d + 4 * k8 + r;
      if (f < A.D) to_m[f] = om[d][r], to_S[f] = oS[d][r];
    }
}

// Rows that see a key of a block from key0 on: [first, end).
struct RowRange {
  int64_t first, end;
};
__device__ __forceinline__ RowRange rows_of(const Args& A, const Seq& s, int key0) {
  if (key0 >= s.len) return {0, 0};
  // positions from 0, and with causal from the first key, to the length
  int64_t first = (A.causal ? key0 : 0) - s.start, last = s.len - s.start;
  if (first < 0) first = 0;
  if (last > A.T) last = A.T;
  return first < last ? RowRange{first * A.R, last * A.R} : RowRange{0, 0};
}

// Deltas of the keys and values: a wave holds 16 keys, the block walks the rows that see them.
// Parts of a row: c q 0, c^2 Sq 3, (c q)^2 6 (against k, k^2 + Sk, Sk); dm 9, dS 12. The scale of the
// scores' deltas is that of the queries they multiply.
// KEYS, VALUES: which of the two: both where registers hold four sums of a head (up to 96 features),
// else one after the other, with the scores formed once more.
template <int DP, bool VEC, int W, bool KEYS, bool VALUES>
__global__ void __launch_bounds__(64 * W) dkv_kernel(const Args A) {
  constexpr int S = DP / 32, DT = DP / 16, kKeys = 16 * W;
  typedef Tile<DP, 15> Queries;
  constexpr int bufs = 2 * Queries::bytes + 2 * 5 * kTile * 4 <= kLdsBytes ? 2 : 1;
  extern __shared__ __align__(16) short lds[];
  constexpr bool ahead = units_of<DP, W>(2) == 1;
  // [buffer][5][kTile]: 1 / mt, vt, c_mt, 1 / s, limit
  float* const stats = reinterpret_cast<float*>(lds + bufs * Queries::halves);
  const Place p = place(A, (A.N + kKeys - 1) / kKeys);
  const Seq s = sequence(A, p.b);
  const int wave = wave_id(), lane = threadIdx.x & 63, k8 = lane >> 4;
  const int key0 = (int)p.block * kKeys, wave_key = key0 + wave * 16, key = wave_key + (lane & 15);
  const RowRange all = rows_of(A, s, key0), mine = rows_of(A, s, wave_key);
  const int64_t chunk0 = ((int64_t)A.launch * A.splits + p.split) * A.chunk, chunk1 = chunk0 + A.chunk;
  const int64_t from = all.first > chunk0 ? all.first : chunk0, to = all.end < chunk1 ? all.end : chunk1;
  if (from >= to && A.parted) return;
  // zeros in place of a key behind the last query: whatever it holds would be NaN times a weight of 0
  const bool on = key < s.len && (!A.causal || key < s.start + A.T);
  constexpr int DK = KEYS ? DT : 1, DV = VALUES ? DT : 1;
  Right<DP> k, K, Sk, vm, vv;
  load_right<DP, VEC>(A.mk, A.Sk, on ? key_at(A.lk, p.b, p.g, key) : 0, A.D, on, k8,
                      [&](int st, float (&m)[8], float (&x)[8]) {
                        k.p[st] = split<3>(m), Sk.p[st] = split<3>(x);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = fmaf(m[i], m[i], x[i]);
                        K.p[st] = split<3>(x);
                      });
  if constexpr (KEYS)
    load_right<DP, VEC>(A.mv, A.mv, on ? key_at(A.lv, p.b, p.g, key) : 0, A.D, on, k8,
                      [&](int st, float (&m)[8], float (&x)[8]) {
                        vm.p[st] = split<3>(m);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] *= x[i];
                        vv.p[st] = split<3>(x);
                      });
  acc4 okm[DK], okS[DK], ovm[DV], ovS[DV];
#pragma unroll
  for (int d = 0; d < DK; ++d) okm[d] = okS[d] = acc4{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < DV; ++d) ovm[d] = ovS[d] = acc4{0, 0, 0, 0};
  auto fetch_unit = [&](int64_t rho0, int i, int ln, Unit& u) {
    const bool delta = i >= 2 * S;
    const int n = delta ? i - 2 * S : i, kt = n / S, st = n % S;
    const int64_t rho = rho0 + 16 * kt + (ln & 15);
    const bool in = rho < to;
    const int64_t at = in ? row_at(A, delta ? A.ld : A.lq, p.b, p.g, rho) : 0;
    load8<VEC>((delta ? A.dm : A.mq) + at, 32 * st + 8 * (ln >> 4), A.D, in, u.m);
    load8<VEC>((delta ? A.dS : A.Sq) + at, 32 * st + 8 * (ln >> 4), A.D, in, u.S);
  };
  auto store_unit = [&](short* tile, int i, int ln, Unit& u) {
    const bool delta = i >= 2 * S;
    const int n = delta ? i - 2 * S : i, kt = n / S, st = n % S, first = delta ? 9 : 0;
    const float c = delta ? 1.f : A.c, c2 = delta ? 1.f : A.c2;
#pragma unroll
    for (int e = 0; e < 8; ++e) u.m[e] *= c, u.S[e] *= c2;
    put<DP>(tile, first, kt, st, ln, split<3>(u.m));
    put<DP>(tile, first + 3, kt, st, ln, split<3>(u.S));
    if (!delta) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u.m[e] *= u.m[e];
      put<DP>(tile, 6, kt, st, ln, split<3>(u.m));
    }
  };
  // a row of the tile for each of the first threads
  auto row_stats = [&](int64_t rho0, int buf) {
    const int tid = wave * 64 + hidden(lane);
    if (tid >= kTile) return;
    const int64_t rho = rho0 + tid;
    const int lim = rho < to ? row_limit(A, s, rho) : 0;
    float x[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) x[i] = lim ? A.rows[stat_at(A, p.b, p.g, rho, i)] : 0.f;
    const RowSums r = row_sums(x[0], x[1]);
    float* o = stats + buf * 5 * kTile + tid;
    o[0] = r.inv_mt, o[kTile] = r.vt, o[2 * kTile] = r.c_mt, o[3 * kTile] = fast_rcp(fmaxf(x[2], kRemaxFloor));
    o[4 * kTile] = __int_as_float(lim);
  };
  auto pass_rows = [&](int64_t rho0, int buf) {
    Unit u;
#pragma unroll 1
    for (int i = wave; i < 4 * S; i += W) {
      fetch_unit(rho0, i, hidden(lane), u);
      store_unit(lds + buf * Queries::halves, i, hidden(lane), u);
    }
    row_stats(rho0, buf);
  };
  Unit u;
  if (from < to) pass_rows(from, 0);
  __syncthreads();
  int buf = 0;
  at_line();
  for (int64_t rho0 = from; rho0 < to; rho0 += kTile) {
    const short *left = lds + hidden(buf * Queries::halves + 8 * lane),
                *turned = lds + hidden(buf * Queries::halves + turned_at(lane));
    const float* st = stats + buf * 5 * kTile;
    const bool more = rho0 + kTile < to;
    const bool busy = wave_key < s.len && rho0 + kTile > mine.first;
    if (busy) {
      float a[8], J[8];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        fence();
        acc4 m, v;
        scores<DP>(left, kt, k, K, Sk, m, v);
        const float* const row = st + 16 * kt + 4 * k8;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if ((r & 1) == 0) fence();  // two scores at a time: the registers of four are not there
          const RowSums rs{row[r], row[kTile + r], row[2 * kTile + r]};
          const Rectified z = rectify(m[r], v[r]);
          const Weight w = weigh(z, rs);
          const float n = key < __float_as_int(row[4 * kTile + r]) ? w.w * row[3 * kTile + r] : 0.f;
          a[4 * kt + r] = n;
          formed(a[4 * kt + r]);
          if constexpr (KEYS) {
            J[4 * kt + r] = remax_jacobian(z, w, a[4 * kt + r]);
            formed(J[4 * kt + r]);
          }
        }
      }
      if constexpr (KEYS) {
        float x[8];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          fence();
          acc4 e = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < S; ++i) e = mma_left<DP>(left, 9, kt, i, vm.p[i], e);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[4 * kt + r] = e[r] * J[4 * kt + r];
        }
        fence();
        {
          const Parts<3> b = split<3>(x);
#pragma unroll
          for (int d = 0; d < DT; ++d) okm[d] = mma_transposed<DP>(turned, 0, d, b, okm[d]);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          fence();
          acc4 E = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < S; ++i) E = mma_left<DP>(left, 12, kt, i, vv.p[i], E);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[4 * kt + r] = E[r] * (J[4 * kt + r] * J[4 * kt + r]);
        }
        fence();
        {
          const Parts<3> b = split<3>(x);
#pragma unroll
          for (int d = 0; d < DT; ++d) okS[d] = mma_transposed<DP>(turned, 6, d, b, okS[d]);
        }
      }
      fence();
      if (ahead && more && wave < 4 * S) fetch_unit(rho0 + kTile, wave, hidden(lane), u);  // here its registers are free
      if constexpr (VALUES) {
        fence();
        {
          const Parts<3> b = split<3>(a);
#pragma unroll
          for (int d = 0; d < DT; ++d) ovm[d] = mma_transposed<DP>(turned, 9, d, b, ovm[d]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] *= a[i];
        fence();
        {
          const Parts<3> b = split<3>(a);
#pragma unroll
          for (int d = 0; d < DT; ++d) ovS[d] = mma_transposed<DP>(turned, 12, d, b, ovS[d]);
        }
      }
    }
    if (ahead && more && !busy && wave < 4 * S) fetch_unit(rho0 + kTile, wave, hidden(lane), u);
    if (bufs == 2) buf ^= 1;
    short* const next = lds + buf * Queries::halves;
    if constexpr (ahead) {
      if (bufs == 1) __syncthreads();
      if (more && wave < 4 * S) store_unit(next, wave, hidden(lane), u);
    } else {
      constexpr int n = 4 * S / W;
      static_assert(n * W == 4 * S, "whole units for each wave");
      const int64_t rho1 = more ? rho0 + kTile : to;
      Unit v[n];  // only here: it would take the products' registers
      fence();
#pragma unroll
      for (int j = 0; j < n; ++j) fetch_unit(rho1, wave + j * W, hidden(lane), v[j]);
      if (bufs == 1) __syncthreads();
#pragma unroll
      for (int j = 0; j < n; ++j) {
        fence();
        store_unit(next, wave + j * W, hidden(lane), v[j]);
      }
    }
    if (more) row_stats(rho0 + kTile, buf);
    __syncthreads();
  }
  if (key >= A.N) return;
  const bool whole = !A.parted;
  const int64_t at = whole ? key_at(A.lokv, p.b, p.g, key) : (((int64_t)p.split * A.B * A.G + p.bg) * A.N + key) * (4 * A.D);
  auto put_out = [&](float* out, int i, const auto& x) {
    float* const o = (whole ? out : A.parts + i * A.D) + at;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * d + 4 * k8 + r;
        if (f < A.D) o[f] = x[d][r];
      }
  };
  if constexpr (KEYS) put_out(A.dmk, 0, okm), put_out(A.dSk, 1, okS);
  if constexpr (VALUES) put_out(A.dmv, 2, ovm), put_out(A.dSv, 3, ovS);
}

// The parts of the rows that see a key, in order, added to what earlier launches left; a wave to a key.
// kv_keys: keys of a dkv block.
__global__ void __launch_bounds__(256) join_keys_kernel(const Args A, int kv_keys) {
  const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= A.B * A.G * A.N) return;
  const int64_t bg = i / A.N, b = bg / A.G, step = A.B * A.G * A.N * (4 * A.D);
  const int key = (int)(i - bg * A.N), g = (int)(bg - b * A.G);
  const RowRange r = rows_of(A, sequence(A, b), key / kv_keys * kv_keys);
  // chunks of rows, from those of this launch on
  const int before = A.launch * A.splits, k0 = (int)(r.first / A.chunk) - before;
  const int k1 = (int)((r.end + A.chunk - 1) / A.chunk) - before;
  if (A.launch > 0 && (k1 <= 0 || k0 >= A.splits)) return;
  const bool more = k0 < 0;
  const int from = k0 < 0 ? 0 : k0, to = k1 < A.splits ? k1 : A.splits;
  const float* p = A.parts + i * (4 * A.D);
  const int64_t o = key_at(A.lokv, b, g, key);
  for (int f = threadIdx.x & 63; f < 4 * A.D; f += 64) {
    const int q = f / A.D;
    float* const out = (q == 0 ? A.dmk : (q == 1 ? A.dSk : (q == 2 ? A.dmv : A.dSv))) + o + f - q * A.D;
    float x = more ? *out : 0.f;
    if (r.first < r.end)
      for (int k = from; k < to; ++k) x += p[k * step + f];
    *out = x;
  }
}

// ------------------------------------------------------------------------------------ plans
constexpr int kStatsWaves = 8, kOutWaves = 8;
// Nothing lies in scratch memory (build.py refuses it here): in kernels of four waves operands of four
// registers that the compiler had put there, beside accumulation registers, came back wrong.
//
// Waves of a backward block. Five right operands of 96 (128) features take 180 (240) registers: one
// wave a SIMD has 512; eight waves would keep them in scratch memory.
template <int DP>
constexpr int back_waves() {
  return DP > 64 ? 4 : 8;
}
int back_rows(int64_t D) { return 16 * (D > 64 ? 4 : 8); }

// Chunks of `walked` for blocks of `rows` of `own` on each of BG key heads: as many as fill the
// GPU three times over, at least 256 walked each (a block's own operands are loaded and split again
// for each) and at most `most`. A launch's splits have their own parts in the workspace, 8192 blocks' worth
// at most, so that it does not grow with both lengths; further chunks take further launches, whose last
// rounds causal blocks leave half empty: 16384 tokens, 32 heads of 128 over 8, both directions, 360 ms and
// 1.1 GB; 16384 blocks' worth 358 and 2.2; 4096 blocks' 369 and 0.5; all chunks at once 353 and 8.7.
struct Splits {
  int n, chunk, launches, stat_chunk;
  bool parted() const { return n > 1 || launches > 1; }
};
Splits splits_of(int64_t own, int64_t rows, int64_t BG, int64_t walked, int64_t most) {
  const int64_t blocks = cdiv(own, rows) * BG, room = cdiv(8192, blocks < 1 ? 1 : blocks);
  int64_t n = cdiv(768, blocks < 1 ? 1 : blocks);
  if (n > cdiv(walked, 256)) n = cdiv(walked, 256);
  if (n < cdiv(walked, most)) n = cdiv(walked, most);
  if (n < 1) n = 1;
  const int64_t launches = cdiv(n, room), splits = cdiv(n, launches);
  auto tiles = [&](int64_t chunks) {
    const int64_t x = cdiv(cdiv(walked, chunks), kTile) * kTile;
    return (int)(x < kTile ? kTile : x);
  };
  return {(int)splits, tiles(splits * launches), (int)launches, tiles(splits)};
}
void set(Args& a, const Splits& sp) {
  a.splits = sp.n, a.chunk = sp.chunk, a.parted = sp.parted(), a.stat_chunk = sp.stat_chunk;
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t N, int64_t H, int64_t G, int64_t D) {
  TAGI_REQUIRE(B >= 0 && T >= 0 && N >= 0 && H > 0 && G > 0 && D > 0 && H % G == 0, "%s: bad sizes", what);
  if (D > kMaxDim) return fail(TAGI_ERR_UNSUPPORTED, "%s: head dimension above %d", what, kMaxDim);
  TAGI_REQUIRE(B < 65536 && G < 65536 && B * G < 65536 && H < (1 << 20) && T < (1 << 30) && N < (1 << 30) &&
                   T * (H / G) < (1ll << 30), "%s: too large", what);
  return TAGI_OK;
}

// 1-D launches of blocks * splits on every key head: fewer than 2^32 threads.
int grid_of(const char* what, int64_t own, int64_t rows, int64_t BG, int splits, int threads, dim3* grid) {
  const int64_t n = cdiv(own, rows) * BG * splits;
  TAGI_REQUIRE(n * threads < (1ll << 32), "%s: too large", what);
  *grid = dim3((unsigned)n);
  return TAGI_OK;
}
dim3 join_grid(int64_t rows) {
  const int64_t blocks = cdiv(rows, 4), x = blocks < (1 << 20) ? blocks : (1 << 20);
  return dim3((unsigned)x, (unsigned)cdiv(blocks, x));
}
template <typename K>
void go(K kernel, dim3 grid, int threads, int lds, hipStream_t s, const Args& a) {
  if (lds > 64 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, s, a);
}
constexpr int two_or_one(int bytes, int more) { return (2 * (bytes + more) <= kLdsBytes ? 2 : 1) * (bytes + more); }

template <int DP, bool VEC>
int forward(const char* what, Args a, int launches, hipStream_t s) {
  const int64_t BG = a.B * a.G;
  constexpr int NC = DP > 64 ? 1 : 2, kept = DP == 128 ? 2 * 16 * 64 * kOutWaves : 0;
  dim3 grid;
  if (int rc = grid_of(what, a.M, 16 * kStatsWaves * NC, BG, a.splits, 64 * kStatsWaves, &grid)) return rc;
  dim3 out;
  if (int rc = grid_of(what, a.M, 16 * kOutWaves, BG, a.splits, 64 * kOutWaves, &out)) return rc;
  go(stats_kernel<DP, VEC, kStatsWaves, NC>, grid, 64 * kStatsWaves, 2 * Tile<DP, 9>::bytes, s, a);
  for (a.launch = 0; a.launch < launches; ++a.launch) {
    go(outputs_kernel<DP, VEC, kOutWaves>, out, 64 * kOutWaves, two_or_one(Tile<DP, 18>::bytes, 0) + kept, s, a);
    if (a.parted) hipLaunchKernelGGL(join_kernel<true>, join_grid(BG * a.M), dim3(256), 0, s, a);
  }
  return TAGI_OK;
}
template <int DP, bool VEC>
int backward(const char* what, Args a, float* ws, hipStream_t s) {
  const int64_t BG = a.B * a.G;
  constexpr int W = back_waves<DP>(), rows = 16 * W;
  if (a.T) {
    const Splits sp = splits_of(a.M, rows, BG, a.N, kMostWalkedBack);
    set(a, sp), a.parts = ws;
    dim3 grid;
    if (int rc = grid_of(what, a.M, rows, BG, sp.n, 64 * W, &grid)) return rc;
    for (a.launch = 0; a.launch < sp.launches; ++a.launch) {
      go(dq_kernel<DP, VEC, W>, grid, 64 * W, two_or_one(Tile<DP, 15>::bytes, 0), s, a);
      if (a.parted) hipLaunchKernelGGL(join_kernel<false>, join_grid(BG * a.M), dim3(256), 0, s, a);
    }
  }
  if (a.N) {
    const Splits sp = splits_of(a.N, rows, BG, a.M, kMostWalkedBack);
    set(a, sp), a.parts = ws;  // the stream's order keeps the joins apart
    dim3 grid;
    if (int rc = grid_of(what, a.N, rows, BG, sp.n, 64 * W, &grid)) return rc;
    const int lds = two_or_one(Tile<DP, 15>::bytes, 5 * kTile * 4);
    for (a.launch = 0; a.launch < sp.launches; ++a.launch) {
      if constexpr (DP == 128) {
        go(dkv_kernel<DP, VEC, W, true, false>, grid, 64 * W, lds, s, a);
        go(dkv_kernel<DP, VEC, W, false, true>, grid, 64 * W, lds, s, a);
      } else {
        go(dkv_kernel<DP, VEC, W, true, true>, grid, 64 * W, lds, s, a);
      }
      if (a.parted) hipLaunchKernelGGL(join_keys_kernel, join_grid(BG * a.N), dim3(256), 0, s, a, rows);
    }
  }
  return TAGI_OK;
}

// rows of whole groups of eight features
bool vec8(int64_t D) { return D % 8 == 0; }
#define BY_DIM_OF(run, vec, ...)                                                       \
  (D <= 32 ? run<32, vec>(__VA_ARGS__)                                                  \
           : (D <= 64 ? run<64, vec>(__VA_ARGS__)                                       \
                      : (D <= 96 ? run<96, vec>(__VA_ARGS__) : run<128, vec>(__VA_ARGS__))))
#define BY_DIM(run, ...) (vec8(D) ? BY_DIM_OF(run, true, __VA_ARGS__) : BY_DIM_OF(run, false, __VA_ARGS__))

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int64_t tagi_remax_attention_fwd_ws_bytes(int64_t B, int64_t T, int64_t N, int64_t H, int64_t G,
                                                     int64_t D) {
  if (B <= 0 || T <= 0 || N < 0 || H <= 0 || G <= 0 || D <= 0 || H % G) return 0;
  const Splits sp = splits_of(T * (H / G), 16 * kOutWaves, B * G, N, kMostWalked);
  return 4 * B * H * T * sp.n * (2 + (sp.parted() ? 2 * D + 1 : 0));
}

extern "C" int tagi_remax_attention_fwd(const float* mq, const float* Sq, const tagi_heads* lq, const float* mk,
                                        const float* Sk, const tagi_heads* lk, const float* mv, const float* Sv,
                                        const tagi_heads* lv, const void* lengths, int len_bytes, const void* starts,
                                        int start_bytes, int causal, float* mo, float* So, float* rows, int64_t B,
                                        int64_t T, int64_t N, int64_t H, int64_t G, int64_t D, double scale, void* ws,
                                        int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_remax_attention_fwd";
  if (int rc = check_sizes(what, B, T, N, H, G, D)) return rc;
  if (B == 0 || T == 0) return TAGI_OK;
  TAGI_REQUIRE(mq && Sq && lq && mo && So && rows && (N == 0 || (mk && Sk && lk && mv && Sv && lv)),
               "%s: null pointer", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(!starts || start_bytes == 4 || start_bytes == 8, "%s: starts are int32 or int64", what);
  TAGI_REQUIRE(ws && ws_bytes >= tagi_remax_attention_fwd_ws_bytes(B, T, N, H, G, D), "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 18.0 * B * H * T * N * D * (causal && T == N ? 0.5 : 1.0),
               16.0 * D * B * (T * H + N * G));
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.Sv = Sv, a.lq = *lq;
  if (N) a.lk = *lk, a.lv = *lv;
  a.lengths = lengths, a.len_bytes = len_bytes, a.starts = starts, a.start_bytes = start_bytes, a.causal = causal != 0;
  a.mo = mo, a.So = So, a.rows = rows, a.loq = tagi_heads{T * H * D, H * D, D};
  a.B = B, a.T = (int)T, a.N = (int)N, a.H = (int)H, a.G = (int)G, a.R = (int)(H / G), a.D = (int)D, a.M = T * (H / G);
  a.c = (float)scale, a.c2 = (float)(scale * scale);
  const Splits sp = splits_of(a.M, 16 * kOutWaves, B * G, N, kMostWalked);
  set(a, sp);
  a.sums = static_cast<float*>(ws), a.parts = a.sums + 2 * a.splits * B * H * T;
  if (int rc = BY_DIM(forward, what, a, sp.launches, s)) return rc;
  return check_launch(what);
}

extern "C" int64_t tagi_remax_attention_bwd_ws_bytes(int64_t B, int64_t T, int64_t N, int64_t H, int64_t G,
                                                     int64_t D) {
  if (B <= 0 || T < 0 || N < 0 || H <= 0 || G <= 0 || D <= 0 || H % G) return 0;
  const int64_t M = T * (H / G), rows = back_rows(D);
  const Splits q = splits_of(M, rows, B * G, N, kMostWalkedBack), kv = splits_of(N, rows, B * G, M, kMostWalkedBack);
  const int64_t a = q.parted() ? q.n * B * G * M * 2 * D : 0, b = kv.parted() ? kv.n * B * G * N * 4 * D : 0;
  return 4 * (a > b ? a : b);
}

extern "C" int tagi_remax_attention_bwd(const float* mq, const float* Sq, const tagi_heads* lq, const float* mk,
                                        const float* Sk, const tagi_heads* lk, const float* mv, const tagi_heads* lv,
                                        const float* dmo, const float* dSo, const tagi_heads* ldo, const float* rows,
                                        const void* lengths, int len_bytes, const void* starts, int start_bytes,
                                        int causal, float* dmq, float* dSq, const tagi_heads* ldq, float* dmk,
                                        float* dSk, float* dmv, float* dSv, const tagi_heads* ldkv, int64_t B,
                                        int64_t T, int64_t N, int64_t H, int64_t G, int64_t D, double scale, void* ws,
                                        int64_t ws_bytes, tagi_stream_t stream) {
  const char* what = "tagi_remax_attention_bwd";
  if (int rc = check_sizes(what, B, T, N, H, G, D)) return rc;
  if (B == 0) return TAGI_OK;
  TAGI_REQUIRE(T == 0 || (mq && Sq && lq && dmo && dSo && ldo && rows && dmq && dSq && ldq), "%s: null pointer", what);
  TAGI_REQUIRE(N == 0 || (mk && Sk && lk && mv && lv && dmk && dSk && dmv && dSv && ldkv), "%s: null pointer", what);
  TAGI_REQUIRE(!lengths || len_bytes == 4 || len_bytes == 8, "%s: lengths are int32 or int64", what);
  TAGI_REQUIRE(!starts || start_bytes == 4 || start_bytes == 8, "%s: starts are int32 or int64", what);
  const int64_t need = tagi_remax_attention_bwd_ws_bytes(B, T, N, H, G, D);
  TAGI_REQUIRE(need == 0 || (ws && ws_bytes >= need), "%s: workspace too small", what);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(FAM_ATTN_SCORES, s, 28.0 * B * H * T * N * D * (causal && T == N ? 0.5 : 1.0),
               D * B * (24.0 * T * H + 28.0 * N * G));
  Args a{};
  a.mq = mq, a.Sq = Sq, a.mk = mk, a.Sk = Sk, a.mv = mv, a.dm = dmo, a.dS = dSo;
  if (T) a.lq = *lq, a.ld = *ldo, a.loq = *ldq;
  if (N) a.lk = *lk, a.lv = *lv, a.lokv = *ldkv;
  a.lengths = lengths, a.len_bytes = len_bytes, a.starts = starts, a.start_bytes = start_bytes, a.causal = causal != 0;
  a.mo = dmq, a.So = dSq, a.rows = const_cast<float*>(rows), a.dmk = dmk, a.dSk = dSk, a.dmv = dmv, a.dSv = dSv;
  a.B = B, a.T = (int)T, a.N = (int)N, a.H = (int)H, a.G = (int)G, a.R = (int)(H / G), a.D = (int)D, a.M = T * (H / G);
  a.c = (float)scale, a.c2 = (float)(scale * scale);
  if (int rc = BY_DIM(backward, what, a, static_cast<float*>(ws), s)) return rc;
  return check_launch(what);
}
