// Newton-Schulz orthogonalisation of a batch of matrices and the Muon update
// built on it (gfx950).
//
//   X0 = G / max(|G|_F, eps);  steps times:  A = X X^T,  B = b A + c A A,
//   X <- a X + B X                            (on G^T where rows > cols)
// (a joins B's diagonal, so X <- B X: the product reads no X beside its operand)
//
// The quintic pushes every singular value of X towards 1 (Muon: K. Jordan,
// 2024; Newton-Schulz iterations: Bjorck & Bowie, 1971).  Muon's update:
//   buf <- beta buf + g,  u = g + beta buf (Nesterov) or buf,
//   W <- (1 - lr decay) W - lr scale NS(u).
//
// Precision.  The iteration amplifies a perturbation of a small singular
// direction by up to a^steps (485 for the default): with X in one fp16 the
// result of a rank-64 gradient is 11 bf16 roundings off.  Every matrix is
// therefore held as two fp16 numbers, v S = hi + lo (22 significant bits), and
// every product is three fp16 MFMA products, hi hi + hi lo + lo hi, summed in
// one fp32 accumulator; the dropped lo lo term is below 2^-22 of the result.
// Three products at the fp16 rate are still five times the rate of the fp32
// MFMA.  S is a power of two per matrix kind: as large as fp16's range allows
// (|X| < 2, |A| < 4, |B| < 16), so that the lo halves stay clear of fp16's
// smallest numbers (X0 of 2^30 entries has a root mean square of 1 in units of
// 1 / S, its lo halves a spacing of 2^-24).
//
// Layout.  A plane (the hi or the lo half of a matrix with R rows and
// contraction length K, both padded to 32 with zeros) is stored as
// [R/32][K/8][32][8] halves: two neighbouring octet columns (32 rows x 16 k) are
// one 1 KB operand fragment of v_mfma_f32_32x32x16_f16, so global -> LDS copies
// and LDS -> register reads are linear.  X is kept in both orientations: Xr
// (rows m, contraction n) for A = X X^T and Xc (rows n, contraction m) for
// B X; an accumulator holds four consecutive i of one j, which is a contiguous
// 8-byte piece of the (row j, contraction i) form, and the other form is
// transposed through LDS.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_common.h"

namespace lcn {

namespace {

constexpr float kSx = 32768.f, kSa = 16384.f, kSb = 4096.f;  // scales of X, A, B
constexpr int kNormParts = 512;                             // most partial sums of squares per matrix

__host__ __device__ inline int64_t pad32(int64_t v) { return (v + 31) / 32 * 32; }

// per-matrix workspace, in bytes from its start
struct NsPlan {
  int m, n;                 // short / long side
  int mp, np;               // padded
  int64_t xplane, aplane;   // bytes of a plane
  int64_t x[2], a, b;       // Xr hi, Xr lo, Xc hi, Xc lo (twice); A hi, lo; B hi, lo
  int64_t stride;
  int slices;               // of K in the Gram product
  int64_t parts;            // bytes of its partial sums, all matrices
};
NsPlan make_plan(int64_t batch, int64_t rows, int64_t cols) {
  NsPlan p;
  p.m = (int)std::min(rows, cols);
  p.n = (int)std::max(rows, cols);
  p.mp = (int)pad32(p.m);
  p.np = (int)pad32(p.n);
  p.xplane = (int64_t)p.mp * p.np * 2;
  p.aplane = (int64_t)p.mp * p.mp * 2;
  p.x[0] = 0;
  p.x[1] = 4 * p.xplane;
  p.a = 8 * p.xplane;
  p.b = p.a + 2 * p.aplane;
  p.stride = p.b + 2 * p.aplane;
  // A 64 x 64 tile goes through 32 of K in 0.2 us; parts of K cost 5 us for their
  // launch and sums, so they are taken where they shorten the product by 40 stages
  // and more: one 333 x 7000 327 -> 194 us, one 140 x 4000 204 -> 139.
  const int64_t c = (p.m + 63) / 64, tiles = batch * c * (c + 1) / 2;
  const int stages = p.np / 32;
  int slices = (int)std::min<int64_t>(256 / tiles, stages / 8);
  if (slices > 1) slices = (stages + (stages + slices - 1) / slices - 1) / ((stages + slices - 1) / slices);  // none empty
  p.slices = slices > 1 && stages - stages / slices >= 40 ? slices : 1;
  p.parts = p.slices > 1 ? p.slices * tiles * 16384 : 0;
  return p;
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// ---- norm (and, for muon, the momentum update) ---------------------------------------------
// part[b][p] = sum of squares, in float64, of the rows this workgroup walks.  A
// wave takes a row at a time, kU pieces of kE elements a lane in flight (16 bytes
// each where the rows are aligned, else single elements); bound by the read of G
// (six 1088 x 1088: 28 us with one element in flight and 64 workgroups, 13.5 with
// eight elements, 7.7 with five pieces; 4352 x 4352 bf16 58 and 15).
template <int T, bool kMuon, bool kWide>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs a, double* __restrict__ part) {
  constexpr int kE = !kWide ? 1 : T == kOpF32 ? 4 : 8, kU = !kWide ? 8 : kMuon && T != kOpF32 ? 2 : 5;
  __shared__ double red[4];
  const int64_t b = blockIdx.y;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int pieces = a.cols / kE;
  double s = 0.0;
  for (int r = blockIdx.x * 4 + ty; r < a.rows; r += gridDim.x * 4) {
    const int64_t g0 = b * a.in.batch + (int64_t)r * a.in.row;
    float* mom = kMuon ? (float*)a.momentum.p + b * a.momentum.batch + (int64_t)r * a.momentum.row : nullptr;
    for (int c0 = tx; c0 < pieces; c0 += 64 * kU) {
      float v[kU][kE], m[kU][kE];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int c = c0 + 64 * u;
        const bool in = c < pieces;
#pragma unroll
        for (int e = 0; e < kE; ++e) v[u][e] = m[u][e] = 0.f;
        if constexpr (!kWide) {
          if (in) v[u][0] = op_load<T>(a.in.p, g0 + c);
          if (kMuon && in) m[u][0] = mom[c];
        } else {
          if (in) unpack_vec<T>(*(const v4u*)((const char*)a.in.p + (g0 + (int64_t)c * kE) * (16 / kE)), v[u]);
          if constexpr (kMuon) {
#pragma unroll
            for (int e = 0; e < kE; e += 4)
              if (in) unpack_vec<kOpF32>(*(const v4u*)(mom + c * kE + e), *(float(*)[4])(m[u] + e));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if constexpr (kMuon) {
#pragma unroll
          for (int e = 0; e < kE; ++e) m[u][e] = fmaf(a.beta, m[u][e], v[u][e]);
          if (c0 + 64 * u < pieces) {
            if constexpr (!kWide) mom[c0 + 64 * u] = m[u][0];
            else
#pragma unroll
              for (int e = 0; e < kE; e += 4) *(float4*)(mom + (c0 + 64 * u) * kE + e) = make_float4(m[u][e], m[u][e + 1], m[u][e + 2], m[u][e + 3]);
          }
#pragma unroll
          for (int e = 0; e < kE; ++e) v[u][e] = a.nesterov ? fmaf(a.beta, m[u][e], v[u][e]) : m[u][e];
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) s = fma((double)v[u][e], (double)v[u][e], s);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (tx == 0) red[ty] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[b * kNormParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// the matrix's sum of squares from its partials, in every lane of a wave
__device__ __forceinline__ double norm2_of(const double* __restrict__ part, int parts) {
  double s = 0.0;
  for (int q = threadIdx.x & 63; q < parts; q += 64) s += part[q];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  return s;
}

// ---- X0 in both orientations ---------------------------------------------------------------
// A workgroup takes 32 rows x 32 kInit columns of X, all its loads in flight
// together; bound by memory (G once, four planes written: six 1088 x 1088 in 21 us,
// 28 with one block of columns a workgroup).
constexpr int kInit = 4;
template <int T, bool kMuon>
__global__ __launch_bounds__(256) void ns_init_kernel(NsArgs a, NsPlan p, int parts, const double* __restrict__ part,
                                                      char* __restrict__ ws) {
  __shared__ unsigned tile[kInit][32 * 33];
  const int64_t b = blockIdx.y;
  const int nb = p.np / 32, strips = (nb + kInit - 1) / kInit;
  const int bi = blockIdx.x / strips, bj0 = (blockIdx.x - bi * strips) * kInit;  // 32-row block of X, first 32-column block
  const bool tall = a.rows > a.cols;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float v[kInit][4], m[kInit][4];
#pragma unroll
  for (int z = 0; z < kInit; ++z)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // fast index tx along the source's rows; (i, j) of X
      const int sr = ty + 8 * q;
      const int gi = bi * 32 + (tall ? tx : sr), gj = (bj0 + z) * 32 + (tall ? sr : tx);
      const bool in = gi < p.m && gj < p.n;
      const int64_t r = tall ? gj : gi, c = tall ? gi : gj;
      v[z][q] = in ? op_load<T>(a.in.p, b * a.in.batch + r * a.in.row + c) : 0.f;
      if constexpr (kMuon) m[z][q] = in ? ((const float*)a.momentum.p)[b * a.momentum.batch + r * a.momentum.row + c] : 0.f;
    }
  const double s = norm2_of(part + b * kNormParts, parts);
  const double inv = (double)kSx / fmax(sqrt(s), (double)a.eps);
  const bool bad = !(s < 1e300);  // an infinity or a NaN in the matrix: every entry becomes NaN
#pragma unroll
  for (int z = 0; z < kInit; ++z)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int sr = ty + 8 * q, i = tall ? tx : sr, j = tall ? sr : tx;
      const int gi = bi * 32 + i, gj = (bj0 + z) * 32 + j;
      float u = v[z][q];
      if constexpr (kMuon) u = a.nesterov ? fmaf(a.beta, m[z][q], u) : m[z][q];
      u = gi < p.m && gj < p.n ? bad ? __builtin_nanf("") : (float)((double)u * inv) : 0.f;
      _Float16 hi, lo;
      split(u, hi, lo);
      tile[z][i * 33 + j] = (unsigned)__builtin_bit_cast(unsigned short, hi) | ((unsigned)__builtin_bit_cast(unsigned short, lo) << 16);
    }
  __syncthreads();
  // 32 x 4 octets in either form: threads 0..127 Xr (row i, contraction j), 128..255 Xc
  const int t = threadIdx.x & 127, row = t & 31, u = t >> 5;
  const bool xc = threadIdx.x >= 128;
#pragma unroll
  for (int z = 0; z < kInit; ++z) {
    const int bj = bj0 + z;
    if (bj >= nb) break;
    unsigned short hs[8], ls[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned w = xc ? tile[z][(8 * u + e) * 33 + row] : tile[z][row * 33 + 8 * u + e];
      hs[e] = (unsigned short)w;
      ls[e] = (unsigned short)(w >> 16);
    }
    const int64_t unit = xc ? ((int64_t)bj * (p.mp / 8) + bi * 4 + u) * 32 + row : ((int64_t)bi * (p.np / 8) + bj * 4 + u) * 32 + row;
    char* x = ws + b * p.stride + p.x[0] + (xc ? 2 * p.xplane : 0);
    *(v4u*)(x + unit * 16) = *(v4u*)hs;
    *(v4u*)(x + p.xplane + unit * 16) = *(v4u*)ls;
  }
}

// one element or four aligned neighbours of a row
template <int E>
__device__ __forceinline__ void load_some(const float* p, int64_t o, float (&v)[E]) {
  if constexpr (E == 1) {
    v[0] = p[o];
  } else {
    const float4 f = *(const float4*)(p + o);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
}
template <int T, int E>
__device__ __forceinline__ void store_some(void* p, int64_t o, const float (&v)[E]) {
  if constexpr (E == 1) {
    op_store<T>(p, o, v[0]);
  } else if constexpr (T == kOpF32) {
    *(float4*)((float*)p + o) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    half4 u;  // four 16-bit values of either type
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = T == kOpF16 ? (_Float16)v[e] : __builtin_bit_cast(_Float16, (__bf16)v[e]);
    *(half4*)((_Float16*)p + o) = u;
  }
}

// ---- the three products --------------------------------------------------------------------
// kPart, kJoin: a Gram matrix of few tiles and long K in two launches, fp32 sums of
// parts of K by different workgroups, then their total
enum { kGram = 0, kSquare = 1, kUpdate = 2, kFinal = 3, kPart = 4, kJoin = 5 };

struct NsProd {
  const char* P; const char* Q;       // hi planes of matrix 0; lo planes follow at p_lo / q_lo
  int64_t p_lo, q_lo;
  int Rp, Rq, K;                      // rows (multiples of 32) of P and Q, contraction length
  int64_t stride;                     // bytes between the matrices' workspaces
  int ti, tj;                         // tiles of P and Q that are whole
  int whole, rest;                    // tiles of a matrix: whole ones, ones with a partial row block
  const char* E; int64_t e_lo;        // kSquare: A (= Q), in (row j, contraction i) form
  char* Y; int64_t y_lo;              // result in (row j, contraction i) form
  char* Z; int64_t z_lo;              // result in (row i, contraction j) form
  float* part; int slices;            // kPart, kJoin: [slice of K][tile][4 waves][16][64]
  float f, e;                         // result = f * sum (+ e * E, + a on the diagonal: kSquare), in the stored forms' scales
};

#define NS_LDS(SRC, VOFF, SOFF, DST) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(SRC, (__attribute__((address_space(3))) void*)(DST), 16, VOFF, SOFF, 0, 0)

// One tile of D = P Q^T of 64 NI x 64 NJ, four waves of 32 NI x 32 NJ; K in steps of
// 16 (64 x 64: 32) through a ring of four LDS buffers filled by LDS-DMA (16 KB a
// stage, 12 KB for 128 x 64: hi and lo of both operands), three to four stages in
// flight (eight buffers measured the same, two 20 us for 12 where CUs are idle):
// with one stage in flight a lone workgroup of a CU spent three quarters of its
// time waiting for the next (46 us for six 1088 x 1088 Gram matrices).  The
// buffers are LDS objects of their own, and a stage's object is known at compile
// time, so the compiler adds no waits of its own for loads into the others.
template <int MODE, int T, int NI, int NJ>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void ns_prod_kernel(NsProd g, NsArgs a, NsPlan pl) {
  constexpr int KK = 2 / NI, TI = 2 * NI, TJ = 2 * NJ;  // 16-wide pieces of K a stage, row blocks of a tile's sides
  constexpr int kP = TI * KK * 1024, kQ = TJ * KK * 1024, kStage = 2 * (kP + kQ);  // bytes of a plane's part of a stage
  constexpr int R = 4, L = kStage / 4096;  // ring buffers, loads of a wave per stage
  __shared__ __attribute__((aligned(16))) char l0[kStage], l1[kStage], l2[kStage], l3[kStage];
#define NS_BUF(I) ((I) % R == 0 ? l0 : (I) % R == 1 ? l1 : (I) % R == 2 ? l2 : l3)
  // The whole tiles of all matrices come first, then those with fewer row blocks
  // of either operand.
  const int nwhole = g.whole * (int)a.batch, ntiles = MODE == kPart ? gridDim.x / g.slices : gridDim.x;
  const int slice = MODE == kPart ? blockIdx.x / ntiles : 0, block = MODE == kPart ? blockIdx.x % ntiles : blockIdx.x;
  const bool rest = block >= nwhole;
  const int id = rest ? xcd_remap(block - nwhole, ntiles - nwhole) : xcd_remap(block, nwhole);
  const int mat = id / (rest ? g.rest : g.whole);
  int t = id - mat * (rest ? g.rest : g.whole);
  int ti, tj;
  if constexpr (NI != NJ) {
    // symmetric: pairs of 64-row blocks ti with the columns up to theirs, then, if
    // the number of blocks is odd, all rows with the last block's columns
    if (rest) {
      ti = t;
      tj = 2 * g.ti;
    } else {
      ti = (int)((sqrtf(4.f * t + 1.f) - 1.f) * 0.5f);
      while (ti * (ti + 1) > t) --ti;
      while ((ti + 1) * (ti + 2) <= t) ++ti;
      tj = t - ti * (ti + 1);
    }
  } else if constexpr (MODE != kUpdate && MODE != kFinal) {  // lower triangle, ti >= tj, row after row
    if (rest) t += g.whole;
    ti = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
  } else if (!rest) {
    ti = t % g.ti;
    tj = t / g.ti;
  } else {  // the last column of tiles, if partial, then the last row
    const int side = g.Rq / 32 > g.tj * TJ ? g.ti : 0;
    ti = t < side ? t : g.ti;
    tj = t < side ? g.tj : t - side;
  }
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = w >> 1, wj = w & 1, h = lane >> 5, l31 = lane & 31;
  const char* Pm = g.P + mat * g.stride;
  const char* Qm = g.Q + mat * g.stride;
  const int nPb = g.Rp / 32, nQb = g.Rq / 32;
  // this wave stages one row block (64 x 64: one 16-wide piece of it) of both operand
  // tiles (128 x 64: of one half of Q's; a block past the end repeats the last one,
  // its results are not stored)
  const int sb = NI == 2 ? w : w >> 1, sk = NI == 2 ? 0 : (w & 1) * 1024;
  const int rb_bytes = g.K * 64;
  const int pb = min(ti * TI + sb, nPb - 1), qb = min(tj * TJ + (NI == NJ ? sb : w & 1), nQb - 1);
  const __amdgpu_buffer_rsrc_t rph = __builtin_amdgcn_make_buffer_rsrc((void*)(Pm + (int64_t)pb * rb_bytes), 0, rb_bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t rpl = __builtin_amdgcn_make_buffer_rsrc((void*)(Pm + g.p_lo + (int64_t)pb * rb_bytes), 0, rb_bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t rqh = __builtin_amdgcn_make_buffer_rsrc((void*)(Qm + (NI != NJ && w >= 2 ? g.q_lo : 0) + (int64_t)qb * rb_bytes), 0, rb_bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t rql = __builtin_amdgcn_make_buffer_rsrc((void*)(Qm + g.q_lo + (int64_t)qb * rb_bytes), 0, rb_bytes, 0x00020000);
  const int vo = lane * 16;
  // stage layout: P hi | P lo | Q hi | Q lo, row blocks x 1 KB pieces of K
  const int all = g.K / (16 * KK), share = MODE == kPart ? (all + g.slices - 1) / g.slices : all;
  const int first = slice * share, nk = MODE == kJoin ? 0 : min(share, all - first);  // this workgroup's stages
  auto stage = [&](int ks, char* buf) {
    char* d = buf + w * 1024;
    const int so = (first + ks) * (1024 * KK) + sk;
    NS_LDS(rph, vo, so, d);
    NS_LDS(rpl, vo, so, d + kP);
    NS_LDS(rqh, vo, so, d + 2 * kP);
    if constexpr (NI == NJ) NS_LDS(rql, vo, so, d + 2 * kP + kQ);
  };
  f32x16 acc[NI][NJ] = {}, cr = {};  // cr: 64 x 64 alternates between two sums, which do not wait for each other
  struct Frag { half8 ph[NI * KK], pl[NI * KK], qh[NJ * KK], ql[NJ * KK]; };  // [row block][piece of K]
  auto fetch = [&](const char* buf, Frag& f) {
    const char *p = buf + wi * NI * KK * 1024 + vo, *q = buf + 2 * kP + wj * NJ * KK * 1024 + vo;
#pragma unroll
    for (int x = 0; x < NI * KK; ++x) f.ph[x] = *(const half8*)(p + x * 1024);
#pragma unroll
    for (int x = 0; x < NJ * KK; ++x) f.qh[x] = *(const half8*)(q + x * 1024);
#pragma unroll
    for (int x = 0; x < NJ * KK; ++x) f.ql[x] = *(const half8*)(q + kQ + x * 1024);
#pragma unroll
    for (int x = 0; x < NI * KK; ++x) f.pl[x] = *(const half8*)(p + kP + x * 1024);
  };
#define NS_MFMA(A, B, C) __builtin_amdgcn_mfma_f32_32x32x16_f16(A, B, C, 0, 0, 0)
  auto multiply = [&](const Frag& f) {
    if constexpr (NI == 1) {
      acc[0][0] = NS_MFMA(f.ph[0], f.qh[0], acc[0][0]);
      cr = NS_MFMA(f.ph[0], f.ql[0], cr);
      acc[0][0] = NS_MFMA(f.pl[0], f.qh[0], acc[0][0]);
      cr = NS_MFMA(f.ph[1], f.qh[1], cr);
      acc[0][0] = NS_MFMA(f.ph[1], f.ql[1], acc[0][0]);
      cr = NS_MFMA(f.pl[1], f.qh[1], cr);
    } else {
#pragma unroll
      for (int x = 0; x < NI; ++x)
#pragma unroll
        for (int y = 0; y < NJ; ++y) acc[x][y] = NS_MFMA(f.ph[x], f.qh[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < NI; ++x)
#pragma unroll
        for (int y = 0; y < NJ; ++y) acc[x][y] = NS_MFMA(f.ph[x], f.ql[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < NI; ++x)
#pragma unroll
        for (int y = 0; y < NJ; ++y) acc[x][y] = NS_MFMA(f.pl[x], f.qh[y], acc[x][y]);
    }
  };
  // Step s multiplies stage s, whose fragments are in `cur`, and reads those of
  // stage s + 1 meanwhile.  Past the barrier stage s + 1 has landed for every
  // wave, and every wave holds stage s in registers: its buffer takes stage
  // s + R.  (Without the fetch ahead a lone workgroup of a CU waits for its LDS
  // reads before each stage's products.)
  auto step = [&](int s, char* mine, const char* after, Frag& cur, Frag& next, bool more, bool load) {
    if (more) {
      if (load) stage_barrier<(R - 2) * L>();
      else stage_barrier<0>();
      if (load) stage(s + R, mine);
      fetch(after, next);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(cur);
  };
  Frag f[2];
  int ks = 0;
  if (nk >= 2 * R) {  // (a block of its own: the compiler then knows how many loads are outstanding in the loop)
#pragma unroll
    for (int i = 0; i < R; ++i) stage(i, NS_BUF(i));
    stage_barrier<(R - 1) * L>();
    fetch(l0, f[0]);
    do {  // every step has a stage left to load
#pragma unroll
      for (int i = 0; i < R; ++i) step(ks + i, NS_BUF(i), NS_BUF(i + 1), f[i & 1], f[(i + 1) & 1], true, true);
      ks += R;
    } while (ks + 2 * R <= nk);
  } else if (MODE != kJoin) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < nk) stage(i, NS_BUF(i));
    stage_barrier<0>();
    fetch(l0, f[0]);
  }
  for (; ks < nk; ks += R) {  // at most 2 R - 1 stages remain
    const int left = nk - ks;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (left > i) step(ks + i, NS_BUF(i), NS_BUF(i + 1), f[i & 1], f[(i + 1) & 1], left > i + 1, left > R + i);
  }
#undef NS_BUF
  if constexpr (NI == 1) acc[0][0] += cr;
  if constexpr (MODE == kPart || MODE == kJoin) {
    const int64_t tile = (int64_t)mat * (g.whole + g.rest) + t, tiles = (int64_t)(g.whole + g.rest) * a.batch;
    float* sums = g.part + (tile * 4 + w) * 1024 + lane;
    if constexpr (MODE == kPart) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sums[slice * tiles * 4096 + e * 64] = acc[0][0][e];
      return;
    }
    constexpr int kAhead = 4;
    for (int q0 = 0; q0 < g.slices; q0 += kAhead) {  // in their order
      float v[kAhead][16];
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) v[q][e] = q0 + q < g.slices ? sums[(q0 + q) * tiles * 4096 + e * 64] : 0.f;
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[0][0][e] += v[q][e];
    }
  }
  __syncthreads();
  // epilogue, one 32 x 32 block at a time; the wave transposes in a ring buffer of its own
  unsigned* tr = (unsigned*)(w == 0 ? l0 : w == 1 ? l1 : w == 2 ? l2 : l3);
  const float lr = MODE == kFinal && a.momentum.p ? (a.lr_dev ? *a.lr_dev : a.lr) : 0.f;
  const int out_bytes = a.momentum.p || T == kOpF32 ? 16 : 8;  // of four neighbours
  const bool wide = MODE == kFinal && ((uintptr_t)a.out.p % out_bytes | a.cols % 4 | a.out.row % 4 | (a.batch > 1 ? a.out.batch % 4 : 0)) == 0;
#pragma unroll
  for (int x = 0; x < NI; ++x)
#pragma unroll
    for (int y = 0; y < NJ; ++y) {
      const int rbi = ti * TI + wi * NI + x, rbj = tj * TJ + wj * NJ + y;
      if (rbi >= nPb || rbj >= nQb) continue;
      // (128 x 64: a block above the diagonal belongs to the tile that holds its mirror)
      if (NI != NJ && !rest && rbj / 2 > rbi / 2) continue;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[x][y][e] * g.f;
      // (row j, contraction i): octet 4 rbi + q of row block rbj, row l31, halves 4h .. 4h + 3
      const int64_t at = (((int64_t)rbj * (g.Rp / 8) + rbi * 4) * 32 + l31) * 16 + h * 8;
      if constexpr (MODE == kSquare) {
        const char* E = g.E + mat * g.stride + at;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const half4 eh = *(const half4*)(E + q * 512), el = *(const half4*)(E + g.e_lo + q * 512);
#pragma unroll
          for (int s2 = 0; s2 < 4; ++s2) v[4 * q + s2] = fmaf((float)eh[s2] + (float)el[s2], g.e, v[4 * q + s2]);
        }
        if (rbi == rbj)
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] += 8 * (e >> 2) + 4 * h + (e & 3) == l31 ? a.a * kSb : 0.f;
      }
      if constexpr (MODE == kFinal) {
        // through LDS, so that a wave's lanes follow the output's rows: four elements
        // a lane where they are aligned, else one (parameters: all loads before the
        // first store)
        const bool tall = a.rows > a.cols;
        float* block = (float*)tr;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = 8 * (e >> 2) + 4 * h + (e & 3);
          block[tall ? l31 * 33 + i : i * 33 + l31] = v[e];
        }
        __builtin_amdgcn_wave_barrier();
        auto write = [&](auto four) {
          constexpr int E = decltype(four)::value ? 4 : 1, kQ = 16 / E, kRow = 32 / E;  // pieces of E, kRow lanes a row
          const int lr0 = lane / kRow, lc = lane % kRow * E;
          const int r0 = 32 * (tall ? rbj : rbi) + lr0, c0 = 32 * (tall ? rbi : rbj) + lc;  // of the output
          if (c0 >= a.cols) return;
          float D[kQ][E], W[kQ][E];
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const int r = r0 + 64 / kRow * q;
            if (a.momentum.p && r < a.rows) load_some((const float*)a.out.p, (int64_t)mat * a.out.batch + (int64_t)r * a.out.row + c0, W[q]);
#pragma unroll
            for (int e = 0; e < E; ++e) D[q][e] = block[(lr0 + 64 / kRow * q) * 33 + lc + e];
          }
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const int r = r0 + 64 / kRow * q;
            if (r >= a.rows) continue;
            const int64_t o = (int64_t)mat * a.out.batch + (int64_t)r * a.out.row + c0;
            if (a.momentum.p) {
#pragma unroll
              for (int e = 0; e < E; ++e) D[q][e] = fmaf(-lr * a.scale, D[q][e], W[q][e] * (1.f - lr * a.decay));
              store_some<kOpF32>(a.out.p, o, D[q]);
            } else {
              store_some<T>(a.out.p, o, D[q]);
            }
          }
        };
        if (wide) write(std::true_type{});
        else write(std::false_type{});
        __builtin_amdgcn_wave_barrier();
      } else {
        char* Y = g.Y + mat * g.stride + at;
        unsigned word[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          half4 hv, lv;
#pragma unroll
          for (int s2 = 0; s2 < 4; ++s2) {
            _Float16 hi, lo;
            split(v[4 * q + s2], hi, lo);
            hv[s2] = hi;
            lv[s2] = lo;
            word[4 * q + s2] = (unsigned)__builtin_bit_cast(unsigned short, hi) | ((unsigned)__builtin_bit_cast(unsigned short, lo) << 16);
          }
          *(half4*)(Y + q * 512) = hv;
          *(half4*)(Y + g.y_lo + q * 512) = lv;
        }
        if (MODE == kUpdate || rbi / TJ != rbj / TJ) {  // the other form: (row i, contraction j)
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int e = 0; e < 16; ++e) tr[(8 * (e >> 2) + 4 * h + (e & 3)) * 33 + l31] = word[e];
          __builtin_amdgcn_wave_barrier();
          char* Z = g.Z + mat * g.stride + (((int64_t)rbi * (g.Rq / 8) + rbj * 4) * 32 + l31) * 16;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            unsigned short hs[8], ls[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const unsigned wd = tr[l31 * 33 + 8 * (2 * u + h) + e];
              hs[e] = (unsigned short)wd;
              ls[e] = (unsigned short)(wd >> 16);
            }
            *(v4u*)(Z + (2 * u + h) * 512) = *(v4u*)hs;
            *(v4u*)(Z + g.z_lo + (2 * u + h) * 512) = *(v4u*)ls;
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
}

// ---- matrices with a short side of at most 64 ----------------------------------------------
// The short side's Gram matrix fits into LDS, so a workgroup does a whole step
// for its own columns of X: A (from all workgroups' partial sums), B = a I + b A +
// c A A (every workgroup for itself), X <- B X, and the next Gram matrix's partial
// sum.  A step is one launch instead of three, and a matrix of few columns is
// one launch in all.  X is held as chunks of W columns, each an LDS image of Xc
// and Xr; a workgroup (slab) takes chunks slab, slab + S, ...
// Bound by latency (barriers, LDS round trips, cold code), so the work is spread
// over NW waves in blocks of 16 x 16 (v_mfma_f32_16x16x32_f16: a lane supplies
// row l % 16, k = 8 (l / 16) .. + 7 of either operand, which the planes' octets
// hold, and receives four consecutive i of one j).
enum { kSolo = 0, kFirst = 1, kMid = 2, kLast = 3 };

struct ThinPlan {
  int m, n, chunks, slabs;
  int64_t grams, images, stride;  // per matrix: offsets of the partial sums (two sets) and the images; bytes
};
template <int MB, int WB, int NW>
struct ThinGeo {
  static constexpr int M = 32 * MB, W = 32 * WB;
  static constexpr int kA = M * M * 2, kX = M * W * 2;     // bytes of a plane of A / B and of X
  static constexpr int kImage = 4 * kX;                    // Xc hi, Xc lo, Xr hi, Xr lo
  static constexpr int kLds = kImage + 2 * kA;
  static constexpr int kGram = M * M * 4;                  // bytes of a partial Gram matrix
  static constexpr int kThreads = 64 * NW;
  static constexpr int MT = M / 16, WT = W / 16;           // blocks along the sides
  static constexpr int GB = MT * MT / NW, XB = MT * WT / NW;  // blocks a wave holds
  static_assert(MT * MT % NW == 0 && MT * WT % NW == 0 && M * W % kThreads == 0 && kImage / 2 % (16 * kThreads) == 0, "");
};
template <int MB, int WB, int NW>
ThinPlan make_thin(int64_t batch, int64_t rows, int64_t cols) {
  using G = ThinGeo<MB, WB, NW>;
  ThinPlan p;
  p.m = (int)std::min(rows, cols);
  p.n = (int)std::max(rows, cols);
  p.chunks = (p.n + G::W - 1) / G::W;
  // Slabs of a matrix, equal shares: the more, the fewer chunks each, but each reads
  // all partial sums of a step and squares them (about a chunk's time), and past a
  // workgroup a CU (M 32: two, of four waves) they take turns.  Measured: 14 x 48 x
  // 4253 (34 chunks) 34 / 17 slabs 174 / 130 us; 54 x 57 x 2789 (22) 22 / 8 / 6 / 4:
  // 363 / 258 / 262 / 225; 132 x 54 x 1902 (15) 15 / 3 / 2 / 1: 515 / 300 / 385 / 363;
  // one 64 x 7000 (55) 28 / 19: 77 / 85; M 32: 72 x 29 x 3946 (31) 11 / 8 / 7: 228 /
  // 223 / 216, 51 x 21 x 2150 (17) 17 / 9: 111 / 99.
  float best = 1e30f;
  for (int each = 1; each <= p.chunks; each = each < 32 || each == p.chunks ? each + 1 : p.chunks) {
    const int slabs = (p.chunks + each - 1) / each;
    const float wgs = (float)slabs * batch;
    const float cost = (MB == 1 ? std::max(1.f, wgs / 512) : std::ceil(wgs / 256)) * (each + 0.08f * slabs + 1);
    if (slabs <= 48 && cost < best) {
      best = cost;
      p.slabs = slabs;
    }
  }
  p.grams = 0;
  p.images = 2 * (int64_t)p.slabs * G::kGram;
  p.stride = p.chunks == 1 ? 0 : p.images + (int64_t)p.chunks * G::kImage;
  return p;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// D += P Q^T for one 16 x 16 block: rows 16 rp .. of plane pair P, 16 rq .. of Q,
// contraction length K; both in LDS with their lo plane behind by p_lo / q_lo
// (three sums that do not wait for each other: hi hi, hi lo, lo hi)
template <int K>
__device__ __forceinline__ void lds_product(const char* P, int p_lo, int rp, const char* Q, int q_lo, int rq, int lane, f32x4& acc) {
  f32x4 cr = {}, cs = {};
  const int at = (lane >> 4) * 512 + (lane & 15) * 16;
  const char* p = P + (rp >> 1) * (K * 64) + (rp & 1) * 256 + at;
  const char* q = Q + (rq >> 1) * (K * 64) + (rq & 1) * 256 + at;
#pragma unroll
  for (int kk = 0; kk < K / 32; ++kk) {
    const half8 ph = *(const half8*)(p + kk * 2048), pl = *(const half8*)(p + p_lo + kk * 2048);
    const half8 qh = *(const half8*)(q + kk * 2048), ql = *(const half8*)(q + q_lo + kk * 2048);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
    cr = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, cr, 0, 0, 0);
    cs = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, cs, 0, 0, 0);
  }
  acc += cr + cs;
}

template <int MB, int WB, int NW, int T, bool kMuon, int MODE>
__global__ __launch_bounds__(64 * NW) void ns_thin_kernel(NsArgs a, ThinPlan p, int parts, const double* __restrict__ part,
                                                          char* __restrict__ ws, int set) {
  using G = ThinGeo<MB, WB, NW>;
  constexpr int M = G::M, W = G::W, kThreads = G::kThreads;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *sc = lds, *sr = lds + 2 * G::kX, *sa = lds + G::kImage;
  __shared__ double red[NW];
  const int64_t b = blockIdx.y;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, l4 = lane >> 4;
  const bool tall = a.rows > a.cols;
  char* mine = ws + b * p.stride;

  // This thread's elements of chunk `ch` of the source (the gradient, or muon's
  // update direction), element e of the chunk at kThreads k + thread; zero outside
  // the matrix.  All loads are in flight together.
  constexpr int kMine = M * W / kThreads;
  auto place = [&](int k, int& i, int& j) {
    const int e = kThreads * k + threadIdx.x;
    i = tall ? e % M : e / W;
    j = tall ? e / M : e % W;
  };
  auto load_source = [&](int ch, float (&v)[kMine]) {
    float mo[kMuon ? kMine : 1];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      int i, j;
      place(k, i, j);
      const bool in = i < p.m && ch * W + j < p.n;
      const int64_t r = tall ? ch * W + j : i, c = tall ? i : ch * W + j;
      v[k] = in ? op_load<T>(a.in.p, b * a.in.batch + r * a.in.row + c) : 0.f;
      if constexpr (kMuon) mo[k] = in ? ((const float*)a.momentum.p)[b * a.momentum.batch + r * a.momentum.row + c] : 0.f;
    }
    if constexpr (kMuon) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        if constexpr (MODE == kSolo) {  // (elsewhere the norm's launch updated the momentum)
          int i, j;
          place(k, i, j);
          mo[k] = fmaf(a.beta, mo[k], v[k]);
          if (i < p.m && j < p.n)
            ((float*)a.momentum.p)[b * a.momentum.batch + (int64_t)(tall ? j : i) * a.momentum.row + (tall ? i : j)] = mo[k];
        }
        v[k] = a.nesterov ? fmaf(a.beta, mo[k], v[k]) : mo[k];
      }
    }
  };
  // byte offset of element (row, k) in a plane of contraction length K
  auto half_at = [](int row, int k, int K) { return ((((row >> 5) * (K / 8) + (k >> 3)) * 32 + (row & 31)) * 8 + (k & 7)) * 2; };
  // X0 from the source into both LDS forms
  auto put_source = [&](const float (&v)[kMine], double norm2) {
    const double inv = (double)kSx / fmax(sqrt(norm2), (double)a.eps);
    const bool bad = !(norm2 < 1e300);
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      int i, j;
      place(k, i, j);
      _Float16 hi, lo;
      split(bad ? __builtin_nanf("") : (float)((double)v[k] * inv), hi, lo);
      char *c = sc + half_at(j, i, M), *r = sr + half_at(i, j, W);
      *(_Float16*)c = hi;
      *(_Float16*)(c + G::kX) = lo;
      *(_Float16*)r = hi;
      *(_Float16*)(r + G::kX) = lo;
    }
  };
  // one block (block row bi, block column bj) in (row j, contraction i) form into plane pair `to`
  auto put = [&](char* to, int lo_at, int bj, int bi, f32x4 v) {
    half4 hv, lv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      _Float16 hi, lo;
      split(v[e], hi, lo);
      hv[e] = hi;
      lv[e] = lo;
    }
    char* y = to + half_at(16 * bj + l15, 16 * bi + 4 * l4, M);
    *(half4*)y = hv;
    *(half4*)(y + lo_at) = lv;
  };
  // this wave's blocks of X X^T of the chunk in LDS, added to g
  auto gram = [&](f32x4 (&g)[G::GB]) {
#pragma unroll
    for (int k = 0; k < G::GB; ++k) {
      const int t = w + NW * k;
      lds_product<W>(sr, G::kX, t % G::MT, sr, G::kX, t / G::MT, lane, g[k]);
    }
  };
  // A (scaled sums g) into sa, then B = a I + b A + c A A in its place
  auto square = [&](f32x4 (&g)[G::GB]) {
#pragma unroll
    for (int k = 0; k < G::GB; ++k) {
      const int t = w + NW * k;
      g[k] *= kSa / (kSx * kSx);
      put(sa, G::kA, t / G::MT, t % G::MT, g[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < G::GB; ++k) {
      const int t = w + NW * k, bi = t % G::MT, bj = t / G::MT;
      f32x4 acc = {};
      lds_product<M>(sa, G::kA, bi, sa, G::kA, bj, lane, acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[k][e] = fmaf(acc[e], a.c * kSb / (kSa * kSa), g[k][e] * (a.b * kSb / kSa));
        if (bi == bj && 4 * l4 + e == l15) g[k][e] += a.a * kSb;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < G::GB; ++k) {
      const int t = w + NW * k;
      put(sa, G::kA, t / G::MT, t % G::MT, g[k]);
    }
    __syncthreads();
  };
  // X <- B X for the chunk in LDS; the last step writes the result
  auto update = [&](int ch, bool last) {
    f32x4 v[G::XB];
    const float sy = last ? 1.f : kSx;
#pragma unroll
    for (int k = 0; k < G::XB; ++k) {
      const int t = w + NW * k;
      v[k] = f32x4{};
      lds_product<M>(sa, G::kA, t % G::MT, sc, G::kX, t / G::MT, lane, v[k]);
      v[k] *= sy / (kSb * kSx);
    }
    if (last) {
      const float lr = kMuon ? (a.lr_dev ? *a.lr_dev : a.lr) : 0.f;
#pragma unroll
      for (int k = 0; k < G::XB; ++k) {
        const int t = w + NW * k, i0 = 16 * (t % G::MT) + 4 * l4, j = ch * W + 16 * (t / G::MT) + l15;
        if (j >= p.n) continue;
        const int64_t o0 = b * a.out.batch + (tall ? (int64_t)j * a.out.row + i0 : (int64_t)i0 * a.out.row + j), step = tall ? 1 : a.out.row;
        float W[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (kMuon && i0 + e < p.m) W[e] = ((const float*)a.out.p)[o0 + e * step];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i0 + e >= p.m) continue;
          if constexpr (kMuon) ((float*)a.out.p)[o0 + e * step] = fmaf(-lr * a.scale, v[k][e], W[e] * (1.f - lr * a.decay));
          else op_store<T>(a.out.p, o0 + e * step, v[k][e]);
        }
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < G::XB; ++k) {
      const int t = w + NW * k, bi = t % G::MT, bj = t / G::MT;
      put(sc, G::kX, bj, bi, v[k]);
      // the (row i, contraction j) form, a half at a time
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        _Float16 hi, lo;
        split(v[k][e], hi, lo);
        char* r = sr + half_at(16 * bi + 4 * l4 + e, 16 * bj + l15, W);
        *(_Float16*)r = hi;
        *(_Float16*)(r + G::kX) = lo;
      }
    }
    __syncthreads();
  };

  f32x4 g[G::GB] = {};
  if constexpr (MODE == kSolo) {
    float v[kMine];
    load_source(0, v);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kMine; ++k) s = fma((double)v[k], (double)v[k], s);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) red[w] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int q = 1; q < NW; ++q) s += red[q];
    put_source(v, s);
    __syncthreads();
    for (int k = 0; k < a.steps; ++k) {
#pragma unroll
      for (int q = 0; q < G::GB; ++q) g[q] = f32x4{};
      gram(g);
      square(g);
      update(0, k + 1 == a.steps);
    }
    return;
  }

  const int slab = blockIdx.x;
  float* gin = (float*)(mine + p.grams + (int64_t)set * p.slabs * G::kGram);
  float* gout = (float*)(mine + p.grams + (int64_t)(set ^ 1) * p.slabs * G::kGram) + (int64_t)slab * (G::kGram / 4);
  // a chunk's image into LDS, by LDS-DMA (the last step reads Xc only)
  constexpr int kBytes = MODE == kLast ? G::kImage / 2 : G::kImage;
  auto load_image = [&](int ch) {
    const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc((void*)(mine + p.images + (int64_t)ch * G::kImage), 0, kBytes, 0x00020000);
#pragma unroll
    for (int e = 0; e < kBytes; e += 16 * kThreads) NS_LDS(res, lane * 16, e + w * 1024, lds + e + w * 1024);
  };
  if constexpr (MODE != kFirst) {
    load_image(slab);  // meanwhile: A from the slabs' partial sums, in slab order
#pragma unroll
    for (int k = 0; k < G::GB; ++k) {
      const f32x4* src = (const f32x4*)gin + (w + NW * k) * 64 + lane;
      constexpr int kAhead = 12, kPitch = G::kGram / 16;  // sums in flight
      for (int q0 = 0; q0 < p.slabs; q0 += kAhead) {
        f32x4 f[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) f[q] = q0 + q < p.slabs ? src[(int64_t)(q0 + q) * kPitch] : f32x4{};
#pragma unroll
        for (int q = 0; q < kAhead; ++q) g[k] += f[q];
      }
    }
    square(g);
#pragma unroll
    for (int q = 0; q < G::GB; ++q) g[q] = f32x4{};
  }
  const double norm2 = MODE == kFirst ? norm2_of(part + b * kNormParts, parts) : 0.0;
  for (int ch = slab; ch < p.chunks; ch += p.slabs) {
    char* image = mine + p.images + (int64_t)ch * G::kImage;
    if (ch != slab) {
      __syncthreads();  // the chunk before is done with
      if constexpr (MODE != kFirst) load_image(ch);
    }
    if constexpr (MODE == kFirst) {
      float v[kMine];
      load_source(ch, v);
      put_source(v, norm2);
    }
    __syncthreads();
    if constexpr (MODE != kFirst) update(ch, MODE == kLast);
    if constexpr (MODE != kLast) {
      gram(g);
#pragma unroll
      for (int e = threadIdx.x; e < G::kImage / 16; e += kThreads) ((v4u*)image)[e] = ((const v4u*)lds)[e];
    }
  }
  if constexpr (MODE != kLast) {
#pragma unroll
    for (int k = 0; k < G::GB; ++k) ((f32x4*)gout)[(w + NW * k) * 64 + lane] = g[k];
  }
}

template <int T, bool kMuon>
void launch_norm(const NsArgs& a, int parts, double* part, hipStream_t s) {
  constexpr int kE = T == kOpF32 ? 4 : 8;
  bool wide = ((uintptr_t)a.in.p % 16 | a.cols % kE | a.in.row % kE | (a.batch > 1 ? a.in.batch % kE : 0)) == 0;
  if (kMuon) wide = wide && ((uintptr_t)a.momentum.p % 16 | a.momentum.row % 4 | (a.batch > 1 ? a.momentum.batch % 4 : 0)) == 0;
  const dim3 grid(parts, (unsigned)a.batch);
  if (wide) hipLaunchKernelGGL((ns_norm_kernel<T, kMuon, true>), grid, dim3(256), 0, s, a, part);
  else hipLaunchKernelGGL((ns_norm_kernel<T, kMuon, false>), grid, dim3(256), 0, s, a, part);
}
// workgroups of the norm for a matrix: four rows at a time each, ~1 000 in all
int norm_parts(const NsArgs& a) {
  return std::max(1, std::min({kNormParts, (a.rows + 3) / 4, (int)std::max<int64_t>(1, 1024 / a.batch)}));
}

template <int MB, int WB, int NW, int T, bool kMuon>
void launch_thin(const NsArgs& a, void* workspace, hipStream_t s) {
  using G = ThinGeo<MB, WB, NW>;
  const ThinPlan p = make_thin<MB, WB, NW>(a.batch, a.rows, a.cols);
  double* part = (double*)workspace;
  char* ws = (char*)workspace + a.batch * kNormParts * 8;
  if (p.chunks == 1) {
    hipLaunchKernelGGL((ns_thin_kernel<MB, WB, NW, T, kMuon, kSolo>), dim3(1, (unsigned)a.batch), dim3(G::kThreads), G::kLds, s, a, p, 0, part, ws, 0);
    return;
  }
  if constexpr (G::W > 64) {  // (of 64 columns at most there is one chunk)
    const dim3 grid(p.slabs, (unsigned)a.batch);
    const int parts = norm_parts(a);
    launch_norm<T, kMuon>(a, parts, part, s);
    hipLaunchKernelGGL((ns_thin_kernel<MB, WB, NW, T, kMuon, kFirst>), grid, dim3(G::kThreads), G::kLds, s, a, p, parts, part, ws, 1);
    int set = 0;
    for (int k = 0; k + 1 < a.steps; ++k, set ^= 1)
      hipLaunchKernelGGL((ns_thin_kernel<MB, WB, NW, T, kMuon, kMid>), grid, dim3(G::kThreads), G::kLds, s, a, p, parts, part, ws, set);
    hipLaunchKernelGGL((ns_thin_kernel<MB, WB, NW, T, kMuon, kLast>), grid, dim3(G::kThreads), G::kLds, s, a, p, parts, part, ws, set);
  }
}

// The path of a matrix by its sides: short side at most 64 in one launch where the
// long side is at most 64 too, else in chunks of 128 columns, with a Gram matrix of
// 32 x 32 or 64 x 64; larger ones in tiles.  Measured, M 32 / 64: one 20 x 1088 33 /
// 43 us, 58 x 30 x 528 54 / 77; a Gram matrix of 128 x 128 in LDS / tiles: one 128 x
// 1000 108 / 100 us, 96 x 71 x 846 261 / 230.  Waves, measured with 4 / 8 / 16:
// 175 x 64 x 64 20 / 15 / 15 us (4 000 of them 176 / 156 / 180), a step of 51 x 1088
// 10.4 / 7.8 / 7.2.
enum { kThinSmall, kThin32, kThin64, kTiled };
constexpr int kWavesSmall = 8, kWaves32 = 4, kWaves64 = 16;
int path_of(int64_t rows, int64_t cols) {
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  if (n <= 64) return kThinSmall;
  return m <= 32 ? kThin32 : m <= 64 ? kThin64 : kTiled;
}

// Tiles of 128 x 128, 128 x 64 (symmetric products) or 64 x 64.  A launch lasts as
// long as its fullest CU; smaller tiles spread more evenly and read more of their
// operands from LDS for a product.  Measured with 128 x 128 / 128 x 64 / 64 x 64:
// six 1088 Gram matrices (270 / 486 / 918 tiles) 42 / 32 / 35 us, one (45 / 81 /
// 153) 24 / 16 / 11; five steps of 2048 x 8192 (136 / 272 / 528) 2063 / 1994 /
// 2131 us, of 4352 x 4352 (595 / 1190 / 2346) 4812 / 4791 / 6145, of twelve 1000 x
// 1000 (432 / 864 / 1632) 939 / 980 / 1020 (4352 on another card 4750 / 4965).  The
// update X <- B X, 128 x 128 / 64 x 64: six 1088 (486 / 1734) 54 / 62 us, one (81 /
// 289) 26 / 16, one 2000 54 / 76.
// The rules compare rounds (256 tiles each) times what a round of a tile size takes.
// The times of a round are fitted to these measurements, in units of their own:
// symmetric products, 128 x 64 : 128 x 128 as 13 : 21, a single round of the latter 27
// (nothing runs under its first loads and last stores); the update, 64 x 64 : 128 x
// 128 as 13 : 40 (8.9 : 27 us for six 1088).
template <int MODE, int T>
void launch_prod(NsProd g, const NsArgs& a, const NsPlan& p, hipStream_t s) {
  constexpr bool kSym = MODE == kGram || MODE == kSquare;
  auto tiles = [&](int side) {  // whole tiles, and one more a side where a partial one follows
    const int tm = g.Rp / side, tn = g.Rq / side, pm = g.Rp % side != 0, pn = g.Rq % side != 0;
    g.ti = tm;
    g.tj = tn;
    if (kSym) {
      g.whole = tm * (tm + 1) / 2;
      g.rest = pm * (tm + 1);
    } else {
      g.whole = tm * tn;
      g.rest = (tm + pm) * (tn + pn) - tm * tn;
    }
    return (g.whole + g.rest) * a.batch;
  };
  auto pairs = [&]() {
    const int c = (g.Rp + 63) / 64;
    g.ti = c / 2;
    g.whole = g.ti * (g.ti + 1);
    g.rest = c % 2 * (g.ti + 1);
    return (g.whole + g.rest) * a.batch;
  };
  auto rounds = [](int64_t n) { return (n + 255) / 256; };
  if constexpr (kSym) {
    if (tiles(64) > 384) {
      const int64_t n = tiles(128), np = pairs();
      if (13 * rounds(np) <= (n <= 256 ? 27 : 21 * rounds(n))) {
        hipLaunchKernelGGL((ns_prod_kernel<MODE, T, 2, 1>), dim3((unsigned)np), dim3(256), 0, s, g, a, p);
        return;
      }
    }
  }
  const int64_t n64 = tiles(64), n = tiles(128);
  if (kSym ? n64 <= 384 : 13 * rounds(n64) < 40 * rounds(n)) {
    tiles(64);
    hipLaunchKernelGGL((ns_prod_kernel<MODE, T, 1, 1>), dim3((unsigned)n64), dim3(256), 0, s, g, a, p);
  } else {
    hipLaunchKernelGGL((ns_prod_kernel<MODE, T, 2, 2>), dim3((unsigned)n), dim3(256), 0, s, g, a, p);
  }
}

template <int T, bool kMuon>
void launch_ns_t(const NsArgs& a, void* workspace, hipStream_t s) {
  switch (path_of(a.rows, a.cols)) {
    case kThinSmall: return launch_thin<2, 2, kWavesSmall, T, kMuon>(a, workspace, s);
    case kThin32: return launch_thin<1, 4, kWaves32, T, kMuon>(a, workspace, s);
    case kThin64: return launch_thin<2, 4, kWaves64, T, kMuon>(a, workspace, s);
  }
  const NsPlan p = make_plan(a.batch, a.rows, a.cols);
  double* part = (double*)workspace;
  char* ws = (char*)workspace + a.batch * kNormParts * 8;
  float* parts_at = (float*)(ws + a.batch * p.stride);
  const int parts = norm_parts(a);
  launch_norm<T, kMuon>(a, parts, part, s);
  hipLaunchKernelGGL((ns_init_kernel<T, kMuon>), dim3((p.mp / 32) * ((p.np / 32 + kInit - 1) / kInit), (unsigned)a.batch), dim3(256), 0, s, a, p, parts, part, ws);
  int cur = 0;
  for (int k = 0; k < a.steps; ++k, cur ^= 1) {
    char *xr = ws + p.x[cur], *xc = xr + 2 * p.xplane, *yr = ws + p.x[cur ^ 1], *yc = yr + 2 * p.xplane;
    NsProd g{};
    g.stride = p.stride;
    // A = X X^T
    g.P = g.Q = xr;
    g.p_lo = g.q_lo = p.xplane;
    g.Rp = g.Rq = p.mp;
    g.K = p.np;
    g.Y = g.Z = ws + p.a;
    g.y_lo = g.z_lo = p.aplane;
    g.f = kSa / (kSx * kSx);
    if (p.slices > 1) {
      const int c = p.mp / 64, odd = p.mp % 64 != 0;
      g.whole = c * (c + 1) / 2;
      g.rest = odd * (c + 1);
      g.part = parts_at;
      g.slices = p.slices;
      const unsigned tiles = (unsigned)((g.whole + g.rest) * a.batch);
      hipLaunchKernelGGL((ns_prod_kernel<kPart, kOpF32, 1, 1>), dim3(tiles * p.slices), dim3(256), 0, s, g, a, p);
      hipLaunchKernelGGL((ns_prod_kernel<kJoin, kOpF32, 1, 1>), dim3(tiles), dim3(256), 0, s, g, a, p);
    } else {
      launch_prod<kGram, kOpF32>(g, a, p, s);
    }
    // B = a I + b A + c A A
    g.P = g.Q = g.E = ws + p.a;
    g.p_lo = g.q_lo = g.e_lo = p.aplane;
    g.K = p.mp;
    g.Y = g.Z = ws + p.b;
    g.f = a.c * kSb / (kSa * kSa);
    g.e = a.b * kSb / kSa;
    launch_prod<kSquare, kOpF32>(g, a, p, s);
    // X <- B X
    g.P = ws + p.b;
    g.Q = xc;
    g.q_lo = p.xplane;
    g.Rq = p.np;
    g.Y = yc;
    g.Z = yr;
    g.y_lo = g.z_lo = p.xplane;
    const bool last = k + 1 == a.steps;
    const float sy = last ? 1.f : kSx;
    g.f = sy / (kSb * kSx);
    if (last) launch_prod<kFinal, T>(g, a, p, s);
    else launch_prod<kUpdate, kOpF32>(g, a, p, s);
  }
}

}  // namespace

int64_t ns_workspace(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  int64_t stride = 0;
  switch (path_of(rows, cols)) {
    case kThinSmall: stride = make_thin<2, 2, kWavesSmall>(batch, rows, cols).stride; break;
    case kThin32: stride = make_thin<1, 4, kWaves32>(batch, rows, cols).stride; break;
    case kThin64: stride = make_thin<2, 4, kWaves64>(batch, rows, cols).stride; break;
    default: {
      const NsPlan p = make_plan(batch, rows, cols);
      return batch * (kNormParts * 8 + p.stride) + p.parts;
    }
  }
  return batch * (kNormParts * 8 + stride);
}

namespace {
template <int T>
void launch_by_kind(const NsArgs& a, void* workspace, hipStream_t s) {
  if (a.momentum.p) launch_ns_t<T, true>(a, workspace, s);
  else launch_ns_t<T, false>(a, workspace, s);
}
}  // namespace

void launch_ns(const NsArgs& a, void* workspace, hipStream_t s) {
  // T: the type read (and, by orthogonalize, written); the parameter of muon is fp32
  if (a.dtype == kOpF32) launch_by_kind<kOpF32>(a, workspace, s);
  else if (a.dtype == kOpBF16) launch_by_kind<kOpBF16>(a, workspace, s);
  else launch_by_kind<kOpF16>(a, workspace, s);
}

}  // namespace lcn
