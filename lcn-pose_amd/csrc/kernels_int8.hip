// Matrix product in 8-bit integers with one scale a token and one a channel
// (gfx950): the activations are quantised on the way in, the weights once.
//
//   s[t] = max_k |x[t,k]| / 127,   q[t,k] = rint(x[t,k] * (127 / max_k |x[t,k]|))
//   y[t,n] = (sum_k q[t,k] w[n,k]) * s[t] * sw[n] + bias[n]
//
// A row whose largest magnitude is below 2^-100 counts as zero (127 / max would
// overflow); a row that holds an infinity or a NaN gives NaN throughout: its
// scale is NaN and its integers are zero.  The sums are exact (int32, K <= 131072).
//
// Quantised tokens are stored in panels of 64 of K: element (t, k) at
// (k / 64) rows 64 + 64 t + k % 64, K padded with zeros.  A panel's rows follow
// each other, so an LDS-DMA of 16 rows x 64 bytes reads 1 KB of whole cache lines
// (from row-major integers it reads half of 16 lines: 65 536 x 1088 x 1088 spent
// 100 of 220 us on that).  Weights that many tiles read are laid out the same way.
#include <algorithm>

#include "ops_common.h"

namespace lcn {

namespace {

__host__ __device__ inline int64_t pad64(int64_t v) { return (v + 63) / 64 * 64; }
__host__ __device__ inline int64_t pad256(int64_t v) { return (v + 255) / 256 * 256; }

constexpr int64_t kPanelTokens = 1024;
constexpr int64_t kGroupTokens = 16384;  // one workgroup of 64 a CU
constexpr int64_t kGroupMost = (int64_t)1 << 29;  // of a launch, whose threads are counted in 32 bits

// largest magnitude of a wave's values, and whether one is an infinity or a NaN
__device__ __forceinline__ void wave_top(float& top, bool& bad) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  bad = __any(bad);
}
__device__ __forceinline__ void see(float v, float& top, bool& bad) {
  v = fabsf(v);
  bad |= !(v < __builtin_inff());
  top = fmaxf(top, v);
}

// Rows are read 16 bytes at a time at any alignment; what a row has past its last
// whole piece comes an element a lane (`tail_piece`).  kOnce: not kept in the
// caches, which then hold the integers for the product.
typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned u32_any __attribute__((aligned(1)));
template <int T> constexpr int kElem = 16 / kVec<T>;  // bytes
template <int T>
__device__ __forceinline__ v4u tail_piece(const void* p, int64_t e, int rem, int lane) {
  unsigned b = 0;
  if (lane < rem) b = T == kOpF32 ? ((const unsigned*)p)[e + lane] : ((const unsigned short*)p)[e + lane];
  v4u u;
#pragma unroll
  for (int d = 0; d < 4; ++d) u[d] = T == kOpF32 ? __shfl(b, d) : __shfl(b, 2 * d) | __shfl(b, 2 * d + 1) << 16;
  return u;
}
// piece c of the row at element r: one of the `whole` pieces, the tail, or zeros
template <int T, bool kOnce>
__device__ __forceinline__ v4u row_piece(const void* p, int64_t r, int c, int whole, v4u tail) {
  v4u u = {0, 0, 0, 0};
  if (c < whole) {
    const v4u_any* at = (const v4u_any*)((const char*)p + (r + (int64_t)c * kVec<T>) * kElem<T>);
    u = kOnce ? __builtin_nontemporal_load(at) : *at;
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) u[d] = c == whole ? tail[d] : u[d];
  return u;
}
template <int T>
__device__ __forceinline__ void see_piece(v4u u, float& top, bool& bad) {
  float v[kVec<T>];
  unpack_vec<T>(u, v);
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e) see(v[e], top, bad);
}
// the piece's integers, kVec bytes at `o`
template <int T>
__device__ __forceinline__ void put_piece(void* o, v4u u, float factor, bool bad) {
  float v[kVec<T>];
  unpack_vec<T>(u, v);
  if constexpr (kVec<T> == 4) *(unsigned*)o = quant4(v[0], v[1], v[2], v[3], factor, bad);
  else *(uint2*)o = make_uint2(quant4(v[0], v[1], v[2], v[3], factor, bad), quant4(v[4], v[5], v[6], v[7], factor, bad));
}
// 16 weights from p (at + 16 may pass the row: zeros of the tokens meet what is
// there; at the end of the weights, byte by byte)
__device__ __forceinline__ v4i weights16(const int8_t* p, int left, const int8_t* end) {
  v4i v = {0, 0, 0, 0};
  if (p + 16 <= end) {
    v = *(const v4i_any*)p;
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (e < left) v[e >> 2] |= (int)((unsigned)(uint8_t)p[e] << (8 * (e & 3)));
  }
  return v;
}

// One wave a row: largest magnitude, then the integers, rows padded to kp with
// zeros.  A lane keeps up to kRegs pieces in registers between the two passes; what
// is past them is read again (from L2).  Bound by memory: 65 536 x 1088 fp32 in 60 us
// (5.9 TB/s).  x is read past the caches: with it in them, the integers had to come
// from memory again (77 us here, and 140 instead of 98 us in the product).
template <int T, int kRegs>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* __restrict__ x, int64_t x_row, int64_t tokens, int k,
                                                         int64_t kp, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int V = kVec<T>;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= tokens) return;
  float top = 0.f, factor, s;
  bool bad = false;
  const int64_t r = t * x_row, panel = tokens * 64;
  int8_t* out = q + t * 64;
  const int whole = k / V, padded = (int)(kp / V);
  v4u keep[kRegs], tail = {0, 0, 0, 0};
  if (k % V) tail = tail_piece<T>(x, r + (int64_t)whole * V, k % V, lane);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) keep[i] = row_piece<T, true>(x, r, lane + 64 * i, whole, tail);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) see_piece<T>(keep[i], top, bad);
  for (int c = lane + 64 * kRegs; c <= whole; c += 64) see_piece<T>(row_piece<T, false>(x, r, c, whole, tail), top, bad);
  wave_top(top, bad);
  row_scale(top, bad, factor, s);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int c = lane + 64 * i;
    if (c < padded) put_piece<T>(out + (c * V >> 6) * panel + (c * V & 63), keep[i], factor, bad);
  }
  for (int c = lane + 64 * kRegs; c < padded; c += 64)
    put_piece<T>(out + (c * V >> 6) * panel + (c * V & 63), row_piece<T, false>(x, r, c, whole, tail), factor, bad);
  if (lane == 0) scale[t] = s;
}

// four weights of a row from k0 on, zeros past K
__device__ __forceinline__ unsigned weights4(const int8_t* row, int k0, int k) {
  unsigned v = 0;
  if (k0 + 4 <= k) {
    v = *(const u32_any*)(row + k0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k0 + e < k) v |= (unsigned)(uint8_t)row[k0 + e] << (8 * e);
  }
  return v;
}
// weight rows -> panels of 64 of K, zero padded
__global__ __launch_bounds__(256) void panels_kernel(const int8_t* __restrict__ w, int64_t w_row, int n, int k, int8_t* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);  // channel
  if (c >= n) return;
  const int at = (threadIdx.x & 15) * 4;
  *(unsigned*)(out + ((int64_t)blockIdx.y * n + c) * 64 + at) = weights4(w + c * w_row, blockIdx.y * 64 + at, k);
}

#define I8_LDS(SRC, VOFF, SOFF, DST) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(SRC, (__attribute__((address_space(3))) void*)(DST), 16, VOFF, SOFF, 0, 0)

struct Int8Gemm {
  const int8_t* q; const float* qs; int64_t kp;    // panels of the tokens, their scales, padded K
  const int8_t* w; int64_t w_row, w_panel;         // 64-byte piece p of row c at p w_panel + c w_row, 16-byte aligned
  int64_t w_bytes;                                 // readable from w
  const float* ws; const float* bias;
  void* out; int64_t out_row;
  int64_t tokens; int n;
  int tn;                                          // channel tiles
};

// A tile of 64 BI tokens x 64 BJ channels, 2 x 2 waves of 32 BI x 32 BJ, 64
// bytes of K a stage through a ring of R LDS buffers filled by LDS-DMA, R - 1 to
// R stages in flight.  A stage holds rows of 64 bytes (four 16-byte units); unit c
// of row r sits at c ^ ((r >> 2) & 3), so the 32 rows of a fragment read spread
// over all banks; the permutation is made by the lane's choice of global
// address.  The buffers are separate LDS objects, so the compiler adds no waits
// for loads into the others.
template <int T, int BI, int BJ, int R>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void int8_gemm_kernel(Int8Gemm g) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass emits no launch stub for this body)
  constexpr int kRows = 64 * (BI + BJ), kStage = kRows * 64, L = BI + BJ;  // L: loads of a wave per stage
  static_assert(R == 3 || R == 4 || R == 8, "buffers named below");
  constexpr int kFourth = R >= 4 ? kStage : 16, kRest = R == 8 ? kStage : 16;
  __shared__ __attribute__((aligned(16))) char l0[kStage], l1[kStage], l2[kStage], l3[kFourth], l4[kRest], l5[kRest], l6[kRest], l7[kRest];
#define I8_BUF(I) ((I) % R == 0 ? l0 : (I) % R == 1 ? l1 : (I) % R == 2 ? l2 : (I) % R == 3 ? l3 : (I) % R == 4 ? l4 : (I) % R == 5 ? l5 : (I) % R == 6 ? l6 : l7)
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t t0 = (int64_t)(id / g.tn) * (64 * BI);
  const int n0 = (id % g.tn) * (64 * BJ);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = w >> 1, wj = w & 1, h = lane >> 5, l31 = lane & 31;
  // rows past the end repeat the last one; their results are not stored
  const int trows = (int)min((int64_t)(64 * BI), g.tokens - t0), nrows = min(64 * BJ, g.n - n0);
  const int64_t wat = (int64_t)n0 * g.w_row;
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(g.q + t0 * 64), 0, (int)(g.kp * g.tokens - t0 * 64), 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(g.w + wat), 0, (int)(g.w_bytes - wat), 0x00020000);
  const int qp = (int)g.tokens * 64, wp = (int)g.w_panel;
  // load i of a wave: 16 rows x 64 bytes
  int voq[BI], vow[BJ];
#pragma unroll
  for (int i = 0; i < BI; ++i) {
    const int r = (i * 4 + w) * 16 + (lane >> 2);
    voq[i] = min(r, trows - 1) * 64 + (((lane & 3) ^ ((r >> 2) & 3)) * 16);
  }
#pragma unroll
  for (int i = 0; i < BJ; ++i) {
    const int r = (i * 4 + w) * 16 + (lane >> 2);
    vow[i] = min(r, nrows - 1) * (int)g.w_row + (((lane & 3) ^ ((r >> 2) & 3)) * 16);
  }
  auto stage = [&](int ks, char* buf) {
    char* d = buf + w * 1024;
    const int sq = ks * qp, sw = ks * wp;
#pragma unroll
    for (int i = 0; i < BI; ++i) I8_LDS(rq, voq[i], sq, d + i * 4096);
#pragma unroll
    for (int i = 0; i < BJ; ++i) I8_LDS(rw, vow[i], sw, d + (BI + i) * 4096);
  };
  __shared__ float qs[64 * BI];  // the tokens' scales
  if (threadIdx.x < trows) qs[threadIdx.x] = g.qs[t0 + threadIdx.x];
  v16i acc[BI][BJ];
#pragma unroll
  for (int x = 0; x < BI; ++x)
#pragma unroll
    for (int y = 0; y < BJ; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0;
  const int nk = (int)(g.kp / 64);
  struct Frag { v4i p[BI], q[BJ]; };
  auto fetch = [&](const char* buf, int kk, Frag& f) {
    const int c = ((2 * kk + h) ^ ((l31 >> 2) & 3)) * 16 + l31 * 64;
#pragma unroll
    for (int x = 0; x < BI; ++x) f.p[x] = *(const v4i*)(buf + (wi * BI + x) * 2048 + c);
#pragma unroll
    for (int y = 0; y < BJ; ++y) f.q[y] = *(const v4i*)(buf + BI * 4096 + (wj * BJ + y) * 2048 + c);
  };
  auto multiply = [&](const Frag& f) {
#pragma unroll
    for (int x = 0; x < BI; ++x)
#pragma unroll
      for (int y = 0; y < BJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.p[x], f.q[y], acc[x][y], 0, 0, 0);
  };
  // A stage is two halves of 32 bytes.  Step s multiplies the first, held in f0,
  // while the second is read, then the second while the next stage's first is
  // read.  Past the barrier stage s + 1 has landed for every wave, and every wave
  // holds the rest of stage s in registers: its buffer takes stage s + R.
  Frag f0, f1;
  auto step = [&](int s, char* mine, const char* after, bool more, bool load) {
    fetch(mine, 1, f1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(f0);
    if (more) {
      if (load) stage_barrier<(R - 2) * L>();
      else stage_barrier<0>();
      if (load) stage(s + R, mine);
      fetch(after, 0, f0);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(f1);
  };
  int ks = 0;
  if (nk >= 2 * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) stage(i, I8_BUF(i));
    stage_barrier<(R - 1) * L>();
    fetch(l0, 0, f0);
    do {
#pragma unroll
      for (int i = 0; i < R; ++i) step(ks + i, I8_BUF(i), I8_BUF(i + 1), true, true);
      ks += R;
    } while (ks + 2 * R <= nk);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < nk) stage(i, I8_BUF(i));
    stage_barrier<0>();
    fetch(l0, 0, f0);
  }
  for (; ks < nk; ks += R) {  // at most 2 R - 1 stages remain
    const int left = nk - ks;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (left > i) step(ks + i, I8_BUF(i), I8_BUF(i + 1), left > i + 1, left > R + i);
  }
#undef I8_BUF
  // The tile of the output as a buffer: its rows end with the tile, so stores of
  // rows past the tokens are dropped, and lanes past the channels point behind it.
  // Row offsets are scalar: a store costs no address arithmetic.
  constexpr int kOut = T == kOpF32 ? 4 : 2;
  const int64_t obytes = ((int64_t)(trows - 1) * g.out_row + nrows) * kOut;
  const bool near = (int64_t)(64 * BI) * g.out_row * kOut + nrows * kOut < 0x7fffffff;  // no offset wraps, dropped rows' neither
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc((char*)g.out + (t0 * g.out_row + n0) * kOut, 0, (int)obytes, 0x00020000);
#pragma unroll
  for (int y = 0; y < BJ; ++y) {
    const int c = (wj * BJ + y) * 32 + l31;
    const bool in = c < nrows;
    const float sw = in ? g.ws[n0 + c] : 0.f, b = in && g.bias ? g.bias[n0 + c] : 0.f;
    const int vout = in ? (4 * h * (int)g.out_row + c) * kOut : -1;
#pragma unroll
    for (int x = 0; x < BI; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = (wi * BI + x) * 32 + 8 * q;
        const float4 s4 = *(const float4*)(qs + r + 4 * h);
        const float se[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = (float)acc[x][y][4 * q + e] * se[e] * sw;
          if (g.bias) v += b;
          if (near) {
            const int so = (r + e) * (int)g.out_row * kOut;
            if constexpr (T == kOpF32) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), ro, vout, so, 0);
            else if constexpr (T == kOpBF16) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)v), ro, vout, so, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (_Float16)v), ro, vout, so, 0);
          } else if (in && r + 4 * h + e < trows) {
            op_store<T>(g.out, (t0 + r + 4 * h + e) * g.out_row + n0 + c, v);
          }
        }
      }
  }
#endif
}

// ---- many tokens of moderate length ----------------------------------------------------------
// A workgroup quantises 64 tokens into LDS and multiplies them by every channel:
// x is read once, and no integers go through memory.  The integers lie as the
// matrix instruction reads them: unit u (16 of K) of token r at block (u / 2,
// r / 32), half u % 2, slot (r ^ u) % 32 of 16 bytes, so that 64 lanes write (16
// units of one row) and read (32 rows of two units) all banks evenly.  Weights lie
// the same way without the permutation, 1 KB a load, straight from L2 into
// registers, four panels of 64 ahead.  A wave takes 64 channels at a time and runs
// alone after the one barrier; two workgroups share a CU, so one's loads of x run
// under the other's products.
// Against the integers through memory (quantise, lay out, multiply), K 1088:
// 65 536 tokens x 1088 channels 182 -> 160 us (fp32), 163 -> 130 (bf16); x 4352
// channels 618 -> 465, 552 -> 377; 16 384 x 1088 60 -> 53, 59 -> 49; 8192 x 1088,
// where half the CUs would have no workgroup, 39 -> 52: taken from one workgroup a
// CU on.  What is left against the bytes' time (110 us) is the first workgroups'
// loads, under which nothing runs yet.
constexpr int kGroup = 64;                   // tokens
constexpr int kGroupLds = 80 * 1024 - 512;   // half a CU's

__global__ __launch_bounds__(256) void fragments_kernel(const int8_t* __restrict__ w, int64_t w_row, int n, int k, int kp, int8_t* __restrict__ out) {
  const int c = blockIdx.x * 16 + (threadIdx.x >> 4);  // channel, up to n rounded up to 64
  const int k0 = blockIdx.y * 64 + (threadIdx.x & 15) * 4;
  const unsigned v = c < n ? weights4(w + (int64_t)c * w_row, k0, k) : 0u;
  *(unsigned*)(out + (int64_t)(c >> 5) * kp * 32 + (k0 >> 5) * 1024 + ((k0 >> 4) & 1) * 512 + (c & 31) * 16 + (k0 & 15)) = v;
}

// kFar: output rows more than 2^22 elements apart, stored at 64-bit addresses.
template <int T, bool kFar>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void int8_group_kernel(Int8Gemm g, const void* __restrict__ x, int64_t x_row, int k) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ __attribute__((aligned(16))) float qs[kGroup];
  const int64_t t0 = (int64_t)blockIdx.x * kGroup;
  const int trows = (int)min((int64_t)kGroup, g.tokens - t0);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, l31 = lane & 31;
  const int nk = (int)(g.kp / 64), tiles = (g.n + 63) / 64;
  // weights: panel p of tile t, block y, half kk at ((2 t + y) 2 nk + 2 p + kk) KB
  const int first = (w + blockIdx.x) & 3;  // the waves with a tile more change from workgroup to workgroup
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)g.w, 0, (int)g.w_bytes, 0x00020000);
  struct Panel { v4i v[2][2]; };
  int lt = first, lp = 0;
  auto weights = [&](Panel& b) {
    const int at = lt < tiles ? (lt * 4 * nk + 2 * lp) * 1024 : 0;  // (past the last tile: not used)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int y = 0; y < 2; ++y)
        b.v[y][kk] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, lane * 16, at + (y * 2 * nk + kk) * 1024, 0));
    if (++lp == nk) { lp = 0; lt += 4; }
  };
  {
    // four groups of four rows a wave, the next group's loads in flight
    constexpr int V = kVec<T>, kRegs = T == kOpF32 ? 5 : 3, kRows = 4;
    const int whole = k / V, padded = (int)(g.kp / V);
    struct Rows { v4u u[kRows][kRegs]; };
    auto load = [&](int r0, Rows& m) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int64_t r = (t0 + min(r0 + j, trows - 1)) * x_row;
        v4u tail = {0, 0, 0, 0};
        if (k % V) tail = tail_piece<T>(x, r + (int64_t)whole * V, k % V, lane);
#pragma unroll
        for (int i = 0; i < kRegs; ++i) m.u[j][i] = row_piece<T, true>(x, r, lane + 64 * i, whole, tail);
      }
    };
    auto quantise = [&](int r0, const Rows& m) {
      float top[kRows];
      bool bad[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        top[j] = 0.f;
        bad[j] = false;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) see_piece<T>(m.u[j][i], top[j], bad[j]);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) wave_top(top[j], bad[j]);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int r = r0 + j;
        float factor, s;
        row_scale(top[j], bad[j], factor, s);
        if (lane == 0) qs[r] = s;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          const int at = (lane + 64 * i) * V, u = at >> 4;
          if (lane + 64 * i < padded)
            put_piece<T>(lds + (u >> 1) * 2048 + (r >> 5) * 1024 + (u & 1) * 512 + ((r ^ u) & 31) * 16 + (at & 15), m.u[j][i], factor, bad[j]);
        }
      }
    };
    Rows m0, m1;
    const int r0 = w * 16;
    load(r0, m0);
    __builtin_amdgcn_sched_barrier(0);
    load(r0 + 4, m1);
    __builtin_amdgcn_sched_barrier(0);
    quantise(r0, m0);
    load(r0 + 8, m0);
    __builtin_amdgcn_sched_barrier(0);
    quantise(r0 + 4, m1);
    load(r0 + 12, m1);
    __builtin_amdgcn_sched_barrier(0);
    quantise(r0 + 8, m0);
    quantise(r0 + 12, m1);
  }
  Panel b0, b1, b2, b3;
  const int total = (tiles - first + 3) / 4 * nk;  // panels of this wave (none: first >= tiles)
  if (first < tiles) {
    weights(b0);
    __builtin_amdgcn_sched_barrier(0);
    weights(b1);
    __builtin_amdgcn_sched_barrier(0);
    weights(b2);
    __builtin_amdgcn_sched_barrier(0);
    weights(b3);
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  if (first >= tiles) return;
  v16i acc[2][2];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  };
  clear();
  constexpr int kOut = T == kOpF32 ? 4 : 2;
  const int64_t obytes = ((int64_t)(trows - 1) * g.out_row + g.n) * kOut;
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc((char*)g.out + t0 * g.out_row * kOut, 0, (int)obytes, 0x00020000);
  int tile = first;
  float scales[2], biases[2];  // of this tile's channels
  const float* bias = g.bias ? g.bias : g.ws;  // (read without a branch, whose merge would wait for the loads in flight)
  auto channels = [&]() {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = min(tile * 64 + y * 32 + l31, g.n - 1);
      scales[y] = g.ws[c];
      biases[y] = bias[c];
    }
  };
  channels();
  auto finish = [&]() {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = tile * 64 + y * 32 + l31;
      const bool in = c < g.n;
      const float sw = scales[y], b = g.bias ? biases[y] : 0.f;
      const int vout = kFar ? 0 : in ? (4 * h * (int)g.out_row + c) * kOut : -1;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = i * 32 + 8 * q;
          const float4 s4 = *(const float4*)(qs + r + 4 * h);
          const float se[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = (float)acc[i][y][4 * q + e] * se[e] * sw + b;
            if constexpr (kFar) {
              if (in && r + 4 * h + e < trows) op_store<T>(g.out, (t0 + r + 4 * h + e) * g.out_row + c, v);
              continue;
            }
            const int so = (r + e) * (int)g.out_row * kOut;
            if constexpr (T == kOpF32) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), ro, vout, so, 0);
            else if constexpr (T == kOpBF16) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)v), ro, vout, so, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (_Float16)v), ro, vout, so, 0);
          }
        }
    }
    clear();
    tile += 4;
    channels();
  };
  struct Frag { v4i v[2][2]; };
  auto fetch = [&](int p, Frag& f) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int u = 4 * p + 2 * kk + h;
#pragma unroll
      for (int i = 0; i < 2; ++i) f.v[kk][i] = *(const v4i*)(lds + (2 * p + kk) * 2048 + i * 1024 + h * 512 + ((l31 ^ u) & 31) * 16);
    }
  };
  Frag f0, f1;
  int p = 0;
  fetch(0, f0);
  auto step = [&](Panel& b, Frag& f, Frag& next) {
    const int after = p + 1 == nk ? 0 : p + 1;
    fetch(after, next);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[i][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.v[kk][i], b.v[y][kk], acc[i][y], 0, 0, 0);
    weights(b);
    if (after == 0 && tile < tiles) finish();
    p = after;
  };
  // (one exit, or the compiler waits for all loads at the top; panels past the last are multiplied and dropped)
  for (int s = 0; s < total; s += 4) {
    step(b0, f0, f1);
    step(b1, f1, f0);
    step(b2, f0, f1);
    step(b3, f1, f0);
  }
#endif
}

// ---- few tokens ----------------------------------------------------------------------------
// At most 16 tokens: a workgroup takes 16 channels, its four waves every fourth
// 64-byte piece of K, straight from memory into v_mfma_i32_16x16x64_i8; the
// partial sums meet in LDS.  kFused: the workgroup also quantises the tokens,
// each time anew (they are small), which makes the product one launch.  Bound by
// latency: one round of loads in flight for the weights.
constexpr int kFewTokens = 16;
constexpr int kFewLds = 65536;   // bytes of quantised tokens a workgroup holds

template <int T, bool kFused>
__global__ __launch_bounds__(256) void int8_few_kernel(Int8Gemm g, const void* __restrict__ x, int64_t x_row, int k) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int red[4][256];
  __shared__ float qs[kFewTokens], tops[4][4];
  __shared__ int bads[4][4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int kp = (int)g.kp, tokens = (int)g.tokens;
  const int n0 = blockIdx.x * 16;
  const int c16 = lane & 15, kq = lane >> 4;  // channel (or token) of the fragment, its 16-byte quarter of a piece
  const int8_t* wrow = g.w + (int64_t)min(n0 + c16, g.n - 1) * g.w_row;
  const int8_t* wend = g.w + g.w_bytes;
  auto weights = [&](int ks) {
    const int at = ks * 64 + kq * 16;
    return at < k ? weights16(wrow + at, k - at, wend) : v4i{0, 0, 0, 0};
  };
  const int nk = kp / 64;
  constexpr int kAhead = 4;  // pieces of a wave in flight
  v4i wv[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (w + 4 * i < nk) wv[i] = weights(w + 4 * i);
  const int pitch = kp + 16;  // rows start 16 bytes apart in the banks
  if constexpr (kFused) {
    // four rows at a time, one a wave, or (fewer tokens than waves) one row after
    // another by the whole workgroup; up to kRegs elements a thread stay in registers
    constexpr int kRegs = 8;
    const bool wide = tokens < 4;
    const int step = wide ? 256 : 64, at = wide ? threadIdx.x : lane;
    for (int t = wide ? 0 : w; t < tokens; t += wide ? 1 : 4) {
      float top = 0.f, factor, s, keep[kRegs];
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kRegs; ++i) keep[i] = at + i * step < k ? op_load<T>(x, t * x_row + at + i * step) : 0.f;
#pragma unroll
      for (int i = 0; i < kRegs; ++i) see(keep[i], top, bad);
      for (int c = at + kRegs * step; c < k; c += step) see(op_load<T>(x, t * x_row + c), top, bad);
      wave_top(top, bad);
      if (wide) {
        if (lane == 0) { tops[t][w] = top; bads[t][w] = bad; }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) { top = fmaxf(top, tops[t][i]); bad |= bads[t][i] != 0; }
      }
      row_scale(top, bad, factor, s);
      if (at == 0) qs[t] = s;
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (at + i * step < kp) lds[t * pitch + at + i * step] = bad ? (char)0 : quant(keep[i], factor);
      for (int c = at + kRegs * step; c < kp; c += step)
        lds[t * pitch + c] = c < k && !bad ? quant(op_load<T>(x, t * x_row + c), factor) : (char)0;
    }
    __syncthreads();
  } else if (threadIdx.x < tokens) {
    qs[threadIdx.x] = g.qs[threadIdx.x];
  }
  v4i acc = {0, 0, 0, 0};
  const int tr = min(c16, tokens - 1);  // rows past the tokens repeat the last
  for (int ks = w; ks < nk; ks += 4 * kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = ks + 4 * i;
      if (p >= nk) break;
      v4i q;
      if constexpr (kFused) q = *(const v4i*)(lds + tr * pitch + p * 64 + kq * 16);
      else q = *(const v4i*)(g.q + ((int64_t)p * tokens + tr) * 64 + kq * 16);
      const v4i ww = wv[i];
      if (p + 4 * kAhead < nk) wv[i] = weights(p + 4 * kAhead);
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q, ww, acc, 0, 0, 0);
    }
  }
  // lane holds tokens 4 kq .. 4 kq + 3 of channel c16
#pragma unroll
  for (int e = 0; e < 4; ++e) red[w][(4 * kq + e) * 16 + c16] = acc[e];
  __syncthreads();
  const int t = threadIdx.x >> 4, n = n0 + (threadIdx.x & 15);
  if (t < tokens && n < g.n) {
    const int sum = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
    float v = (float)sum * qs[t] * g.ws[n];
    if (g.bias) v += g.bias[n];
    op_store<T>(g.out, t * g.out_row + n, v);
  }
}

// ---- up to some hundred tokens ---------------------------------------------------------------
// A workgroup takes 16 tokens x 64 channels: each of its 16 waves quantises a token
// into LDS, each of the n / 64 workgroups anew (they come from L2), then multiplies
// the 16 tokens by 16 channels over every fourth 64-byte piece of K, whose weights
// are asked for before the quantisation starts; the four sums of a block meet in
// LDS.  One launch, no workspace.  Bound by latency (the rows, their largest
// magnitude, the weights): 200 x 1088 x 1088 in 6.3 us a launch of a graph (5.8 us the
// kernel itself), 8.8 with 4 waves, 6.9 with 8.
constexpr int kMidWaves = 16;
template <int T>
__global__ __launch_bounds__(64 * kMidWaves) __attribute__((amdgpu_waves_per_eu(8))) void int8_mid_kernel(Int8Gemm g, const void* __restrict__ x, int64_t x_row, int k) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kKs = kMidWaves / 4, kRows = 16 / kMidWaves;  // waves that share 16 channels, rows of a wave
  constexpr int kMidAhead = 4;  // 64-byte pieces of K of a wave in flight
  __shared__ float qs[16];
  __shared__ int sums[kKs - 1][4][4][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kp = (int)g.kp, nk = kp / 64, pitch = kp + 16;
  const int64_t t0 = (int64_t)blockIdx.x * 16;
  const int rows = (int)min((int64_t)16, g.tokens - t0);
  const int c16 = lane & 15, kq = lane >> 4, n0 = blockIdx.y * 64 + (w & 3) * 16, part = w >> 2;
  // channels past the last repeat it, K past its end meets zeros of the tokens
  const int8_t* wrow = g.w + (int64_t)min(n0 + c16, g.n - 1) * g.w_row;
  const int8_t* wend = g.w + g.w_bytes;
  auto weights = [&](int ks) {
    const int at = ks * 64 + kq * 16;
    return at < k ? weights16(wrow + at, k - at, wend) : v4i{0, 0, 0, 0};
  };
  v4i wv[kMidAhead];
#pragma unroll
  for (int i = 0; i < kMidAhead; ++i) wv[i] = weights(part + kKs * i);
  {
    // the first kRegs pieces of four rows stay in registers
    constexpr int V = kVec<T>, kRegs = T == kOpF32 ? 5 : 3;
    const int whole = k / V, padded = kp / V;
    int64_t r[kRows];
    v4u keep[kRows][kRegs], tail[kRows];
    float top[kRows];
    bool bad[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      r[j] = (t0 + min(w * kRows + j, rows - 1)) * x_row;
      tail[j] = v4u{0, 0, 0, 0};
      if (k % V) tail[j] = tail_piece<T>(x, r[j] + (int64_t)whole * V, k % V, lane);
#pragma unroll
      for (int i = 0; i < kRegs; ++i) keep[j][i] = row_piece<T, false>(x, r[j], lane + 64 * i, whole, tail[j]);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      top[j] = 0.f;
      bad[j] = false;
#pragma unroll
      for (int i = 0; i < kRegs; ++i) see_piece<T>(keep[j][i], top[j], bad[j]);
    }
    for (int c = lane + 64 * kRegs; c <= whole; c += 64)
#pragma unroll
      for (int j = 0; j < kRows; ++j) see_piece<T>(row_piece<T, false>(x, r[j], c, whole, tail[j]), top[j], bad[j]);
    float factor[kRows];
    char* o = lds + w * kRows * pitch;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      float s;
      wave_top(top[j], bad[j]);
      row_scale(top[j], bad[j], factor[j], s);
      if (lane == 0) qs[w * kRows + j] = s;
#pragma unroll
      for (int i = 0; i < kRegs; ++i) asm volatile("" : "+v"(keep[j][i]));  // unpacked anew, not kept as floats
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (lane + 64 * i < padded) put_piece<T>(o + j * pitch + (lane + 64 * i) * V, keep[j][i], factor[j], bad[j]);
    }
    for (int c = lane + 64 * kRegs; c < padded; c += 64)
#pragma unroll
      for (int j = 0; j < kRows; ++j) put_piece<T>(o + j * pitch + c * V, row_piece<T, false>(x, r[j], c, whole, tail[j]), factor[j], bad[j]);
  }
  __syncthreads();
  v4i acc = {0, 0, 0, 0};
  const char* a = lds + c16 * pitch + kq * 16;
  for (int ks = part; ks < nk; ks += kKs * kMidAhead) {
#pragma unroll
    for (int i = 0; i < kMidAhead; ++i) {
      const int p = ks + kKs * i;
      if (p >= nk) break;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const v4i*)(a + p * 64), wv[i], acc, 0, 0, 0);
      wv[i] = weights(p + kKs * kMidAhead);
    }
  }
  if (part)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[part - 1][w & 3][e][lane] = acc[e];
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int q = 0; q + 1 < kKs; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += sums[q][w & 3][e][lane];
  // lane holds tokens 4 kq .. 4 kq + 3 of channel c16
  const int n = n0 + c16;
  if (n < g.n) {
    const float sw = g.ws[n], b = g.bias ? g.bias[n] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 4 * kq + e;
      if (t >= rows) continue;
      float v = (float)acc[e] * qs[t] * sw;
      if (g.bias) v += b;
      op_store<T>(g.out, (t0 + t) * g.out_row + n, v);
    }
  }
}

// one wave a channel: largest magnitude over k, then the integers
template <int T>
__global__ __launch_bounds__(256) void quant_weight_kernel(QuantWArgs a) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= a.n) return;
  float top = 0.f;
  bool bad = false;
  for (int c = lane; c < a.k; c += 64) {
    const float v = fabsf(op_load<T>(a.w, n * a.w_n + c * a.w_k));
    bad |= !(v < __builtin_inff());
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  bad = __any(bad);
  float factor, s;
  row_scale(top, bad, factor, s);
  if (lane == 0) a.scale[n] = s;
  for (int c = lane; c < a.k; c += 64)
    a.q[(int64_t)n * a.k + c] = bad ? (int8_t)0 : quant(op_load<T>(a.w, n * a.w_n + c * a.w_k), factor);
}

template <int T>
void launch_quant_rows(const Int8Args& a, int64_t kp, int8_t* q, float* qs, hipStream_t s) {
  const dim3 grid((unsigned)((a.tokens + 3) / 4));
  constexpr int kMany = T == kOpF32 ? 18 : 9;  // K up to 4608 in registers
  if (a.k <= 64 * 5 * kVec<T>) hipLaunchKernelGGL((quant_rows_kernel<T, 5>), grid, dim3(256), 0, s, a.x, a.x_row, a.tokens, a.k, kp, q, qs);
  else hipLaunchKernelGGL((quant_rows_kernel<T, kMany>), grid, dim3(256), 0, s, a.x, a.x_row, a.tokens, a.k, kp, q, qs);
}

template <int T, int BI, int BJ, int R>
void launch_tiles(Int8Gemm& g, hipStream_t s) {
  g.tn = (g.n + 64 * BJ - 1) / (64 * BJ);
  const int64_t tt = (g.tokens + 64 * BI - 1) / (64 * BI);
  hipLaunchKernelGGL((int8_gemm_kernel<T, BI, BJ, R>), dim3((unsigned)(tt * g.tn)), dim3(256), 0, s, g);
}

// every workgroup quantises the tokens for itself while that is little work
bool fused(int64_t tokens, int64_t k) {
  return tokens <= kFewTokens && tokens * (pad64(k) + 16) <= kFewLds && tokens * k <= 16384;
}

// The same for a few hundred tokens, 16 at a time: at most two workgroups a CU, and
// rows that stay in registers.  Measured against quantise + multiply (aligned rows)
// or lay out + quantise + multiply, in a graph: 200 x 1088 x 1088 6.3 / 8.8 us, 480 x
// 1088 x 1088 8.6 / 8.9, 200 x 1003 x 333 7.8 / 10.6, 4000 x 1088 x 51 6.4 / 13.5;
// beyond the limit 512 x 1088 x 1088 11.4 / 9.1; with rows of 4032 read twice 30 / 16.
bool mid(int64_t tokens, int64_t k, int64_t n) {
  return !fused(tokens, k) && k <= 1536 && (tokens + 15) / 16 * ((n + 63) / 64) <= 512;
}

// Many tokens, two workgroups' integers in a CU's LDS (K up to 1216), weights at
// 32-bit offsets.
bool group(int64_t tokens, int64_t k, int64_t n) {
  return tokens >= kGroupTokens && pad64(k) * kGroup <= kGroupLds && pad64(n) * pad64(k) < 0x40000000;
}

// Tokens of one quantise + multiply round: their integers stay below 1 GiB, which
// 32-bit offsets reach.
int64_t round_tokens(int64_t tokens, int64_t k) { return std::min(tokens, std::max<int64_t>(256, ((int64_t)1 << 30) / pad64(k) / 256 * 256)); }

template <int T>
void launch_int8_t(Int8Args a, void* workspace, hipStream_t s) {
  const int64_t kp = pad64(a.k), most = round_tokens(a.tokens, a.k);
  char* p = (char*)workspace;
  float* qs = (float*)p;
  p += pad256(most * 4);
  int8_t* q = (int8_t*)p;
  p += pad256(most * kp);
  int8_t* wp = (int8_t*)p;
  Int8Gemm g{};
  g.q = q; g.qs = qs; g.kp = kp;
  g.w = a.w; g.w_row = a.w_row; g.w_panel = 64;
  g.w_bytes = (int64_t)(a.n - 1) * a.w_row + a.k;
  g.ws = a.w_scale; g.bias = a.bias;
  g.out = a.out; g.out_row = a.out_row;
  g.tokens = a.tokens; g.n = a.n;
  if (mid(a.tokens, a.k, a.n)) {
    const dim3 grid((unsigned)((a.tokens + 15) / 16), (unsigned)((a.n + 63) / 64));
    hipLaunchKernelGGL((int8_mid_kernel<T>), grid, dim3(64 * kMidWaves), (unsigned)(16 * (kp + 16)), s, g, a.x, a.x_row, a.k);
    return;
  }
  if (a.tokens <= kFewTokens) {
    const dim3 grid((a.n + 15) / 16);
    if (fused(a.tokens, a.k)) {
      hipLaunchKernelGGL((int8_few_kernel<T, true>), grid, dim3(256), (unsigned)(a.tokens * (kp + 16)), s, g, a.x, a.x_row, a.k);
    } else {
      launch_quant_rows<T>(a, kp, q, qs, s);
      hipLaunchKernelGGL((int8_few_kernel<T, false>), grid, dim3(256), 0, s, g, a.x, a.x_row, a.k);
    }
    return;
  }
  if (group(a.tokens, a.k, a.n)) {  // the workspace holds the weights alone
    const int64_t n64 = pad64(a.n);
    int8_t* fragments = (int8_t*)workspace;
    hipLaunchKernelGGL(fragments_kernel, dim3((unsigned)(n64 / 16), (unsigned)(kp / 64)), dim3(256), 0, s, a.w, a.w_row, a.n, a.k, (int)kp, fragments);
    g.w = fragments;
    g.w_bytes = n64 * kp;
    for (int64_t t0 = 0; t0 < a.tokens; t0 += kGroupMost) {
      g.tokens = std::min(kGroupMost, a.tokens - t0);
      g.out = (char*)a.out + t0 * a.out_row * kElem<T>;
      const dim3 grid((unsigned)((g.tokens + kGroup - 1) / kGroup));
      const void* x = (const char*)a.x + t0 * a.x_row * kElem<T>;
      if (a.out_row <= 1 << 22) hipLaunchKernelGGL((int8_group_kernel<T, false>), grid, dim3(256), (unsigned)(kp * kGroup), s, g, x, a.x_row, a.k);
      else hipLaunchKernelGGL((int8_group_kernel<T, true>), grid, dim3(256), (unsigned)(kp * kGroup), s, g, x, a.x_row, a.k);
    }
    return;
  }
  // The weights as panels where many token tiles read them, and where 16-byte
  // loads at 32-bit offsets cannot address their rows (k % 4: the loads' bounds
  // check drops a dword that ends past the last row).
  const bool four = a.k % 4 == 0 && a.w_row % 4 == 0 && (uintptr_t)a.w % 4 == 0;
  if (a.tokens >= kPanelTokens || !four || a.w_row % 16 || (uintptr_t)a.w % 16 || g.w_bytes > 0x7fffffff) {
    const dim3 grid((a.n + 15) / 16, (unsigned)(kp / 64));
    hipLaunchKernelGGL(panels_kernel, grid, dim3(256), 0, s, a.w, a.w_row, a.n, a.k, wp);
    g.w = wp;
    g.w_row = 64;
    g.w_panel = (int64_t)a.n * 64;
    g.w_bytes = a.n * kp;
  }
  for (int64_t t0 = 0; t0 < a.tokens; t0 += most) {
    Int8Args r = a;
    r.tokens = g.tokens = std::min(most, a.tokens - t0);
    r.x = (const char*)a.x + t0 * a.x_row * (T == kOpF32 ? 4 : 2);
    g.out = (char*)a.out + t0 * a.out_row * (T == kOpF32 ? 4 : 2);
    launch_quant_rows<T>(r, kp, q, qs, s);
    const int64_t t256 = (r.tokens + 255) / 256 * ((a.n + 127) / 128), t128 = (r.tokens + 127) / 128 * ((a.n + 127) / 128);
    if (t256 >= 512) launch_tiles<T, 4, 2, 3>(g, s);
    else if (t128 >= 256) launch_tiles<T, 2, 2, 4>(g, s);
    else launch_tiles<T, 1, 1, 8>(g, s);
  }
}

}  // namespace

int64_t int8_workspace(int64_t tokens, int64_t k, int64_t n) {
  if (tokens <= 0 || k <= 0 || n <= 0) return 0;
  if (fused(tokens, k) || mid(tokens, k, n)) return 0;
  if (group(tokens, k, n)) return pad256(pad64(n) * pad64(k));
  const int64_t most = round_tokens(tokens, k);
  return pad256(most * 4) + pad256(most * pad64(k)) + pad256(pad64(n) * pad64(k));
}

void launch_int8(const Int8Args& a, void* workspace, hipStream_t s) {
  if (a.dtype == kOpF32) launch_int8_t<kOpF32>(a, workspace, s);
  else if (a.dtype == kOpBF16) launch_int8_t<kOpBF16>(a, workspace, s);
  else launch_int8_t<kOpF16>(a, workspace, s);
}

void launch_quant_weight(const QuantWArgs& a, hipStream_t s) {
  const dim3 g((a.n + 3) / 4);
  if (a.dtype == kOpF32) hipLaunchKernelGGL((quant_weight_kernel<kOpF32>), g, dim3(256), 0, s, a);
  else if (a.dtype == kOpBF16) hipLaunchKernelGGL((quant_weight_kernel<kOpBF16>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quant_weight_kernel<kOpF16>), g, dim3(256), 0, s, a);
}

}  // namespace lcn
