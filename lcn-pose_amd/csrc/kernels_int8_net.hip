// The hidden layers of a prediction in 8-bit integers (gfx950): z = a . We + b
// (models_att.py:662, :692) with one scale a pose and one an output channel.
//
//   s[b] = max_c |a[b,c]| / 127,   q = rint(a * (127 / max))     every prediction
//   t[n] = max_k |We[k,n]| / 127,  w = rint(We * (127 / max))    from the fp32 blocks
//   z[b,n] = (sum_k q[b,k] w[k,n]) s[b] t[n] + bias[n]
//
// The activations are read from the row tiles (BN apply + LeakyReLU on the way,
// where the layer's input is a z), the result is written to them with the BN
// statistics of the fp32 GEMM's epilogue; absent blocks are skipped as there.
// Bound by memory: a layer of 65 536 poses x 1088 reads 285 MB of activations and
// writes 71 MB of integers (66 us, 72 with BatchNorm: 5.0 to 5.4 TB/s), then reads those
// and writes 285 MB of z (128 us, 2.8 TB/s).  The weights of six layers take 15 us.
#include "gemm_epilogue.h"
#include "ops_common.h"

namespace lcn {

namespace {

__device__ __forceinline__ void see4(float4 v, float& top, bool& bad) {
  const float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
  bad |= !(fabsf(v.x) < __builtin_inff() && fabsf(v.y) < __builtin_inff() && fabsf(v.z) < __builtin_inff() && fabsf(v.w) < __builtin_inff());
  top = fmaxf(top, m);
}

// One row tile (32 poses) a workgroup, its slabs dealt to eight waves; a wave
// keeps up to kKeep slabs in registers between the two passes and reads the
// rest (F > 64) again.  q: panels of 64 features, [slab][rows][64] bytes.
constexpr int kQuantWaves = 8, kKeep = 3;
template <bool kBn>
__global__ __launch_bounds__(64 * kQuantWaves) void quant_tiles_kernel(const float* __restrict__ X, int S, int rows,
                                                                       const float* __restrict__ scale, const float* __restrict__ shift,
                                                                       int spj, float alpha, int8_t* __restrict__ q, float* __restrict__ qs) {
  __shared__ float tops[kQuantWaves][32];
  __shared__ int bads[kQuantWaves][32];
  const int rt = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5, row = lane & 31;
  const float4* x = (const float4*)(X + (size_t)rt * S * 2048);
  auto load = [&](int si, float4 (&v)[8]) {
#pragma unroll
    for (int g = 0; g < 8; ++g) {  // read past the caches: they hold the integers for the product
      const v4f_t u = __builtin_nontemporal_load((const v4f_t*)(x + si * 512 + g * 64 + lane));
      v[g] = make_float4(u.x, u.y, u.z, u.w);
    }
    if constexpr (kBn) {
      const int ch = (si % spj) * kSlab + 4 * h;
#pragma unroll
      for (int g = 0; g < 8; ++g) v[g] = bnact4(v[g], *(const float4*)(scale + ch + 8 * g), *(const float4*)(shift + ch + 8 * g), alpha);
    }
  };
  float top = 0.f;
  bool bad = false;
  float4 keep[kKeep][8];
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (w + kQuantWaves * i < S) load(w + kQuantWaves * i, keep[i]);
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (w + kQuantWaves * i < S)
#pragma unroll
      for (int g = 0; g < 8; ++g) see4(keep[i][g], top, bad);
  for (int si = w + kQuantWaves * kKeep; si < S; si += kQuantWaves) {
    float4 v[8];
    load(si, v);
#pragma unroll
    for (int g = 0; g < 8; ++g) see4(v[g], top, bad);
  }
  top = fmaxf(top, __shfl_xor(top, 32));
  int anybad = bad;
  anybad |= __shfl_xor(anybad, 32);
  if (h == 0) { tops[w][row] = top; bads[w][row] = anybad; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantWaves; ++i) { top = fmaxf(top, tops[i][row]); anybad |= bads[i][row]; }
  bad = anybad != 0;
  float factor, scale_of;
  row_scale(top, bad, factor, scale_of);
  if (w == 0 && h == 0) qs[rt * 32 + row] = scale_of;
  auto put = [&](int si, const float4 (&v)[8]) {
    unsigned d[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) d[g] = quant4(v[g].x, v[g].y, v[g].z, v[g].w, factor, bad);
    // features 8 g + 4 h .. of this lane and its partner (same row, other half):
    // half h stores bytes 32 h .. 32 h + 31 of the row
    unsigned o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned got = __shfl_xor(h ? d[i] : d[4 + i], 32);
      o[2 * i] = h ? got : d[i];
      o[2 * i + 1] = h ? d[4 + i] : got;
    }
    v4u* dst = (v4u*)(q + ((int64_t)si * rows + rt * 32 + row) * 64 + h * 32);
    dst[0] = v4u{o[0], o[1], o[2], o[3]};
    dst[1] = v4u{o[4], o[5], o[6], o[7]};
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (w + kQuantWaves * i < S) put(w + kQuantWaves * i, keep[i]);
  for (int si = w + kQuantWaves * kKeep; si < S; si += kQuantWaves) {
    float4 v[8];
    load(si, v);
    put(si, v);
  }
}

// the 64 output channels of slab blockIdx.x of hidden layer blockIdx.y: every
// present block of the slab's list, [n][k] fragment-packed fp32 -> rows of 64 bytes
__global__ __launch_bounds__(256) void quant_blocks_kernel(const WPrepHidden* __restrict__ items, const int* __restrict__ ptr,
                                                           const int2* __restrict__ idx, int nblk, int H, int8_t* __restrict__ w8,
                                                           float* __restrict__ ws) {
  __shared__ float tops[4][64];
  __shared__ int bads[4][64];
  const int so = blockIdx.x, n = threadIdx.x & 63, part = threadIdx.x >> 6;
  const float4* blocks = (const float4*)items[blockIdx.y].fwd;
  int8_t* out = w8 + (int64_t)blockIdx.y * nblk * 4096;
  const int beg = ptr[so], end = ptr[so + 1];
  // the thread's 16 k of a block: four float4
  auto load = [&](int blk, float4 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = blocks[(int64_t)blk * 1024 + frag_ix(n, 16 * part + 4 * i) / 4];
  };
  float top = 0.f;
  bool bad = false;
  // the blocks of a slab four at a time: their loads in flight together
  for (int e = beg; e < end; e += 4) {
    float4 v[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) load(idx[min(e + u, end - 1)].y, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) see4(v[u][i], top, bad);
  }
  tops[part][n] = top;
  bads[part][n] = bad;
  __syncthreads();
  int anybad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) { top = fmaxf(top, tops[i][n]); anybad |= bads[i][n]; }
  float factor, scale;
  row_scale(top, anybad != 0, factor, scale);
  if (part == 0) ws[blockIdx.y * H + so * 64 + n] = scale;
  for (int e = beg; e < end; e += 4) {
    float4 v[4][4];
    int blk[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      blk[u] = idx[min(e + u, end - 1)].y;
      load(blk[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e + u >= end) break;
      unsigned d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = quant4(v[u][i].x, v[u][i].y, v[u][i].z, v[u][i].w, factor, anybad != 0);
      *(v4u*)(out + (int64_t)blk[u] * 4096 + n * 64 + part * 16) = v4u{d[0], d[1], d[2], d[3]};
    }
  }
}

constexpr int kMaxSlabs = 17 * 512 / 64;  // F is at most 512

#define I8_LDS(SRC, VOFF, SOFF, DST) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(SRC, (__attribute__((address_space(3))) void*)(DST), 16, VOFF, SOFF, 0, 0)

// 128 poses (a row tile a wave) x one output slab, one input slab of the slab's
// list a stage: 8 KB of activations and a 4 KB weight block through a ring of
// three LDS buffers.  Weights on the MFMA's i side, poses on its j side, so the
// accumulator is a row tile's and the fp32 GEMM's epilogue takes it from there.
// A row's four 16-byte units are permuted by its number against bank conflicts.
template <int EPI>
__global__ __launch_bounds__(256) void int8_slab_kernel(GemmArgs a, const int8_t* __restrict__ q, const float* __restrict__ qs,
                                                        const int8_t* __restrict__ w8, const float* __restrict__ ws) {
  static_assert(kGemmWaves == 4, "one row tile a wave");
  constexpr int kStage = 12288, R = 3, L = 3;
  __shared__ __attribute__((aligned(16))) char l0[kStage], l1[kStage], l2[kStage];
  __shared__ __attribute__((aligned(16))) float4 red[2048];
  __shared__ float comb[4 * 64 * 3];
  __shared__ int2 list[kMaxSlabs];
  const int nso = a.n_out_slabs;
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int rtg = id / nso, so = id - rtg * nso;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, l31 = lane & 31;
  const int rt_raw = rtg * 4 + w;
  const bool live = rt_raw < a.n_rt;
  const int rt = live ? rt_raw : a.n_rt - 1;  // waves past the last row tile recompute it
  const int rows = a.n_rt * 32;
  const int beg = a.ptr[so], nk = a.ptr[so + 1] - beg;
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)w8, 0, a.n_blocks * 4096, 0x00020000);
  // lane: row lane / 4 of 16, 16-byte unit lane % 4
  const int r16 = lane >> 2, u16 = ((lane & 3) ^ ((r16 >> 2) & 3)) * 16;
  const int vo = r16 * 64 + u16;
  // the slab's list in LDS: from memory an entry would queue behind the stages' loads
  for (int e = threadIdx.x; e < nk; e += 256) list[e] = a.idx[beg + e];
  __syncthreads();
  int ahead = 0;  // entry of the next stage to load
  int2 entry = list[0];
  auto stage = [&](char* buf) {
    const int si = __builtin_amdgcn_readfirstlane(entry.x), blk = __builtin_amdgcn_readfirstlane(entry.y);
    entry = list[min(++ahead, nk - 1)];
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(q + ((int64_t)si * rows + rt * 32) * 64), 0, 2048, 0x00020000);
    I8_LDS(rq, vo, 0, buf + w * 2048);
    I8_LDS(rq, vo, 1024, buf + w * 2048 + 1024);
    I8_LDS(rw, vo, blk * 4096 + w * 1024, buf + 8192 + w * 1024);
  };
  v16i acc0 = {}, acc1 = {};
  struct Frag { v4i p0, p1, q; };
  const int fo = l31 * 64, fx = (l31 >> 2) & 3;
  auto fetch = [&](const char* buf, int kk, Frag& f) {
    const int c = fo + ((2 * kk + h) ^ fx) * 16;
    f.q = *(const v4i*)(buf + w * 2048 + c);
    f.p0 = *(const v4i*)(buf + 8192 + c);
    f.p1 = *(const v4i*)(buf + 8192 + 2048 + c);
  };
  auto multiply = [&](const Frag& f) {
    acc0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.p0, f.q, acc0, 0, 0, 0);
    acc1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.p1, f.q, acc1, 0, 0, 0);
  };
  Frag f0, f1;
  // as in the tiled int8 product: past the barrier the next stage has landed and
  // every wave holds the rest of this one in registers
  auto step = [&](char* mine, const char* after, bool more, bool load) {
    fetch(mine, 1, f1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(f0);
    if (more) {
      if (load) stage_barrier<(R - 2) * L>();
      else stage_barrier<0>();
      if (load) stage(mine);
      fetch(after, 0, f0);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(f1);
  };
  // (every output slab has at least one input block)
  stage(l0);
  if (nk > 1) stage(l1);
  if (nk > 2) stage(l2);
  stage_barrier<0>();
  fetch(l0, 0, f0);
  for (int ks = 0; ks < nk; ks += R) {
    const int left = nk - ks;
    step(l0, l1, left > 1, left > 3);
    if (left > 1) step(l1, l2, left > 2, left > 4);
    if (left > 2) step(l2, l0, left > 3, left > 5);
  }
  const float sq = qs[rt * 32 + l31];
  const float* wsc = ws + so * 64;
  f32x16 v0, v1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float4 t0 = *(const float4*)(wsc + 8 * k + 4 * h), t1 = *(const float4*)(wsc + 32 + 8 * k + 4 * h);
    const float4 b0 = a.bias ? *(const float4*)(a.bias + so * 64 + 8 * k + 4 * h) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 b1 = a.bias ? *(const float4*)(a.bias + so * 64 + 32 + 8 * k + 4 * h) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float s0[4] = {t0.x, t0.y, t0.z, t0.w}, s1[4] = {t1.x, t1.y, t1.z, t1.w};
    const float c0[4] = {b0.x, b0.y, b0.z, b0.w}, c1[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v0[4 * k + e] = (float)acc0[4 * k + e] * sq * s0[e] + c0[e];
      v1[4 * k + e] = (float)acc1[4 * k + e] * sq * s1[e] + c1[e];
    }
  }
  gemm_epilogue<EPI>(a, red, nullptr, comb, rtg, rt, live, so, v0, v1);
}

}  // namespace

void launch_quant_tiles(const float* X, int S, int B, const float* scale, const float* shift, int F, float alpha, int8_t* q,
                        float* qs, hipStream_t s) {
  const int n_rt = (B + kRT - 1) / kRT, spj = F / kSlab;
  if (scale)
    hipLaunchKernelGGL(quant_tiles_kernel<true>, dim3(n_rt), dim3(64 * kQuantWaves), 0, s, X, S, n_rt * kRT, scale, shift, spj, alpha, q, qs);
  else
    hipLaunchKernelGGL(quant_tiles_kernel<false>, dim3(n_rt), dim3(64 * kQuantWaves), 0, s, X, S, n_rt * kRT, scale, shift, spj, alpha, q, qs);
}

void launch_quant_blocks(const WPrepHidden* items, int n_layers, int nslab, const int* ptr, const int2* idx, int nblk, int8_t* w8,
                         float* ws, hipStream_t s) {
  if (n_layers <= 0) return;
  hipLaunchKernelGGL(quant_blocks_kernel, dim3(nslab, n_layers), dim3(256), 0, s, items, ptr, idx, nblk, nslab * kSlab, w8, ws);
}

void launch_int8_slabs(const GemmArgs& a, const int8_t* q, const float* qs, const int8_t* w8, const float* ws, hipStream_t s) {
  const int grid = (a.n_rt + 3) / 4 * a.n_out_slabs;
  if (a.epi_mode == EPI_BNFWD) hipLaunchKernelGGL(int8_slab_kernel<EPI_BNFWD>, dim3(grid), dim3(256), 0, s, a, q, qs, w8, ws);
  else hipLaunchKernelGGL(int8_slab_kernel<EPI_NONE>, dim3(grid), dim3(256), 0, s, a, q, qs, w8, ws);
}

}  // namespace lcn
