// Matrix product in 8-bit integers with one scale a token and one a channel
// (gfx950): the activations are quantised on the way in, the weights once.
//
//   s[t] = max_k |x[t,k]| / 127,   q[t,k] = rint(x[t,k] * (127 / max_k |x[t,k]|))
//   y[t,n] = (sum_k q[t,k] w[n,k]) * s[t] * sw[n] + bias[n]
//
// A row whose largest magnitude is below 2^-100 counts as zero (127 / max would
// overflow); a row that holds an infinity or a NaN gives NaN throughout: its
// scale is NaN and its integers are zero.  The sums are exact (int32, K <= 131072).
#include <algorithm>

#include "ops_common.h"

namespace lcn {

namespace {

__host__ __device__ inline int64_t pad64(int64_t v) { return (v + 63) / 64 * 64; }
__host__ __device__ inline int64_t pad256(int64_t v) { return (v + 255) / 256 * 256; }

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100

// the factor 127 / top of a row and its scale, from the largest magnitude
__device__ __forceinline__ void row_scale(float top, bool bad, float& factor, float& scale) {
  factor = !bad && top >= kTiny ? 127.f / top : 0.f;
  scale = bad ? __builtin_nanf("") : top >= kTiny ? top / 127.f : 0.f;
}
__device__ __forceinline__ int quant(float v, float factor) {
  const float r = rintf(v * factor);
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// one wave a row: largest magnitude, then the integers, rows padded to kp with zeros
template <int T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* __restrict__ x, int64_t x_row, int64_t tokens, int k,
                                                         int64_t kp, int8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= tokens) return;
  float top = 0.f;
  bool bad = false;
  for (int c = lane; c < k; c += 64) {
    const float v = fabsf(op_load<T>(x, t * x_row + c));
    bad |= !(v < __builtin_inff());
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  bad = __any(bad);
  float factor, s;
  row_scale(top, bad, factor, s);
  if (lane == 0) scale[t] = s;
  for (int64_t c = lane; c < kp; c += 64)
    q[t * kp + c] = c < k && !bad ? (int8_t)quant(op_load<T>(x, t * x_row + c), factor) : (int8_t)0;
}

// weight rows of any alignment -> rows of kp bytes, zero padded
__global__ __launch_bounds__(256) void repack_kernel(const int8_t* __restrict__ w, int64_t w_row, int k, int64_t kp,
                                                     int8_t* __restrict__ out) {
  const int64_t n = blockIdx.x;
  for (int64_t c = threadIdx.x; c < kp; c += 256) out[n * kp + c] = c < k ? w[n * w_row + c] : (int8_t)0;
}

#define I8_LDS(SRC, VOFF, SOFF, DST) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(SRC, (__attribute__((address_space(3))) void*)(DST), 16, VOFF, SOFF, 0, 0)

struct Int8Gemm {
  const int8_t* q; const float* qs; int64_t kp;    // [tokens][kp], [tokens]
  const int8_t* w; int64_t w_row, kw;              // rows of kw bytes (a multiple of 4), 16-byte aligned
  const float* ws; const float* bias;
  void* out; int64_t out_row;
  int64_t tokens; int n;
  int tn;                                          // channel tiles
};

// 128 tokens x 128 channels, four waves of 64 x 64, 64 bytes of K a stage
// through a double LDS buffer.  A stage holds rows of 64 bytes (four 16-byte
// units); unit c of row r sits at c ^ ((r >> 2) & 3), so the 32 rows of a
// fragment read spread over all banks; the permutation is made by the lane's
// choice of global address.
template <int T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void int8_gemm_kernel(Int8Gemm g) {
  __shared__ __attribute__((aligned(16))) char lds[2 * 16384];
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t t0 = (int64_t)(id / g.tn) * 128;
  const int n0 = (id % g.tn) * 128;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = w >> 1, wj = w & 1, h = lane >> 5, l31 = lane & 31;
  // rows past the end repeat the last one; their results are not stored
  const int trows = (int)min((int64_t)128, g.tokens - t0), nrows = min(128, g.n - n0);
  const int64_t qbytes = (int64_t)trows * g.kp, wbytes = (int64_t)(nrows - 1) * g.w_row + g.kw;
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(g.q + t0 * g.kp), 0, (int)qbytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(g.w + n0 * g.w_row), 0, (int)wbytes, 0x00020000);
  int voq[2], vow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = w * 32 + i * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 2) & 3);
    voq[i] = min(r, trows - 1) * (int)g.kp + c * 16;
    vow[i] = min(r, nrows - 1) * (int)g.w_row + c * 16;
  }
  auto stage = [&](int ks, int buf) {
    char* d = lds + buf * 16384 + w * 2048;
    const int so = ks * 64;
    I8_LDS(rq, voq[0], so, d);        I8_LDS(rq, voq[1], so, d + 1024);
    I8_LDS(rw, vow[0], so, d + 8192); I8_LDS(rw, vow[1], so, d + 8192 + 1024);
  };
  v16i acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0;
  const int nk = (int)(g.kp / 64);
  stage(0, 0);
  __syncthreads();
  for (int ks = 0; ks < nk; ++ks) {
    const char* s = lds + (ks & 1) * 16384;
    v4i p[2][2], q[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int rp = wi * 64 + x * 32 + l31, rw_ = wj * 64 + x * 32 + l31, c = (2 * kk + h) ^ ((l31 >> 2) & 3);
        p[x][kk] = *(const v4i*)(s + rp * 64 + c * 16);
        q[x][kk] = *(const v4i*)(s + 8192 + rw_ * 64 + c * 16);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (ks + 1 < nk) stage(ks + 1, (ks + 1) & 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(p[x][kk], q[y][kk], acc[x][y], 0, 0, 0);
    __syncthreads();
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int n = n0 + wj * 64 + y * 32 + l31;
    if (n >= g.n) continue;
    const float sw = g.ws[n], b = g.bias ? g.bias[n] : 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t t = t0 + wi * 64 + x * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
        if (t >= g.tokens) continue;
        float v = (float)acc[x][y][e] * g.qs[t] * sw;
        if (g.bias) v += b;
        op_store<T>(g.out, t * g.out_row + n, v);
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
    a.q[(int64_t)n * a.k + c] = bad ? (int8_t)0 : (int8_t)quant(op_load<T>(a.w, n * a.w_n + c * a.w_k), factor);
}

template <int T>
void launch_int8_t(const Int8Args& a, void* workspace, hipStream_t s) {
  const int64_t kp = pad64(a.k);
  char* p = (char*)workspace;
  float* qs = (float*)p;
  p += pad256(a.tokens * 4);
  int8_t* q = (int8_t*)p;
  p += pad256(a.tokens * kp);
  int8_t* wp = (int8_t*)p;
  hipLaunchKernelGGL((quant_rows_kernel<T>), dim3((unsigned)((a.tokens + 3) / 4)), dim3(256), 0, s, a.x, a.x_row, a.tokens, a.k, kp, q, qs);
  Int8Gemm g{};
  g.q = q; g.qs = qs; g.kp = kp;
  g.w = a.w; g.w_row = a.w_row; g.kw = a.k;
  // rows that 16-byte loads at 32-bit offsets cannot address are laid out again
  // (k % 4: the loads' bounds check drops a dword that ends past the last row)
  if (a.k % 4 || a.w_row % 16 || (uintptr_t)a.w % 16 || a.w_row > (1 << 20)) {
    hipLaunchKernelGGL(repack_kernel, dim3(a.n), dim3(256), 0, s, a.w, a.w_row, a.k, kp, wp);
    g.w = wp;
    g.w_row = g.kw = kp;
  }
  g.ws = a.w_scale; g.bias = a.bias;
  g.out = a.out; g.out_row = a.out_row;
  g.tokens = a.tokens; g.n = a.n;
  g.tn = (a.n + 127) / 128;
  hipLaunchKernelGGL((int8_gemm_kernel<T>), dim3((unsigned)((a.tokens + 127) / 128 * g.tn)), dim3(256), 0, s, g);
}

}  // namespace

int64_t int8_workspace(int64_t tokens, int64_t k, int64_t n) {
  if (tokens <= 0 || k <= 0 || n <= 0) return 0;
  return pad256(tokens * 4) + pad256(tokens * pad64(k)) + pad256(n * pad64(k));
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
