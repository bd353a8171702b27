// Device helpers of the operator kernels (gfx950).
#pragma once
#include "gemm_common.h"
#include "lcn_ops.h"

namespace lcn {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// element e of a kOpF32 / kOpBF16 / kOpF16 array as float, and back (round to nearest even)
template <int T>
__device__ __forceinline__ float op_load(const void* p, int64_t e) {
  if constexpr (T == kOpF32) return ((const float*)p)[e];
  else if constexpr (T == kOpBF16) return __uint_as_float((unsigned)((const unsigned short*)p)[e] << 16);
  else return (float)((const _Float16*)p)[e];
}
template <int T>
__device__ __forceinline__ void op_store(void* p, int64_t e, float v) {
  if constexpr (T == kOpF32) ((float*)p)[e] = v;
  else if constexpr (T == kOpBF16) ((__bf16*)p)[e] = (__bf16)v;
  else ((_Float16*)p)[e] = (_Float16)v;
}

// 16 bytes of a row as floats: 4 of fp32, 8 of the 16-bit types
template <int T> constexpr int kVec = T == kOpF32 ? 4 : 8;
template <int T>
__device__ __forceinline__ void unpack_vec(v4u u, float (&v)[kVec<T>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == kOpF32) v[i] = __uint_as_float(u[i]);
    else if constexpr (T == kOpBF16) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    else {
      v[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)u[i]);
      v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(u[i] >> 16));
    }
  }
}

// ---- int8 quantisation of a row --------------------------------------------------------------
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100: a row below it counts as zero

// the factor 127 / top of a row and its scale, from the largest magnitude
__device__ __forceinline__ void row_scale(float top, bool bad, float& factor, float& scale) {
  factor = !bad && top >= kTiny ? 127.f / top : 0.f;
  scale = bad ? __builtin_nanf("") : top >= kTiny ? top / 127.f : 0.f;
}
// rint(v factor) in the low byte.  |v factor| <= 127 (1 + 2^-22), which rounds to
// 127: no clamp.  Adding 1.5 2^23 rounds to the nearest integer, ties to even.
__device__ __forceinline__ unsigned quant_bits(float v, float factor) {
#pragma clang fp contract(off)  // the product is rounded before the sum
  return __float_as_uint(v * factor + 12582912.f);
}
__device__ __forceinline__ int8_t quant(float v, float factor) { return (int8_t)quant_bits(v, factor); }
// four integers as bytes, zeros for a bad row
__device__ __forceinline__ unsigned quant4(float a, float b, float c, float d, float factor, bool bad) {
  const unsigned lo = __builtin_amdgcn_perm(quant_bits(b, factor), quant_bits(a, factor), 0x0c0c0400);
  const unsigned hi = __builtin_amdgcn_perm(quant_bits(d, factor), quant_bits(c, factor), 0x04000c0c);
  return bad ? 0u : lo | hi;
}

// Waits until at most N of this wave's vector loads are outstanding and all its
// LDS reads have returned, then for the other waves of the workgroup.  Nothing
// that touches memory moves across.
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

}  // namespace lcn
