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
