// Launch interface of the operators that work on weights and activations
// outside a training step's own schedule: Newton-Schulz orthogonalisation, the
// Muon update and the int8 product.  gfx950 only.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lcn {

// element types of the operators' operands; kF32 / kF64 are lcn_internal.h's 0 / 1
enum { kOpF32 = 0, kOpBF16 = 2, kOpF16 = 3 };

// batch x rows x cols matrices with a contiguous last dimension:
// element (b, r, c) at p + b * batch + r * row + c (in elements)
struct MatView {
  void* p;
  int64_t batch, row;
};

struct NsArgs {
  int64_t batch;
  int rows, cols;
  int steps;
  float a, b, c;            // X <- a X + (b A + c A A) X,  A = X X^T
  float eps;
  int dtype;                // of `in` (the gradient of muon)
  MatView in;
  int out_dtype;            // orthogonalize: type of `out`
  MatView out;              // orthogonalize: the result; muon: the parameter (fp32, updated in place)
  // muon (momentum.p != null): buf = beta buf + g; u = g + beta buf (nesterov) or buf;
  // W = (1 - lr decay) W - lr scale NS(u), lr = lr_dev ? *lr_dev : lr
  MatView momentum;
  float beta;
  int nesterov;
  float lr, scale, decay;
  const float* lr_dev;
};
int64_t ns_workspace(int64_t batch, int64_t rows, int64_t cols);
void launch_ns(const NsArgs& a, void* workspace, hipStream_t s);

struct Int8Args {
  int64_t tokens;
  int k, n;
  int dtype;                // of x and out
  const void* x; int64_t x_row;
  const int8_t* w; int64_t w_row;
  const float* w_scale;     // [n]
  const float* bias;        // [n] or null
  void* out; int64_t out_row;
};
int64_t int8_workspace(int64_t tokens, int64_t k, int64_t n);
void launch_int8(const Int8Args& a, void* workspace, hipStream_t s);

constexpr int64_t kInt8MaxK = 131072;  // 127 * 127 * K stays below 2^31

struct QuantWArgs {
  int n, k;
  int dtype;
  const void* w; int64_t w_n, w_k;   // element strides along channel and reduction
  int8_t* q;                         // [n][k]
  float* scale;                      // [n]
};
void launch_quant_weight(const QuantWArgs& a, hipStream_t s);

}  // namespace lcn
