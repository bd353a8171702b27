// C entry points of the handle-free device operators: lcn_orthogonalize,
// lcn_muon_update, lcn_int8_linear, lcn_int8_quantize_weight.  Every argument
// is checked here before anything is launched; the kernels run on the caller's
// stream with the caller's workspace, so two calls never share memory of the
// library's, and a call can be captured into a graph.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "../../include/lcn.h"
#include "lcn_internal.h"
#include "lcn_ops.h"

using namespace lcn;

namespace {

int fail(const char* who, const std::string& what, int code = LCN_E_ARG) {
  set_global_error(std::string(who) + ": " + what);
  return code;
}

// The operator runs on `device`; the calling thread's current device is put back.
// HIP keeps a thread's last error until it is asked for: what an earlier call left
// (or a refused device, here) is taken away, so that `launched` sees the launches only.
struct DeviceGuard {
  int before = -1;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else before = -1;
    (void)hipGetLastError();
  }
  ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
};

int elem_bytes(int dtype) { return dtype == LCN_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == LCN_DTYPE_F32 || dtype == LCN_DTYPE_BF16 || dtype == LCN_DTYPE_F16; }

// batch x rows x cols elements of `bytes`, last dimension contiguous
struct View {
  const void* p;
  int64_t batch, rows, cols, s_batch, s_row;
  int bytes;
  uint64_t begin() const { return (uint64_t)(uintptr_t)p; }
  uint64_t end() const { return begin() + (uint64_t)((batch - 1) * s_batch + (rows - 1) * s_row + cols) * bytes; }
};

// elements past 2^46 cannot be addressed; keeps the products below from overflowing
constexpr int64_t kMaxStride = (int64_t)1 << 46;

// strides of an operand that is only read: any that are not negative
bool readable(const View& v) {
  return v.s_batch >= 0 && v.s_row >= 0 && v.s_batch <= kMaxStride / v.batch && v.s_row <= kMaxStride / v.rows;
}
// strides of an operand that is written: no element twice
bool writable(const View& v) {
  if (!readable(v)) return false;
  if (v.rows > 1 && v.s_row < v.cols) return false;
  return v.batch == 1 || v.s_batch >= (v.rows - 1) * v.s_row + v.cols ||
         (v.s_batch >= v.cols && v.rows > 1 && v.s_row >= (v.batch - 1) * v.s_batch + v.cols);
}
bool aligned(const View& v) { return v.begin() % v.bytes == 0; }

// Whether two operands may share an element.  Address ranges that meet still
// do not where both are columns of the same rows (slices of one buffer).
bool overlap(const View& a, const View& b) {
  if (a.begin() >= b.end() || b.begin() >= a.end()) return false;
  const uint64_t ra = (uint64_t)a.s_row * a.bytes, rb = (uint64_t)b.s_row * b.bytes;
  if (ra && ra == rb && (a.batch == 1 || (uint64_t)a.s_batch * a.bytes % ra == 0) &&
      (b.batch == 1 || (uint64_t)b.s_batch * b.bytes % rb == 0)) {
    const uint64_t wa = (uint64_t)a.cols * a.bytes, wb = (uint64_t)b.cols * b.bytes;
    // b's columns relative to a's, within one row
    const uint64_t d = a.begin() <= b.begin() ? (b.begin() - a.begin()) % ra : (ra - (a.begin() - b.begin()) % ra) % ra;
    if (d >= wa && d + wb <= ra) return false;
  }
  return true;
}
bool same_place(const View& a, const View& b) {
  return a.p == b.p && a.bytes == b.bytes && (a.batch == 1 || a.s_batch == b.s_batch) && (a.rows == 1 || a.s_row == b.s_row);
}
// (a null block: the call needs none)
bool in_block(const View& v, const void* block, int64_t bytes) {
  if (!block) return false;
  const uint64_t b = (uint64_t)(uintptr_t)block;
  return v.begin() < b + (uint64_t)bytes && b < v.end();
}

int ns_sizes(const char* who, int64_t batch, int64_t rows, int64_t cols) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(who, "negative size");
  if (batch > 65535) return fail(who, "batch " + std::to_string(batch) + " > 65535");
  if (rows > 65536 || cols > 65536 || (rows + 31) * (cols + 31) > ((int64_t)1 << 30))
    return fail(who, "a matrix of " + std::to_string(rows) + " x " + std::to_string(cols) + " is too large (sides <= 65536, 2^30 elements)");
  const int64_t tiles = ((rows + 31) / 32) * ((cols + 31) / 32);
  if (batch * tiles > ((int64_t)1 << 23)) return fail(who, "batch x matrix too large (2^33 elements)");
  return LCN_OK;
}
int ns_iteration(const char* who, int32_t steps, const float* c, float eps) {
  if (steps < 1 || steps > 64) return fail(who, "steps " + std::to_string(steps) + " outside [1, 64]");
  if (!c || !std::isfinite(c[0]) || !std::isfinite(c[1]) || !std::isfinite(c[2])) return fail(who, "coefficients must be three finite numbers");
  if (!(eps >= 1e-30f) || !std::isfinite(eps)) return fail(who, "eps must be a finite number >= 1e-30");
  return LCN_OK;
}
int check_workspace(const char* who, const void* ws, int64_t bytes, int64_t need) {
  if (need == 0) return LCN_OK;
  if (!ws) return fail(who, "null workspace");
  if ((uintptr_t)ws % 256) return fail(who, "the workspace must be 256-byte aligned");
  if (bytes < need) return fail(who, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
  return LCN_OK;
}
int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LCN_OK : fail(who, hipGetErrorString(e), LCN_E_HIP);
}

#define OP_CHECK(expr)                    \
  do {                                    \
    const int rc_ = (expr);               \
    if (rc_ != LCN_OK) return rc_;        \
  } while (0)
// no C++ exception leaves a C entry
#define OP_BEGIN(WHO)                     \
  static const char* who = WHO;           \
  try {                                   \
    set_global_error("");
#define OP_END                                                                   \
  }                                                                              \
  catch (const std::exception&) { return LCN_E_NOMEM; }                          \
  catch (...) { return LCN_E_STATE; }

}  // namespace

extern "C" {

int64_t lcn_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
  OP_BEGIN("lcn_orthogonalize_workspace")
  OP_CHECK(ns_sizes(who, batch, rows, cols));
  return ns_workspace(batch, rows, cols);
  OP_END
}

int lcn_orthogonalize(int32_t device, void* stream, int32_t dtype, int64_t batch, int64_t rows, int64_t cols,
                      const void* in, int64_t in_batch, int64_t in_row, void* out, int64_t out_batch, int64_t out_row,
                      int32_t steps, const float* coefficients, float eps, void* workspace, int64_t workspace_bytes) {
  OP_BEGIN("lcn_orthogonalize")
  OP_CHECK(ns_sizes(who, batch, rows, cols));
  OP_CHECK(ns_iteration(who, steps, coefficients, eps));
  if (!known_dtype(dtype)) return fail(who, "dtype must be LCN_DTYPE_F32, _BF16 or _F16");
  if (batch == 0 || rows == 0 || cols == 0) return LCN_OK;
  if (!in || !out) return fail(who, "null operand");
  const View vi{in, batch, rows, cols, in_batch, in_row, elem_bytes(dtype)}, vo{out, batch, rows, cols, out_batch, out_row, elem_bytes(dtype)};
  if (!readable(vi)) return fail(who, "bad strides of the input");
  if (!writable(vo)) return fail(who, "the output's strides let elements overlap");
  if (!aligned(vi) || !aligned(vo)) return fail(who, "operand not aligned to its type");
  if (overlap(vi, vo) && !same_place(vi, vo)) return fail(who, "the output overlaps the input (it may be the input itself)");
  OP_CHECK(check_workspace(who, workspace, workspace_bytes, ns_workspace(batch, rows, cols)));
  if (in_block(vi, workspace, workspace_bytes) || in_block(vo, workspace, workspace_bytes)) return fail(who, "the workspace overlaps an operand");
  DeviceGuard dev(device);
  if (dev.err != hipSuccess) return fail(who, hipGetErrorString(dev.err), LCN_E_HIP);
  NsArgs a{};
  a.batch = batch;
  a.rows = (int)rows;
  a.cols = (int)cols;
  a.steps = steps;
  a.a = coefficients[0];
  a.b = coefficients[1];
  a.c = coefficients[2];
  a.eps = eps;
  a.dtype = a.out_dtype = dtype;
  a.in = MatView{(void*)in, in_batch, in_row};
  a.out = MatView{out, out_batch, out_row};
  launch_ns(a, workspace, (hipStream_t)stream);
  return launched(who);
  OP_END
}

int lcn_muon_update(int32_t device, void* stream, int32_t grad_dtype, int64_t batch, int64_t rows, int64_t cols,
                    float* param, int64_t param_batch, int64_t param_row, float* momentum, int64_t momentum_batch,
                    int64_t momentum_row, const void* grad, int64_t grad_batch, int64_t grad_row, float lr,
                    const float* lr_dev, float scale, float beta, int32_t nesterov, float weight_decay, int32_t steps,
                    const float* coefficients, float eps, void* workspace, int64_t workspace_bytes) {
  OP_BEGIN("lcn_muon_update")
  OP_CHECK(ns_sizes(who, batch, rows, cols));
  OP_CHECK(ns_iteration(who, steps, coefficients, eps));
  if (!known_dtype(grad_dtype)) return fail(who, "grad_dtype must be LCN_DTYPE_F32, _BF16 or _F16");
  if ((!lr_dev && !std::isfinite(lr)) || !std::isfinite(scale) || !std::isfinite(weight_decay)) return fail(who, "lr, scale and weight_decay must be finite");
  if (!(beta >= 0.f && beta < 1.f)) return fail(who, "beta must be in [0, 1)");
  if (batch == 0 || rows == 0 || cols == 0) return LCN_OK;
  if (!param || !momentum || !grad) return fail(who, "null operand");
  const View vp{param, batch, rows, cols, param_batch, param_row, 4}, vm{momentum, batch, rows, cols, momentum_batch, momentum_row, 4},
      vg{grad, batch, rows, cols, grad_batch, grad_row, elem_bytes(grad_dtype)};
  if (!readable(vg)) return fail(who, "bad strides of the gradient");
  if (!writable(vp) || !writable(vm)) return fail(who, "the strides of the parameter or the momentum let elements overlap");
  if (!aligned(vp) || !aligned(vm) || !aligned(vg) || (uintptr_t)lr_dev % 4) return fail(who, "operand not aligned to its type");
  if (overlap(vp, vm) || overlap(vp, vg) || overlap(vm, vg)) return fail(who, "param, momentum and grad must not overlap");
  if (lr_dev) {  // read while param and momentum are written
    const View vl{lr_dev, 1, 1, 1, 0, 1, 4};
    if (overlap(vp, vl) || overlap(vm, vl) || in_block(vl, workspace, workspace_bytes)) return fail(who, "lr_dev lies in an operand or the workspace");
  }
  OP_CHECK(check_workspace(who, workspace, workspace_bytes, ns_workspace(batch, rows, cols)));
  if (in_block(vp, workspace, workspace_bytes) || in_block(vm, workspace, workspace_bytes) || in_block(vg, workspace, workspace_bytes))
    return fail(who, "the workspace overlaps an operand");
  DeviceGuard dev(device);
  if (dev.err != hipSuccess) return fail(who, hipGetErrorString(dev.err), LCN_E_HIP);
  NsArgs a{};
  a.batch = batch;
  a.rows = (int)rows;
  a.cols = (int)cols;
  a.steps = steps;
  a.a = coefficients[0];
  a.b = coefficients[1];
  a.c = coefficients[2];
  a.eps = eps;
  a.dtype = grad_dtype;
  a.out_dtype = LCN_DTYPE_F32;
  a.in = MatView{(void*)grad, grad_batch, grad_row};
  a.out = MatView{param, param_batch, param_row};
  a.momentum = MatView{momentum, momentum_batch, momentum_row};
  a.beta = beta;
  a.nesterov = nesterov != 0;
  a.lr = lr;
  a.lr_dev = lr_dev;
  a.scale = scale;
  a.decay = weight_decay;
  launch_ns(a, workspace, (hipStream_t)stream);
  return launched(who);
  OP_END
}

static int int8_sizes(const char* who, int64_t tokens, int64_t k, int64_t n) {
  if (tokens < 0 || k < 0 || n < 0) return fail(who, "negative size");
  if (k > kInt8MaxK) return fail(who, "k " + std::to_string(k) + " > 131072 (a 32-bit sum could overflow)");
  if (n > ((int64_t)1 << 24) || tokens > ((int64_t)1 << 30)) return fail(who, "too many channels (2^24) or tokens (2^30)");
  if (((tokens + 127) / 128) * ((n + 127) / 128) > ((int64_t)1 << 23)) return fail(who, "tokens x channels too large (2^37)");
  if (n * (k + 63) > ((int64_t)1 << 31) - 64) return fail(who, "weight too large (2^31 bytes)");
  return LCN_OK;
}

int64_t lcn_int8_linear_workspace(int64_t tokens, int64_t k, int64_t n) {
  OP_BEGIN("lcn_int8_linear_workspace")
  OP_CHECK(int8_sizes(who, tokens, k, n));
  return int8_workspace(tokens, k, n);
  OP_END
}

int lcn_int8_linear(int32_t device, void* stream, int32_t dtype, int64_t tokens, int64_t k, int64_t n, const void* x,
                    int64_t x_row, const int8_t* weight, int64_t weight_row, const float* weight_scale, const float* bias,
                    void* out, int64_t out_row, void* workspace, int64_t workspace_bytes) {
  OP_BEGIN("lcn_int8_linear")
  OP_CHECK(int8_sizes(who, tokens, k, n));
  if (!known_dtype(dtype)) return fail(who, "dtype must be LCN_DTYPE_F32, _BF16 or _F16");
  if (tokens == 0 || n == 0) return LCN_OK;
  if (k == 0) return fail(who, "k is zero");
  if (!x || !weight || !weight_scale || !out) return fail(who, "null operand");
  const View vx{x, 1, tokens, k, 0, x_row, elem_bytes(dtype)}, vw{weight, 1, n, k, 0, weight_row, 1}, vo{out, 1, tokens, n, 0, out_row, elem_bytes(dtype)},
      vs{weight_scale, 1, 1, n, 0, n, 4}, vb{bias, 1, 1, n, 0, n, 4};
  if (!readable(vx) || !readable(vw)) return fail(who, "bad strides of an input");
  if (!writable(vo)) return fail(who, "the output's rows overlap");
  if (!aligned(vx) || !aligned(vo) || !aligned(vs) || (bias && !aligned(vb))) return fail(who, "operand not aligned to its type");
  if (overlap(vo, vx) || overlap(vo, vw) || overlap(vo, vs) || (bias && overlap(vo, vb))) return fail(who, "the output overlaps an input");
  const int64_t need = int8_workspace(tokens, k, n);
  OP_CHECK(check_workspace(who, workspace, workspace_bytes, need));
  for (const View* v : {&vx, &vw, &vo, &vs, &vb})
    if (v->p && in_block(*v, workspace, workspace_bytes)) return fail(who, "the workspace overlaps an operand");
  DeviceGuard dev(device);
  if (dev.err != hipSuccess) return fail(who, hipGetErrorString(dev.err), LCN_E_HIP);
  Int8Args a{};
  a.tokens = tokens;
  a.k = (int)k;
  a.n = (int)n;
  a.dtype = dtype;
  a.x = x;
  a.x_row = x_row;
  a.w = weight;
  a.w_row = weight_row;
  a.w_scale = weight_scale;
  a.bias = bias;
  a.out = out;
  a.out_row = out_row;
  launch_int8(a, workspace, (hipStream_t)stream);
  return launched(who);
  OP_END
}

int lcn_int8_quantize_weight(int32_t device, void* stream, int32_t dtype, int64_t n, int64_t k, const void* w, int64_t stride_n,
                             int64_t stride_k, int8_t* q, float* scale) {
  OP_BEGIN("lcn_int8_quantize_weight")
  OP_CHECK(int8_sizes(who, 1, k, n));
  if (!known_dtype(dtype)) return fail(who, "dtype must be LCN_DTYPE_F32, _BF16 or _F16");
  if (n == 0) return LCN_OK;
  if (k == 0) return fail(who, "k is zero");
  if (!w || !q || !scale) return fail(who, "null operand");
  if (stride_n < 0 || stride_k < 0 || stride_n > kMaxStride / n || stride_k > kMaxStride / k) return fail(who, "bad strides of the weight");
  const int eb = elem_bytes(dtype);
  if ((uintptr_t)w % eb || (uintptr_t)scale % 4) return fail(who, "operand not aligned to its type");
  const View vw{w, 1, 1, (n - 1) * stride_n + (k - 1) * stride_k + 1, 0, 0, eb}, vq{q, 1, 1, n * k, 0, 0, 1}, vs{scale, 1, 1, n, 0, 0, 4};
  if (overlap(vw, vq) || overlap(vw, vs) || overlap(vq, vs)) return fail(who, "the operands must not overlap");
  DeviceGuard dev(device);
  if (dev.err != hipSuccess) return fail(who, hipGetErrorString(dev.err), LCN_E_HIP);
  QuantWArgs a{};
  a.n = (int)n;
  a.k = (int)k;
  a.dtype = dtype;
  a.w = w;
  a.w_n = stride_n;
  a.w_k = stride_k;
  a.q = q;
  a.scale = scale;
  launch_quant_weight(a, (hipStream_t)stream);
  return launched(who);
  OP_END
}

}  // extern "C"
