"""Weight and int8 operators on torch device tensors (HIP kernels of liblcn.so).

    orthogonalize(g)                     Newton-Schulz orthogonalisation of matrices
    muon_update(param, momentum, grad)   one Muon step, in place
    quantize_weight(w)                   a float weight as int8 rows and channel scales
    int8_linear(x, weight, scale, bias)  product in 8-bit integers

Each runs on its tensors' device and torch's current stream of that device,
returns without synchronising, takes its scratch memory from torch's allocator
and can be captured into a graph.  There is no CPU path: tensors on the host are
refused.  None gives derivatives: a tensor that requires a gradient (outside
``torch.no_grad()``) or carries a forward-mode tangent is refused.  A bad argument raises ``ValueError``, a failure of the library
``LcnNativeError``.  cgcnn and the CLIs reach the same kernels through
``Network.set_optimizer`` and ``Network.set_precision``.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from .native import DTYPE_BF16, DTYPE_F16, DTYPE_F32, LcnNativeError, load_library

MUON_COEFFICIENTS = (3.4445, -4.775, 2.0315)

_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}


_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def _check(rc: int):
    if rc != 0:
        message = _library().lcn_last_error(None).decode()
        raise ValueError(message) if rc == -1 else LcnNativeError(f"liblcn error {rc}: {message}")


def _expect(cond: bool, message: str):
    if not cond:
        raise ValueError(message)


def _dtype(t: torch.Tensor, name: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} has type {t.dtype}, expected float32, bfloat16 or float16")
    return dt


def _tensor(t, name: str, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} is not a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: these operators run on the GPU only")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.is_neg():
        raise ValueError(f"{name} is a negated view: call resolve_neg() on it")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this operator does not give: call it under torch.no_grad()")
    # (the level is -1 outside forward_ad.dual_level(): asked first, it costs less)
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode tangent, which this operator does not pass on: call it on "
                         "forward_ad.unpack_dual(...).primal")
    return t


# Tensors written through their address: autograd then tells a backward that saved
# them that they changed, as after torch's own in-place operators.
_written = torch.autograd.graph.increment_version


def _matrices(t: torch.Tensor, name: str):
    """(batch, rows, cols, batch stride, row stride) of a [rows, cols] or [batch, rows, cols] tensor."""
    shape, s = t.shape, t.stride()
    if len(shape) not in (2, 3):
        raise ValueError(f"{name} has {len(shape)} dimensions, expected [rows, cols] or [batch, rows, cols]")
    if shape[-1] > 1 and s[-1] != 1:
        raise ValueError(f"{name}'s last dimension is not contiguous")
    if len(shape) == 2:
        return 1, shape[0], shape[1], 0, s[0]
    return shape[0], shape[1], shape[2], s[0], s[1]


# the handle of torch's current stream of a device, without building a Stream object
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_sizes = {}


def _workspace(name: str, a: int, b: int, c: int, device):
    """Scratch memory of a call from torch's allocator, which knows the stream: (tensor, address, bytes).
    The sizes are remembered: they depend on nothing but the numbers."""
    key = (name, a, b, c)
    n = _sizes.get(key)
    if n is None:
        n = getattr(_library(), name)(a, b, c)
        if n < 0:
            _check(n)
        if len(_sizes) < 4096:
            _sizes[key] = n
    if n == 0:
        return None, None, 0
    t = torch.empty(n, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), n


_coefficients = {}


def _triple(c):
    """The three coefficients as a C array (kept: the same few triples come again and again)."""
    a = _coefficients.get(c) if type(c) is tuple else None
    if a is None:
        c = tuple(float(v) for v in c)
        _expect(len(c) == 3, "coefficients are three numbers (a, b, c)")
        a = (ctypes.c_float * 3)(*c)
        if len(_coefficients) < 64:
            _coefficients[c] = a
    return a


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients=MUON_COEFFICIENTS, eps: float = 1e-7,
                  out: torch.Tensor = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of every matrix of g ([rows, cols] or [batch, rows, cols],
    float32, bfloat16 or float16):

        X = G / max(|G|_F, eps);  steps times: A = X X^T, X <- a X + (b A + c A A) X

    on the transpose where rows > cols.  The result has g's type; products are accurate to float32
    whatever that is.  out: a tensor like g for the result, g itself included.  A matrix that holds an
    infinity or a NaN gives NaN; a zero matrix gives zero."""
    _tensor(g, "g")
    dt = _dtype(g, "g")
    n, r, c, sb, sr = _matrices(g, "g")
    given = out is not None
    if not given:
        out = g.new_empty(g.shape)
    else:
        _tensor(out, "out", g.device)
        _expect(out.shape == g.shape and out.dtype == g.dtype, "out differs from g in shape or type")
    _, _, _, ob, orow = _matrices(out, "out")
    lib, device = _library(), g.device.index
    ws, ws_ptr, ws_bytes = _workspace("lcn_orthogonalize_workspace", n, r, c, g.device)
    _check(lib.lcn_orthogonalize(device, _stream(device), dt, n, r, c, g.data_ptr(), sb, sr, out.data_ptr(),
                                 ob, orow, int(steps), _triple(coefficients), eps, ws_ptr, ws_bytes))
    if given:
        _written(out)
    return out


def muon_update(param: torch.Tensor, momentum: torch.Tensor, grad: torch.Tensor, *, lr, beta: float = 0.95,
                nesterov: bool = True, weight_decay: float = 0.0, scale: float = None, steps: int = 5,
                coefficients=MUON_COEFFICIENTS, eps: float = 1e-7) -> None:
    """One Muon step on matrices ([rows, cols] or [batch, rows, cols]), in place:

        momentum <- beta momentum + grad;  u = grad + beta momentum (nesterov) or momentum
        param <- (1 - lr weight_decay) param - lr scale orthogonalize(u)

    param and momentum are float32, grad float32, bfloat16 or float16.  lr: a number, or a float32 device
    tensor of one element (read when the step runs, so a captured graph follows a schedule).  scale
    defaults to 0.2 sqrt(max(rows, cols)), which gives an update the root mean square of Adam's, so
    Adam's learning rates carry over."""
    _tensor(param, "param")
    _tensor(momentum, "momentum", param.device)
    _tensor(grad, "grad", param.device)
    _expect(param.dtype == momentum.dtype == torch.float32, "param and momentum are float32")
    _expect(param.shape == momentum.shape == grad.shape, "param, momentum and grad differ in shape")
    dt = _dtype(grad, "grad")
    n, r, c, pb, pr = _matrices(param, "param")
    _, _, _, mb, mr = _matrices(momentum, "momentum")
    _, _, _, gb, gr = _matrices(grad, "grad")
    lr_ptr, lr_value = None, 0.0
    if isinstance(lr, torch.Tensor):
        _tensor(lr, "lr", param.device)
        _expect(lr.dtype == torch.float32 and lr.numel() == 1, "lr as a tensor is one float32")
        lr_ptr = lr.data_ptr()
    else:
        lr_value = float(lr)
    if scale is None:
        scale = 0.2 * math.sqrt(max(r, c))
    lib, device = _library(), param.device.index
    ws, ws_ptr, ws_bytes = _workspace("lcn_orthogonalize_workspace", n, r, c, param.device)
    _check(lib.lcn_muon_update(device, _stream(device), dt, n, r, c, param.data_ptr(), pb, pr,
                               momentum.data_ptr(), mb, mr, grad.data_ptr(), gb, gr, lr_value, lr_ptr, scale, beta,
                               int(nesterov), weight_decay, int(steps), _triple(coefficients), eps, ws_ptr, ws_bytes))
    _written((param, momentum))


def quantize_weight(w: torch.Tensor, *, channel_dim: int = 0):
    """(int8 weight [n, k], float32 scale [n]) for int8_linear from a float weight: [n, k], or [k, n] with
    channel_dim=1 (any strides).  scale = max |w| / 127 of a channel, weight = rint(w * (127 / max |w|))."""
    _tensor(w, "w")
    dt = _dtype(w, "w")
    _expect(w.dim() == 2, f"w has {w.dim()} dimensions, expected 2")
    _expect(channel_dim in (0, 1), "channel_dim is 0 or 1")
    n, k = w.shape[channel_dim], w.shape[1 - channel_dim]
    q = torch.empty(n, k, dtype=torch.int8, device=w.device)
    scale = torch.empty(n, dtype=torch.float32, device=w.device)
    _check(_library().lcn_int8_quantize_weight(w.device.index, _stream(w.device.index), dt, n, k, w.data_ptr(),
                                                   w.stride(channel_dim), w.stride(1 - channel_dim), q.data_ptr(),
                                                   scale.data_ptr()))
    return q, scale


def int8_linear(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor = None, *,
                out: torch.Tensor = None) -> torch.Tensor:
    """x [..., k] (float32, bfloat16 or float16) times weight [n, k] (int8, one scale a channel):

        s = max_k |x| / 127,  q = rint(x * (127 / max_k |x|))   for each token (row of x)
        y[t, c] = (sum_k q[t, k] weight[c, k]) * s[t] * scale[c] (+ bias[c])

    scale and bias are float32 [n].  The sums are exact.  A token that holds an infinity or a NaN gives
    NaN; one below 2^-100 everywhere counts as zero.  out: [..., n] of x's type, not overlapping the inputs.
    For tensors on two or more leading dimensions x must be viewable as [tokens, k]."""
    _tensor(x, "x")
    dev = x.device
    _tensor(weight, "weight", dev)
    _tensor(scale, "scale", dev)
    dt = _dtype(x, "x")
    shape = x.shape
    if weight.dtype != torch.int8 or weight.dim() != 2:
        raise ValueError("weight is an int8 matrix [n, k]")
    n, k = weight.shape
    ws_row, ws_col = weight.stride()
    if not shape or shape[-1] != k:
        raise ValueError(f"x ends in {tuple(shape[-1:])}, the weight has k = {k}")
    if k > 1 and (x.stride(-1) != 1 or ws_col != 1):
        raise ValueError("the last dimension of x and weight is not contiguous")
    if scale.dtype != torch.float32 or scale.shape != (n,) or not scale.is_contiguous():
        raise ValueError(f"scale is a contiguous float32 [{n}]")
    bias_ptr = None
    if bias is not None:
        _tensor(bias, "bias", dev)
        if bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous():
            raise ValueError(f"bias is a contiguous float32 [{n}]")
        bias_ptr = bias.data_ptr()
    x2 = x if len(shape) == 2 else _rows(x, "x")
    tokens = x2.shape[0]
    given = out is not None
    if not given:
        out2 = x.new_empty(tokens, n)
        out = out2 if len(shape) == 2 else out2.view(shape[:-1] + (n,))
    else:
        _tensor(out, "out", dev)
        _expect(out.shape == shape[:-1] + (n,) and out.dtype == x.dtype, f"out is a {x.dtype} {tuple(shape[:-1]) + (n,)}")
        _expect(n <= 1 or out.stride(-1) == 1, "out's last dimension is not contiguous")
        out2 = out if out.dim() == 2 else _rows(out, "out")
    lib, device = _library(), dev.index
    ws, ws_ptr, ws_bytes = _workspace("lcn_int8_linear_workspace", tokens, k, n, dev)
    _check(lib.lcn_int8_linear(device, _stream(device), dt, tokens, k, n, x2.data_ptr(), x2.stride(0), weight.data_ptr(),
                               ws_row, scale.data_ptr(), bias_ptr, out2.data_ptr(), out2.stride(0), ws_ptr, ws_bytes))
    if given:
        _written(out)
    return out


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    try:
        return t.view(-1, t.shape[-1]) if t.numel() else t.new_empty(math.prod(t.shape[:-1]), t.shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}'s leading dimensions cannot be viewed as one") from None
