"""The handle-free operators on the GPU against plain 64-bit implementations.

Tolerances.  orthogonalize: every product is made of two-part fp16 numbers, off by at most 3 * 2^-22
of |P||Q| (two representation errors of 2^-22 and the dropped lo lo term) plus the fp32 accumulation;
one step's relative perturbation is below 2^-20, and the polynomial stretches a perturbation by at most
|a| a step where singular values are small, so after `steps` steps the result is off by less than
2^-20 * |a|^steps of its norm, plus half a rounding of its type.  int8_linear: the integers and their
sums are exact; what rounds is the sum's conversion, the two scales' products, the scale itself and the
bias: five times 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from lcn_amd import native, ops  # noqa: E402

A_, B_, C_ = ops.MUON_COEFFICIENTS
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def polynomial(g, steps=5, coef=ops.MUON_COEFFICIENTS, eps=1e-7):
    """float64 on the CPU, matrix by matrix."""
    g = g.detach().double().cpu()
    g3 = g.reshape((-1,) + g.shape[-2:])
    out = torch.empty_like(g3)
    for i in range(g3.shape[0]):
        x = g3[i] / max(float(torch.linalg.norm(g3[i])), eps)
        if x.shape[0] > x.shape[1]:
            x = x.T
        for _ in range(steps):
            gram = x @ x.T
            x = coef[0] * x + (coef[1] * gram + coef[2] * gram @ gram) @ x
        out[i] = x if g3.shape[1] <= g3.shape[2] else x.T
    return out.reshape(g.shape)


def tolerance(dtype, steps=5, a=A_):
    return 2.0 ** -20 * abs(a) ** steps + half_step(dtype)


def close(got, want, dtype, steps=5, a=A_):
    got, want = got.detach().double().cpu(), want.double()
    d = torch.linalg.norm((got - want).reshape(-1, want.shape[-2] * want.shape[-1]), dim=1)
    n = torch.linalg.norm(want.reshape(-1, want.shape[-2] * want.shape[-1]), dim=1)
    floor = 2.0 ** -25 * math.sqrt(want.shape[-1] * want.shape[-2]) if dtype == torch.float16 else 0.0
    assert bool((d <= tolerance(dtype, steps, a) * n + floor).all()), f"off by {(d / n).max():.3g}"


def gradient(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=g))).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (5, 5), (17, 34), (31, 33), (32, 32), (33, 31), (51, 1088), (63, 64), (64, 64), (65, 64),
          (64, 200), (127, 129), (128, 128), (129, 127), (160, 96), (257, 300), (300, 257), (1, 300), (40, 7001), (6500, 20), (97, 128), (128, 65), (100, 4001), (4001, 70)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_shapes(shape, dtype):
    for batch in ((), (3,)):
        g = gradient(batch + shape, dtype)
        out = ops.orthogonalize(g)
        assert out.dtype == dtype and out.shape == g.shape
        close(out, polynomial(g), dtype)


def test_orthogonalize_hidden_and_large_batch():
    g = gradient((2, 1088, 1088), torch.float32)
    close(ops.orthogonalize(g), polynomial(g), torch.float32)
    g = gradient((301, 40, 24), torch.float32)
    close(ops.orthogonalize(g), polynomial(g), torch.float32)


# many matrices, of which a workgroup takes several chunks of columns; and few with a long contraction, whose Gram
# matrix is summed in slices
@pytest.mark.parametrize("shape", [(300, 40, 500), (700, 300, 20), (90, 64, 1300), (2, 333, 5000), (3, 5003, 97), (1, 65, 2111), (40, 66, 70)])
def test_orthogonalize_batches_and_long_sides(shape):
    g = gradient(shape, torch.float32, seed=shape[0])
    close(ops.orthogonalize(g), polynomial(g), torch.float32)
    p, m = torch.zeros_like(g), gradient(shape, torch.float32, seed=1)
    want = muon_reference(p, m, g, 0.01, 0.95, True, 0.0, 1.0)
    ops.muon_update(p, m, g, lr=0.01, scale=1.0)
    muon_close(p, m, *want, 0.01, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(192, 192), (48, 40)])
def test_orthogonalize_low_rank(dtype, shape):
    """A gradient of few samples: most singular values are zero and their directions must stay empty."""
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.randn(shape[0], 5, device="cuda", generator=g) @ torch.randn(5, shape[1], device="cuda", generator=g)
    u = u.to(dtype)
    close(ops.orthogonalize(u), polynomial(u), dtype)


@pytest.mark.parametrize("shape", [(40, 56), (96, 200), (200, 96)])
def test_orthogonalize_layouts(shape):
    r, c = shape
    want = None
    base = gradient((3, r, c), torch.float32, 5)
    want = polynomial(base)
    wide = torch.full((3, r, c + 13), float("nan"), device="cuda")
    wide[:, :, 7:7 + c] = base
    close(ops.orthogonalize(wide[:, :, 7:7 + c]), want, torch.float32)                      # rows apart
    inter = base.permute(1, 0, 2).contiguous().permute(1, 0, 2)                              # batch inside the rows
    close(ops.orthogonalize(inter), want, torch.float32)
    close(ops.orthogonalize(base[1:2].expand(3, r, c)), want[1:2].expand(3, r, c), torch.float32)
    dst = torch.full((3, r + 2, c + 5), 77.0, device="cuda")
    got = ops.orthogonalize(base, out=dst[:, 1:-1, 2:2 + c])
    close(got, want, torch.float32)
    keep = torch.ones_like(dst, dtype=torch.bool)
    keep[:, 1:-1, 2:2 + c] = False
    assert bool((dst[keep] == 77.0).all())                                                   # nothing around it was touched
    same = base.clone()
    assert ops.orthogonalize(same, out=same) is same                                         # in place
    close(same, want, torch.float32)


@pytest.mark.parametrize("shape", [(24, 40), (80, 130)])
def test_orthogonalize_special_values(shape):
    g = gradient((6,) + shape, torch.float32, 7)
    g[1] = 0.0
    g[2, 3, 5] = float("nan")
    g[3, 0, 0] = float("-inf")
    g[4] *= 1e-25
    g[5] *= 1e30
    want = polynomial(g, eps=1e-30)
    out = ops.orthogonalize(g, eps=1e-30)
    assert bool((out[1] == 0).all()) and bool(out[2].isnan().all()) and bool(out[3].isnan().all())
    for i in (0, 4, 5):
        close(out[i], want[i], torch.float32)
    one = torch.zeros((1,) + shape, device="cuda")
    one[0, 4, 9] = -3.0                                                                      # a single entry
    close(ops.orthogonalize(one), polynomial(one), torch.float32)


@pytest.mark.parametrize("steps,coef", [(1, ops.MUON_COEFFICIENTS), (2, ops.MUON_COEFFICIENTS), (9, (1.875, -1.25, 0.375)), (7, (1.5, -0.5, 0.0))])
def test_orthogonalize_other_polynomials(steps, coef):
    for shape in ((48, 60), (140, 90)):
        g = gradient(shape, torch.float32, 11)
        close(ops.orthogonalize(g, steps=steps, coefficients=coef), polynomial(g, steps, coef), torch.float32, steps, coef[0])


def test_orthogonalize_repeats_bitwise():
    for shape in ((2, 300, 280), (5, 64, 64)):
        g = gradient(shape, torch.bfloat16)
        a, b = ops.orthogonalize(g), ops.orthogonalize(g)
        assert torch.equal(a, b)


def test_orthogonalize_stays_inside_its_workspace():
    lib = native.load_library()
    for shape in ((2, 70, 300), (3, 64, 64), (1, 300, 70), (1, 1, 1), (4, 33, 95), (2, 200, 140), (1, 40, 6400)):
        g = gradient(shape, torch.float32)
        out = torch.empty_like(g)
        need = lib.lcn_orthogonalize_workspace(*shape)
        ws = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
        ops._check(lib.lcn_orthogonalize(0, torch.cuda.current_stream().cuda_stream, 0, *shape, g.data_ptr(), g.stride(0), g.stride(1),
                                         out.data_ptr(), out.stride(0), out.stride(1), 5, ops._triple(ops.MUON_COEFFICIENTS), 1e-7,
                                         ws.data_ptr() + 4096, need))
        assert bool((ws[:4096] == 0xA5).all()) and bool((ws[4096 + need:] == 0xA5).all())
        close(out, polynomial(g), torch.float32)


# ---- muon ----------------------------------------------------------------------------------------
def muon_reference(p, m, g, lr, beta, nesterov, decay, scale):
    p, m, g = (t.detach().double().cpu() for t in (p, m, g))
    m = beta * m + g
    u = g + beta * m if nesterov else m
    return (1 - lr * decay) * p - lr * scale * polynomial(u), m


def muon_close(p, m, want_p, want_m, lr, scale):
    dm = (m.double().cpu() - want_m).abs()
    assert bool((dm <= 2 * 2.0 ** -24 * want_m.abs().max()).all())
    # the step's own error, and three roundings of the parameter
    d = (p.double().cpu() - want_p).reshape(-1, p.shape[-2] * p.shape[-1])
    n = want_p.reshape(-1, p.shape[-2] * p.shape[-1])
    step = lr * scale * math.sqrt(min(p.shape[-2:])) * 1.25 * (2.0 ** -20 * A_ ** 5)  # |NS(u)|_F <= 1.25 sqrt(min side)
    assert bool((torch.linalg.norm(d, dim=1) <= step + 3 * 2.0 ** -24 * torch.linalg.norm(n, dim=1)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 3), (3, 34, 1088), (2, 60, 64), (130, 51), (2, 257, 140)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(shape, dtype, nesterov):
    p, m = gradient(shape, torch.float32, 1), gradient(shape, torch.float32, 2)
    lr, beta, decay = 0.02, 0.9, 0.1
    scale = 0.2 * math.sqrt(max(shape[-2:]))
    for i in range(3):  # steps of one run: the state goes from one to the next
        g = gradient(shape, dtype, 10 + i)
        want = muon_reference(p, m, g, lr, beta, nesterov, decay, scale)
        assert ops.muon_update(p, m, g, lr=lr, beta=beta, nesterov=nesterov, weight_decay=decay) is None
        muon_close(p, m, *want, lr, scale)


def test_muon_layouts_and_lr_tensor():
    # weights apart in one flat vector, 4-byte aligned only, as a network's parameters are
    r, c, gap = 70, 90, 33
    flat = [torch.full((1 + 3 * (r * c + gap),), 5.0, device="cuda") for _ in range(2)]
    views = [f[1:].view(3, r * c + gap)[:, :r * c].view(3, r, c) for f in flat]
    src = [gradient((3, r, c), torch.float32, 20 + i) for i in range(2)]
    for v, s in zip(views, src):
        v.copy_(s)
    g = gradient((3, r, c), torch.bfloat16, 30)
    lr = torch.tensor([0.05], device="cuda")
    want = muon_reference(src[0], src[1], g, 0.05, 0.95, True, 0.0, 2.5)
    ops.muon_update(views[0], views[1], g, lr=lr, scale=2.5)
    muon_close(views[0], views[1], *want, 0.05, 2.5)
    for f in flat:
        assert bool((f[1:].view(3, -1)[:, r * c:] == 5.0).all()) and float(f[0]) == 5.0
    keep = views[0].clone()
    lr.zero_()
    ops.muon_update(views[0], views[1], g, lr=lr, scale=2.5, weight_decay=0.5)
    assert torch.equal(views[0], keep)  # a zero rate leaves the weights as they are


def test_muon_refuses_on_the_gpu():
    p = torch.zeros(8, 8, device="cuda")
    for args in ((p, p, p.clone()), (p, p.clone(), p), (p.half(), p.clone(), p.clone()), (p, p.clone(), p.double()),
                 (p, p.clone()[:4], p.clone()), (p.t()[:, :4], p.clone()[:, :4], p.clone()[:, :4]),
                 (torch.zeros(8, 8, device="cuda", requires_grad=True), p.clone(), p.clone())):
        with pytest.raises(ValueError):
            ops.muon_update(*args, lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_update(p, p.clone(), p.clone(), lr=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        ops.orthogonalize(torch.zeros(4, 4, 4, 4, device="cuda"))
    with pytest.raises(ValueError):
        ops.orthogonalize(p, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError):
        ops.orthogonalize(p, out=p.half())
    z = torch.randn(8, 16, device="cuda", dtype=torch.complex64)
    negated = z.conj().imag  # the negation is a flag of the view
    assert negated.is_neg()
    with pytest.raises(ValueError, match="negated"):
        ops.orthogonalize(negated)


# ---- int8 ----------------------------------------------------------------------------------------
def int8_case(t, k, n, dtype, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(t, k, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))).to(dtype)
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    s = torch.rand(n, device="cuda", generator=g) * 1e-3 + 1e-4
    b = torch.randn(n, device="cuda", generator=g) if bias else None
    return x, w, s, b


def int8_reference(x, w, s, b):
    x32 = x.detach().float().cpu()
    top = x32.abs().amax(-1, keepdim=True)
    factor = torch.where(top >= 2.0 ** -100, torch.div(torch.full_like(top, 127), top), torch.zeros_like(top))
    q = torch.round(x32 * factor).clamp(-127, 127).double()
    product = (q @ w.cpu().double().T) * torch.where(top >= 2.0 ** -100, top.double() / 127, 0.0) * s.cpu().double()
    return product, product + (0 if b is None else b.cpu().double())


def int8_close(got, x, w, s, b):
    product, want = int8_reference(x, w, s, b)
    d = (got.double().cpu() - want).abs()
    u = half_step(got.dtype)
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = (5 * 2.0 ** -24 * product.abs() + 2.0 ** -24 * want.abs()) * (1 + u) + (u * want.abs() if u > 2.0 ** -24 else 0) + floor
    assert bool((d <= bound).all()), f"{(d - bound).max():.3g} over"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 64, 64), (1, 1088, 1088), (2, 51, 1088), (3, 1003, 333), (15, 16, 17), (16, 128, 128),
                                   (17, 80, 31), (31, 200, 64), (33, 34, 1088), (64, 64, 129), (65, 144, 127), (127, 1088, 51),
                                   (128, 65, 256), (129, 63, 130), (200, 1088, 1088), (777, 1003, 333), (1000, 96, 16), (1030, 1088, 340), (16, 1088, 70), (13, 2520, 40),
                                   (200, 1601, 96), (21, 1535, 130), (600, 1087, 1025)])
def test_int8_linear_shapes(t, k, n, dtype):
    for bias in (True, False):
        x, w, s, b = int8_case(t, k, n, dtype, seed=t + k + n, bias=bias)
        y = ops.int8_linear(x, w, s, b)
        assert y.shape == (t, n) and y.dtype == dtype
        int8_close(y, x, w, s, b)


# many tokens: 64 at a time are quantised next to their product while K fits (1216), panels through memory past that
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,n", [(16384, 1088, 1088), (16447, 64, 64), (16385, 1216, 129), (17001, 80, 1), (16400, 8, 300),
                                   (20000, 320, 200), (16384, 1280, 257), (16401, 1003, 96), (16383, 136, 449)])
def test_int8_linear_many_tokens(t, k, n, dtype):
    x, w, s, b = int8_case(t, k, n, dtype, seed=t + k)
    wide = torch.full((t + 3, n + 5), 7.0, device="cuda", dtype=dtype)
    got = ops.int8_linear(x, w, s, b, out=wide[1:t + 1, 2:n + 2])
    int8_close(got, x, w, s, b)
    wide[1:t + 1, 2:n + 2] = 7.0
    assert bool((wide == 7.0).all())
    x[5, k // 2] = float("nan")
    x[8000] = 0
    plain = ops.int8_linear(x, w, s)
    assert bool(plain[5].isnan().all()) and bool((plain[8000] == 0).all()) and bool(plain[6:].isfinite().all())
    assert torch.equal(plain[6:], ops.int8_linear(x, w, s)[6:])


def test_int8_linear_rows_far_apart():
    # 32 rows of the output span more than 2^31 bytes: offsets of the dropped rows of the last tile do not wrap
    for t in (65, 1030):
        x, w, s, b = int8_case(t, 48, 40, torch.float32, seed=3)
        pitch = (1 << 25) if t == 65 else (1 << 23) + 64
        store = torch.empty((t - 1) * pitch + 40, device="cuda")
        out = store.as_strided((t, 40), (pitch, 1))
        ops.int8_linear(x, w, s, b, out=out)
        int8_close(out.clone(), x, w, s, b)
        del store, out


@pytest.mark.parametrize("t,k,n", [(16500, 131072, 32), (2000100, 1088, 16)])
def test_int8_linear_offsets_past_32_bits(t, k, n):
    # three rounds of at most 1 GiB of integers; and 31 250 groups of 64 tokens in one launch
    x = torch.empty(t, k, device="cuda", dtype=torch.float16).normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    _, w, s, b = int8_case(1, k, n, torch.float16, seed=2)
    s *= 1e-3  # sums of 131 072 products stay inside fp16's range
    got = ops.int8_linear(x, w, s, b)
    rows = [0, 63, 64, 8191, 8192, 8193, t // 2, 16383, 16384, t - 65, t - 2, t - 1]
    int8_close(got[rows], x[rows], w, s, b)


def test_orthogonalize_offsets_past_32_bits():
    store = torch.empty((3 << 31) + 200 * 136, device="cuda", dtype=torch.bfloat16)
    for shape in ((200, 136), (100, 136)):
        g = store.as_strided((3,) + shape, (3 << 30, 136, 1))
        g.copy_(gradient((3,) + shape, torch.bfloat16, 40))
        want = ops.orthogonalize(g.contiguous())
        assert torch.equal(ops.orthogonalize(g, out=g), want)


def test_int8_linear_long_k_and_extreme_integers():
    k = 131072
    x = torch.full((3, k), 2.0, device="cuda")
    x[1] *= -1
    w = torch.full((5, k), 127, dtype=torch.int8, device="cuda")
    w[3] = -128
    s = torch.full((5,), 2.0 ** -20, device="cuda")
    int8_close(ops.int8_linear(x, w, s), x, w, s, None)


@pytest.mark.parametrize("t", [3, 40, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_linear_layouts(t, dtype):
    k, n = 100, 70
    x, w, s, b = int8_case(t, k, n, dtype, 3)
    wide = torch.full((t, k + 9), float("nan"), device="cuda", dtype=dtype)
    wide[:, 5:5 + k] = x
    ww = torch.full((n, k + 11), 99, device="cuda", dtype=torch.int8)
    ww[:, 3:3 + k] = w
    dst = torch.full((t + 2, n + 7), 9.0, device="cuda", dtype=dtype)
    y = ops.int8_linear(wide[:, 5:5 + k], ww[:, 3:3 + k], s, b, out=dst[1:-1, 4:4 + n])
    int8_close(y, x, w, s, b)
    keep = torch.ones_like(dst, dtype=torch.bool)
    keep[1:-1, 4:4 + n] = False
    assert bool((dst[keep] == 9.0).all())
    w16 = torch.zeros(n, 128, device="cuda", dtype=torch.int8)   # rows of 16-byte pieces with something behind k
    w16[:, :k], w16[:, k:] = w, 55
    int8_close(ops.int8_linear(x, w16[:, :k], s, b), x, w, s, b)
    lead = x.view(1, t, 1, k)
    y3 = ops.int8_linear(lead, w, s, b)
    assert y3.shape == (1, t, 1, n)
    int8_close(y3.view(t, n), x, w, s, b)
    row = x[:1].expand(t, k)                                      # every token the same row
    int8_close(ops.int8_linear(row, w, s, b), row, w, s, b)


@pytest.mark.parametrize("t", [7, 150])
def test_int8_linear_special_rows(t):
    k, n = 130, 50
    x, w, s, b = int8_case(t, k, n, torch.float32, 5)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, 129] = float("inf")
    x[3] *= 1e-36                                                  # counts as zero
    x[4] *= 1e-28                                                  # does not
    x[5] *= 1e28
    y = ops.int8_linear(x, w, s, b)
    assert torch.equal(y[0], b) and torch.equal(y[3], b)
    assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    rest = [0, 4, 5, 6] + list(range(7, t))
    int8_close(y[rest], x[rest], w, s, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (5, 3), (64, 64), (1088, 51), (33, 1003)])
@pytest.mark.parametrize("channel_dim", [0, 1])
def test_quantize_weight(n, k, dtype, channel_dim):
    w = gradient((n, k) if channel_dim == 0 else (k, n), dtype, 9)
    q, s = ops.quantize_weight(w, channel_dim=channel_dim)
    wn = (w if channel_dim == 0 else w.t()).float().cpu()
    top = wn.abs().amax(1)
    assert torch.equal(s.cpu(), torch.div(top, torch.full_like(top, 127)))
    assert torch.equal(q.cpu().float(), torch.round(wn * torch.div(torch.full_like(top, 127), top)[:, None]))
    # what they stand for is within half a step (and the roundings of the factor and the product: 2 * 2^-24 * 127 steps)
    assert bool(((q.cpu().double() * s.cpu().double()[:, None] - wn.double()).abs() <= s.cpu().double()[:, None] * (0.5 + 2.0 ** -16)).all())


def test_quantize_weight_special_channels():
    w = gradient((4, 40), torch.float32, 1)
    w[0], w[1, 2], w[2, 39] = 0.0, float("nan"), float("inf")
    q, s = ops.quantize_weight(w)
    assert float(s[0]) == 0.0 and bool(s[1].isnan()) and bool(s[2].isnan()) and bool((q[:3] == 0).all())


def test_int8_refuses_on_the_gpu():
    x, w, s, b = int8_case(4, 32, 16, torch.float32)
    for args in ((x, w.float(), s), (x[:, :31], w, s), (x, w, s[:3]), (x, w, s.half()), (x, w, s, b[:2]), (x.double(), w, s),
                 (x.t(), w, s), (x.cpu(), w, s), (x, w.cpu(), s)):
        with pytest.raises(ValueError):
            ops.int8_linear(*args)
    with pytest.raises(ValueError):
        ops.int8_linear(x[:, :16], w[:, :16], s, out=x[:, :16])
    with pytest.raises(ValueError):
        ops.int8_linear(x.clone().requires_grad_(), w, s)
    with pytest.raises(ValueError):
        ops.int8_linear(torch.zeros(2, 3, 64, device="cuda").transpose(0, 1)[..., :32], w, s)
    assert ops.int8_linear(x[:0], w, s).shape == (0, 16)
    assert ops.int8_linear(torch.zeros(2, 0, 32, device="cuda"), w, s).shape == (2, 0, 16)


# ---- streams and graphs --------------------------------------------------------------------------
def test_other_streams():
    g1, g2 = gradient((2, 200, 150), torch.float32, 1), gradient((2, 200, 150), torch.float32, 2)
    x, w, s, b = int8_case(300, 500, 200, torch.float32)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a1 = [ops.orthogonalize(g1) for _ in range(4)]
        y1 = ops.int8_linear(x, w, s, b)
    with torch.cuda.stream(s2):
        a2 = [ops.orthogonalize(g2) for _ in range(4)]
        y2 = ops.int8_linear(x, w, s, None)
    torch.cuda.synchronize()
    for o in a1:
        close(o, polynomial(g1), torch.float32)
    for o in a2:
        close(o, polynomial(g2), torch.float32)
    int8_close(y1, x, w, s, b)
    int8_close(y2, x, w, s, None)


def test_captured_and_replayed():
    """Two graphs, each with its own scratch memory, replayed in turn with eager work between."""
    sizes = [(2, 90, 140), (3, 64, 50)]
    grads = [gradient(z, torch.float32, i) for i, z in enumerate(sizes)]
    params = [gradient(z, torch.float32, 10 + i) for i, z in enumerate(sizes)]
    moms = [torch.zeros_like(p) for p in params]
    x, w, s, b = int8_case(40, 140, 90, torch.float32)
    lr = torch.tensor([0.01], device="cuda")
    eager_p, eager_m = [p.clone() for p in params], [m.clone() for m in moms]
    ops.orthogonalize(grads[0]), ops.int8_linear(x, w, s, b)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.muon_update(params[i], moms[i], grads[i], lr=lr)
            outs.append(ops.int8_linear(x, w, s, b))
        graphs.append(graph)
    for step in range(4):
        lr.fill_(0.01 / (step + 1))
        for i in range(2):
            grads[i].copy_(gradient(sizes[i], torch.float32, 100 + 10 * step + i))
        x.copy_(int8_case(40, 140, 90, torch.float32, 50 + step)[0])
        for i in (step % 2, 1 - step % 2):
            graphs[i].replay()
        for i in range(2):
            ops.muon_update(eager_p[i], eager_m[i], grads[i], lr=lr)
        y = ops.int8_linear(x, w, s, b)
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(params[i], eager_p[i]) and torch.equal(moms[i], eager_m[i]) and torch.equal(outs[i], y)


def test_a_run_of_them_together():
    """Train a linear map with Muon, lay its weight out in 8 bits, answer with it."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(512, 96, device="cuda", generator=gen)
    target = x @ torch.randn(96, 80, device="cuda", generator=gen) * 0.1
    w = torch.randn(96, 80, device="cuda", generator=gen) * 0.1
    m = torch.zeros_like(w)
    w64, m64 = w.double().cpu(), m.double().cpu()
    for _ in range(6):
        grad = x.t() @ (x @ w - target) / 512
        want_w, want_m = muon_reference(w, m, grad, 0.02, 0.95, True, 0.0, 0.2 * math.sqrt(96))
        ops.muon_update(w, m, grad, lr=0.02)
        muon_close(w, m, want_w, want_m, 0.02, 0.2 * math.sqrt(96))
    q, s = ops.quantize_weight(w, channel_dim=1)
    y = ops.int8_linear(x, q, s)
    int8_close(y, x, q, s, None)
    # 8 bits a number on either side: the worst error of a sum of 96 products of half a step each
    worst = (x.abs().amax(1, keepdim=True) / 254 * w.abs().sum(0) + s / 2 * x.abs().sum(1, keepdim=True) + 96 * x.abs().amax(1, keepdim=True) / 254 * s / 2)
    assert bool(((y - x @ w).abs() <= worst * 1.001 + 1e-5).all())
    assert w64.shape == m64.shape
