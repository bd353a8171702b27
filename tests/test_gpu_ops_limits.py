"""The operators at the ends of their documented ranges."""
import pytest
import torch

from test_gpu_ops import close, gradient, int8_case, int8_close
from test_gpu_ops_accuracy import bound, norms

pytestmark = pytest.mark.gpu

from lcn_amd import native, ops  # noqa: E402


@pytest.mark.parametrize("tokens", [1 << 30, (1 << 29) + 1])
def test_most_tokens(tokens):
    """2^30 tokens, more than the threads of one launch can be counted for."""
    x = torch.empty(tokens, 1, device="cuda", dtype=torch.float16).normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    _, w, s, b = int8_case(1, 1, 1, torch.float16, seed=5)
    s = s + 1e-3
    got = ops.int8_linear(x, w, s, b)
    half = 1 << 29
    rows = [0, 63, 64, half - 65, half - 1, half, tokens - 65, tokens - 64, tokens - 1]
    int8_close(got[rows], x[rows], w, s, b)
    # every token: an integer of 127 times the weight, so y = x w s + b up to the product's roundings (five, of 2^-24) and fp16's
    for at in range(0, tokens, 1 << 27):
        y, v = got[at:at + (1 << 27)].float(), x[at:at + (1 << 27)].float() * (float(w[0, 0]) * float(s[0]))
        assert bool(((y - v - b).abs() <= 2.0 ** -11 * (v + b).abs() + 2.0 ** -20 * (v.abs() + b.abs()) + 2.0 ** -25).all())
    with pytest.raises(ValueError, match="too many"):
        ops.int8_linear(x[:1].expand(tokens + half + 1, 1), w, s, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_tokens_whose_rows_are_far_apart(dtype):
    """16 384 tokens and more, 2^22 elements and more from one row of the output to the next: 137 GB of addresses."""
    t, k, n, pitch = 16385, 64, 33, (1 << 22) + 64
    torch.cuda.empty_cache()
    assert torch.cuda.mem_get_info()[0] > 145e9
    store = torch.empty((t + 2) * pitch, device="cuda", dtype=dtype)
    around = store.as_strided((t + 2, n + 10), (pitch, 1))   # a row before, one behind, columns on either side
    around.fill_(7.0)
    x, w, s, b = int8_case(t, k, n, dtype, seed=6)
    x[77, 5] = float("nan")
    x[78] = 0
    out = around[1:t + 1, 4:n + 4]
    ops.int8_linear(x, w, s, b, out=out)
    got = out.clone()
    out.fill_(7.0)
    assert bool((around == 7.0).all())
    del store, around, out
    torch.cuda.empty_cache()
    near = ops.int8_linear(x, w, s, b)
    assert bool(got[77].isnan().all()) and bool(near[77].isnan().all())
    rest = torch.arange(t, device="cuda") != 77
    int8_close(got[rest], x[rest], w, s, b)
    int8_close(near[rest], x[rest], w, s, b)


@pytest.mark.parametrize("t,k,n", [(16384, 64, 64), (16500, 1088, 129), (20001, 1216, 70), (16384, 1, 1), (17000, 1280, 64), (2000, 320, 500)])
def test_int8_linear_stays_inside_its_workspace(t, k, n):
    lib = native.load_library()
    x, w, s, b = int8_case(t, k, n, torch.bfloat16, seed=t + n)
    out = torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    need = lib.lcn_int8_linear_workspace(t, k, n)
    assert need > 0
    ws = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    ops._check(lib.lcn_int8_linear(0, torch.cuda.current_stream().cuda_stream, native.DTYPE_BF16, t, k, n, x.data_ptr(), x.stride(0), w.data_ptr(),
                                   w.stride(0), s.data_ptr(), b.data_ptr(), out.data_ptr(), out.stride(0), ws.data_ptr() + 4096, need))
    assert bool((ws[:4096] == 0xA5).all()) and bool((ws[4096 + need:] == 0xA5).all())
    int8_close(out, x, w, s, b)


def test_a_plane_of_2_31_bytes():
    """The largest matrix: rows of disjoint columns are orthogonal, so a step multiplies each row by a number of its own,
    p(s) / s of its norm s, and everything else stays zero."""
    r, c = 16384, 65000
    g = torch.zeros(r, c, device="cuda")
    j = torch.arange(c, device="cuda")
    v = torch.randn(c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    g[j % r, j] = v
    ops.orthogonalize(g, out=g)
    x = v.double() / torch.linalg.norm(v.double())
    a, b, d = ops.MUON_COEFFICIENTS
    for _ in range(5):
        s2 = torch.zeros(r, device="cuda", dtype=torch.float64).index_add_(0, j % r, x * x)[j % r]
        x = x * (a + b * s2 + d * s2 * s2)
    got = g[j % r, j].double()
    # five steps of three products with an error of 2^-22 each, which the steps that follow stretch by
    # |s p'(s) / p(s)|, below 4 in all for norms that start at 1/128.  Elements far below a row's norm (v of 1e-5 and
    # less) meet the end of fp16's range: a lo half has a spacing of 2^-24 in units of 1 / 2^15, so each of the five
    # stored X is off by up to 2^-40, which the row's factor, at most a^5, then multiplies
    assert bool(((got - x).abs() <= 2.0 ** -16 * x.abs() + 5 * a ** 5 * 2.0 ** -40).all())
    g[j % r, j] = 0
    assert not bool(g.any())


def _batched(g, dtype, steps=5):
    x = (g.double() / torch.linalg.norm(g.double(), dim=(1, 2), keepdim=True)).to(dtype)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    a, b, c = ops.MUON_COEFFICIENTS
    for _ in range(steps):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


@pytest.mark.parametrize("shape", [(65535, 3, 5), (65535, 50, 40), (40000, 20, 130), (130, 20, 20000), (1, 20, 65536), (1, 65536, 33), (1, 64, 65536),
                                   (1, 65, 65536), (1, 65536, 100), (3000, 70, 66)])
def test_orthogonalize_many_and_long_matrices(shape):
    g = gradient(shape, torch.float32, seed=shape[1])
    want, plain32 = _batched(g, torch.float64), _batched(g, torch.float32)
    got = ops.orthogonalize(g)
    # matrix by matrix the polynomial's own bound; over the batch, where chance evens out, the float32 one
    close(got, want.cpu(), torch.float32)
    whole = (1, shape[0] * shape[1], shape[2])
    err, limit = norms((got.double() - want).view(whole)), bound(want.view(whole), plain32.view(whole))
    assert bool((err <= limit).all()), f"{float(err / limit):.3g} of the bound"


@pytest.mark.parametrize("t", [3, 40, 300, 1030, 16390])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_int8_linear_rows_far_apart_in_its_inputs(t, dtype):
    """Weights 2^28 bytes a row apart, tokens as far as 8 GB allow."""
    k, n, pitch = 100, 17, 1 << 28
    x, w, s, b = int8_case(t, k, n, dtype, seed=t)
    far = torch.zeros(n * pitch, device="cuda", dtype=torch.int8).as_strided((n, k), (pitch, 1), 5)
    far.copy_(w)
    gap = min(1 << 28, (1 << 32) // t // 16 * 8)
    tokens = torch.zeros(t * gap, device="cuda", dtype=dtype).as_strided((t, k), (gap, 1), 3)
    tokens.copy_(x)
    int8_close(ops.int8_linear(tokens, far, s, b), x, w, s, b)


@pytest.mark.parametrize("t,k,n", [(1, 64, 1 << 24), (5, 131072, 16000), (40, 64, 1 << 24), (40, 131071, 16000), (300, 131072, 16000), (1100, 4096, 500000)])
def test_int8_linear_largest_weights(t, k, n):
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, k, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.empty(n, k, device="cuda", dtype=torch.int8).random_(-127, 128, generator=g)
    s = torch.rand(n, device="cuda", generator=g) * 1e-3 + 1e-4
    y = ops.int8_linear(x, w, s)
    pick = torch.cat([torch.arange(0, 40), torch.arange(n // 2 - 20, n // 2 + 20), torch.arange(n - 40, n),
                      torch.arange(7, n, max(1, n // 97))]).cuda()
    int8_close(y[:, pick], x, w[pick], s[pick], None)
