"""The 8-bit product at the ends of its documented ranges."""
import pytest
import torch

from test_gpu_ops import int8_case, int8_close

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
