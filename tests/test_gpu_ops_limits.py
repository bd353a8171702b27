"""The 8-bit product at the ends of its documented ranges."""
import pytest
import torch

from test_gpu_ops import int8_case, int8_close

pytestmark = pytest.mark.gpu

from lcn_amd import ops  # noqa: E402


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
