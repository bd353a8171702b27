"""Float32 accuracy of the weight operators on full-rank gradients, path by path, and infinities and NaN
in every type.

Tolerance.  A matrix is held in two fp16 numbers, 2^-22 of an element off at most; a plain float32
iteration holds it to 2^-24.  A product meets that error in either operand and drops the lo lo term:
three errors of four times the plain one's, so the result is at most 12 times as far from 64 bits as the
plain float32 iteration on the same input, whose distance d32 carries the polynomial's own amplification
of that input.  Fifteen products of 2^-22 each (2^-18) are added for inputs on which the plain form
happens to be exact.  A lo half left out of the last product moves the result by five times that bound
and more (on the shapes below, in a simulation).  What a 16-bit output leaves of the error is the
distance of the exact value from the numbers that round to it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from lcn_amd import ops  # noqa: E402
from test_gpu_ops import TYPES, gradient, int8_case, int8_close  # noqa: E402

A_, B_, C_ = ops.MUON_COEFFICIENTS


def plain(u, dtype, steps=5):
    """The definition in elementary operations of one type, on u's device, matrix by matrix."""
    u3 = u.reshape((-1,) + u.shape[-2:])
    out = torch.empty(u3.shape, dtype=dtype, device=u.device)
    for i in range(u3.shape[0]):
        x = (u3[i].double() / max(float(torch.linalg.norm(u3[i].double())), 1e-7)).to(dtype)
        if x.shape[0] > x.shape[1]:
            x = x.t().contiguous()
        for _ in range(steps):
            gram = x @ x.t().contiguous()
            x = A_ * x + (B_ * gram + C_ * (gram @ gram)) @ x
        out[i] = x if u3.shape[1] <= u3.shape[2] else x.t()
    return out.reshape(u.shape)


def norms(t):
    return torch.linalg.norm(t.double().reshape(-1, t.shape[-2] * t.shape[-1]), dim=1)


def bound(want, plain32):
    """The largest norm of a matrix's error, a matrix."""
    return 12 * norms(plain32.double() - want) + 2.0 ** -18 * norms(want)


def left_of(got, want):
    """want's distance from the numbers that round to got: what a 16-bit result shows of the error."""
    mag = got.abs()
    bits = mag.view(torch.int16)
    up = (bits + 1).view(got.dtype).double()
    down = torch.where(bits > 0, (bits - 1).clamp_min(0).view(got.dtype).double(), -up)
    low, high = (mag.double() + down) / 2, (mag.double() + up) / 2
    v = want * torch.where(got < 0, -1.0, 1.0)
    return (low - v).clamp_min(0) + (v - high).clamp_min(0)


# by path: one workgroup a matrix (sides up to 64; up to 32 and 64 x 128), columns in chunks, tiles of 64 x 64, of
# 128 x 64 and 128 x 128, Gram matrices summed in slices; odd sizes of each, wide and tall
SHAPES = [(5, 5), (17, 34), (33, 31), (64, 64), (3, 60, 48), (32, 128), (100, 20), (64, 128), (70, 50),
          (20, 1088), (34, 1088), (3946, 29), (51, 1088), (1088, 51), (300, 40, 500), (64, 7000),
          (65, 66), (128, 128), (257, 300), (300, 257), (3, 577, 1301), (6, 1088, 1088), (12, 1000, 1000),
          (333, 5000), (2, 5003, 97), (1, 65, 2111)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_is_accurate_to_float32(shape, dtype):
    g = gradient(shape, dtype, seed=31 + shape[-1])
    want = plain(g, torch.float64)
    got = ops.orthogonalize(g)
    err = got.double() - want if dtype == torch.float32 else left_of(got, want)
    limit = bound(want, plain(g.float(), torch.float32))
    assert bool((norms(err) <= limit).all()), f"{float((norms(err) / limit).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_muon_update_is_accurate_to_float32(shape, dtype):
    """From a parameter of zeros with lr = scale = 1 the new parameter is the direction itself, in float32."""
    g, m = gradient(shape, dtype, seed=5 + shape[-1]), gradient(shape, torch.float32, seed=6)
    beta = 0.5
    m64 = beta * m.double() + g.double()
    want = -plain(g.double() + beta * m64, torch.float64)
    m32 = beta * m + g.float()
    limit = bound(want, -plain(g.float() + beta * m32, torch.float32))
    p = torch.zeros(shape, device="cuda")
    ops.muon_update(p, m, g, lr=1.0, scale=1.0, beta=beta)
    assert bool((norms(p.double() - want) <= limit).all()), f"{float((norms(p.double() - want) / limit).max()):.3g} of the bound"
    assert bool(((m.double() - m64).abs() <= 2.0 ** -24 * m64.abs()).all())   # one rounding


def test_the_training_steps_update_is_accurate_to_float32():
    import lcn_oracle as O
    from lcn_testutil import make_cfg, make_network, perturbed_params, synthetic_batch
    cfg = make_cfg(F=64, L=1, knn=2)
    net = make_network(cfg, max_batch=96)
    net.set_optimizer("muon", momentum=0.5)
    net.set_params(O.flatten(cfg, perturbed_params(cfg, seed=21)))
    for step in range(2):
        x, lab = synthetic_batch(96, 2, seed=40 + step)
        before, m = net.get_params(), net.get_optimizer_state()[0]
        lr = float(np.float32(net.train_step(x, lab, update=False, keep_grads=True)[1]))
        grads = net.get_grads()
        net.train_step(x, lab)
        after = net.get_params()
        for name, off, shape in net.param_layout():
            if name[:3] not in ("w2_", "w3_"):
                continue
            sl = slice(off, off + shape[0] * shape[1])
            w, v, g, mom = (torch.from_numpy(t[sl].reshape(shape)) for t in (before, after, grads, m))
            scale = lr * float(np.float32(0.2) * np.sqrt(np.float32(shape[0])))
            o = plain(g.double() + 0.5 * (0.5 * mom.double() + g.double()), torch.float64)
            o32 = plain(g + 0.5 * (0.5 * mom + g), torch.float32)
            want = w.double() - scale * o
            # the direction's error; its product with the rate and the scale (two roundings) and the parameter's
            limit = scale * (bound(o, o32) + 2 * 2.0 ** -24 * norms(o)) + 2.0 ** -24 * norms(want)
            assert bool((norms(v.double() - want) <= limit).all())


# ---- infinities and NaN ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(24, 40), (50, 64), (20, 300), (51, 300), (80, 130), (130, 80), (333, 5000)])
def test_a_bad_matrix_stays_alone(shape, dtype):
    g = gradient((4,) + shape, dtype, 17)
    clean = ops.orthogonalize(g)
    p0, m0 = gradient((4,) + shape, torch.float32, 18), gradient((4,) + shape, torch.float32, 19)
    p, m = p0.clone(), m0.clone()
    ops.muon_update(p, m, g, lr=0.1)
    bad = g.clone()
    bad[0, -1, -1] = float("inf")
    bad[1, 0, 3] = float("-inf")
    bad[3, 7, -2] = float("nan")
    out = ops.orthogonalize(bad)
    pb, mb = p0.clone(), m0.clone()
    ops.muon_update(pb, mb, bad, lr=0.1)
    assert torch.equal(out[2], clean[2]) and torch.equal(pb[2], p[2])
    for i in (0, 1, 3):
        assert bool(out[i].isnan().all()) and bool(pb[i].isnan().all())
    # the momentum is an elementwise sum: bad where the gradient is
    good = bad.isfinite()
    assert torch.equal(mb[good], m[good]) and not bool(mb[~good].isfinite().any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,n", [(3, 130, 50), (14, 2520, 40), (40, 130, 50), (600, 1088, 1025), (2000, 96, 300), (16447, 130, 66), (16500, 1280, 130)])
def test_a_bad_token_stays_alone(t, k, n, dtype):
    x, w, s, b = int8_case(t, k, n, dtype, seed=t + k)
    bad = {0: float("inf"), t // 2: float("nan"), t - 1: float("-inf")}
    clean = x.clone()
    for i, (row, value) in enumerate(bad.items()):
        clean[row] = 0
        x[row, (0, k // 2, k - 1)[i]] = value
    for bias in (b, None):
        y, z = ops.int8_linear(x, w, s, bias), ops.int8_linear(clean, w, s, bias)
        for row in bad:
            assert bool(y[row].isnan().all())
            assert bool((z[row] == (0 if bias is None else bias.to(dtype))).all())
        rest = torch.ones(t, dtype=torch.bool, device="cuda")
        rest[list(bad)] = False
        assert torch.equal(y[rest], z[rest])
        int8_close(z, clean, w, s, bias)
