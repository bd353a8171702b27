"""lcn_amd.ops beside torch's autograd: what gives no derivative says so."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

from lcn_amd import ops  # noqa: E402


def _operands():
    g = torch.Generator(device="cuda").manual_seed(1)
    return dict(a=torch.randn(24, 40, device="cuda", generator=g), b=torch.randn(24, 40, device="cuda", generator=g),
                c=torch.randn(24, 40, device="cuda", generator=g), x=torch.randn(7, 40, device="cuda", generator=g),
                q=torch.randint(-127, 128, (24, 40), device="cuda", generator=g, dtype=torch.int8),
                s=torch.rand(24, device="cuda", generator=g), bias=torch.rand(24, device="cuda", generator=g),
                lr=torch.full((1,), 0.01, device="cuda"))


CALLS = {
    "orthogonalize": (lambda o: ops.orthogonalize(o["a"]), ["a"]),
    "orthogonalize out": (lambda o: ops.orthogonalize(o["a"], out=o["b"]), ["a", "b"]),
    "muon_update": (lambda o: ops.muon_update(o["a"], o["b"], o["c"], lr=o["lr"]), ["a", "b", "c", "lr"]),
    "quantize_weight": (lambda o: ops.quantize_weight(o["a"]), ["a"]),
    "int8_linear": (lambda o: ops.int8_linear(o["x"], o["q"], o["s"], o["bias"]), ["x", "s", "bias"]),
}


@pytest.mark.parametrize("call", CALLS)
def test_forward_mode_tangents_are_refused(call):
    run, names = CALLS[call]
    with forward_ad.dual_level():
        for name in names:
            o = _operands()
            kept = {k: v.clone() for k, v in o.items()}
            o[name] = forward_ad.make_dual(o[name], torch.ones_like(o[name]))
            for context in (torch.enable_grad, torch.no_grad):   # forward mode goes on under no_grad
                with context(), pytest.raises(ValueError, match=f"^(g|w|{name}|param|momentum|grad|scale|out) carries"):
                    run(o)
            for k, v in o.items():                                # and nothing was written before the refusal
                assert torch.equal(forward_ad.unpack_dual(v).primal, kept[k])
        run(_operands())                                          # inside a level, plain tensors are as good as ever


def test_jvp_is_refused():
    o = _operands()
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(ops.orthogonalize, (o["a"],), (o["b"],))


def test_a_backward_through_an_updated_weight_is_an_error():
    """The graph saved the weight; the update changes it in place, and autograd has to know."""
    x = torch.randn(8, 24, device="cuda")
    for update in (lambda w: ops.muon_update(w, torch.zeros_like(w), torch.ones_like(w), lr=0.1),
                   lambda w: ops.orthogonalize(torch.ones_like(w), out=w)):
        w = torch.randn(24, 40, device="cuda", requires_grad=True)
        h = x.clone().requires_grad_() @ w
        with torch.no_grad():
            update(w)
        with pytest.raises(RuntimeError, match="inplace"):
            h.sum().backward()


def test_versions_count_what_was_written():
    o = _operands()
    versions = {k: v._version for k, v in o.items()}
    ops.muon_update(o["a"], o["b"], o["c"], lr=o["lr"])
    ops.orthogonalize(o["c"])
    ops.int8_linear(o["x"], o["q"], o["s"], o["bias"])
    ops.quantize_weight(o["c"])
    assert {k: v._version - versions[k] for k, v in o.items()} == dict.fromkeys(o, 0) | {"a": 1, "b": 1}
    wide = torch.zeros(3, 7, 30, device="cuda")
    before = wide._version
    ops.int8_linear(o["x"], o["q"], o["s"], out=wide[1, :, 2:26])  # a view counts for its base
    assert wide._version == before + 1
    ops.orthogonalize(o["c"], out=o["c"])
    assert o["c"]._version == versions["c"] + 1
    with pytest.raises(ValueError):
        ops.orthogonalize(o["c"], steps=0, out=o["a"])            # nothing written, nothing counted
    assert o["a"]._version == versions["a"] + 1
    with torch.inference_mode():
        p = torch.zeros(8, 9, device="cuda")
        ops.muon_update(p, torch.zeros_like(p), torch.ones_like(p), lr=0.1)
    ops.muon_update(p, torch.zeros(8, 9, device="cuda"), torch.ones(8, 9, device="cuda"), lr=0.1)   # has no counter
