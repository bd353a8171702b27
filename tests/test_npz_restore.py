"""The earlier .npz payload, which holds Adam's state, restored under either optimiser (without a GPU)."""
import numpy as np
import pytest

from lcn_amd import checkpoint as ckpt
from test_optimizer_flags import _Net


@pytest.mark.parametrize("optimizer", ["adam", "muon"])
def test_adam_state_is_not_muons_momentum(tmp_path, optimizer):
    rng = np.random.default_rng(0)
    p, m, v = (rng.standard_normal(10).astype(np.float32) for _ in range(3))
    net = _Net(optimizer)
    np.savez(tmp_path / "model-7.npz", names=np.array([n for n, _, _ in net.param_layout()]), params=p, adam_m=m, adam_v=v,
             global_step=7, beta1_power=0.5, beta2_power=0.25)
    assert ckpt.restore(net, str(tmp_path / "model-7")) is None
    np.testing.assert_array_equal(net.p, p)
    assert net.rest == (7, 0.5, 0.25)
    hidden = 0 if optimizer == "adam" else 8        # w2_0 and w3_0 under Muon: the other optimiser's, so zero
    assert not net.m[:hidden].any() and not net.v[:hidden].any()
    np.testing.assert_array_equal(net.m[hidden:], m[hidden:])
    np.testing.assert_array_equal(net.v[hidden:], v[hidden:])
