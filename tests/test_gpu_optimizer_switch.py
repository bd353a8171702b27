"""A change of the hidden weights' optimiser on a handle that has run steps (lcn_set_optimizer)."""
import numpy as np
import pytest

import lcn_oracle as O
from lcn_testutil import make_cfg, make_network, perturbed_params, synthetic_batch

pytestmark = pytest.mark.gpu


def _hidden(net):
    keep = np.zeros(net.n_params, bool)
    for name, off, shape in net.param_layout():
        if name[:3] in ("w2_", "w3_"):
            keep[off:off + shape[0] * shape[1]] = True
    return keep


def _like(net, cfg, kind):
    """A handle that never ran another optimiser: net's weights and state, the hidden weights' state zero."""
    other = make_network(cfg, max_batch=64)
    if kind == "muon":
        other.set_optimizer("muon")
    other.set_params(net.get_params())
    m, v, gs, b1p, b2p = net.get_optimizer_state()
    hidden = _hidden(net)
    m[hidden] = 0
    v[hidden] = 0
    other.set_optimizer_state(m, v, gs, b1p, b2p)
    return other


@pytest.mark.parametrize("graphs", ["0", "1"])
def test_each_optimiser_starts_from_its_own_state(graphs, monkeypatch):
    monkeypatch.setenv("LCN_GRAPHS", graphs)
    cfg = make_cfg(F=64, L=1, knn=2)
    net = make_network(cfg, max_batch=64)
    net.set_params(O.flatten(cfg, perturbed_params(cfg, seed=11)))
    hidden = _hidden(net)
    batches = [synthetic_batch(64, 2, seed=i) for i in range(9)]
    for x, lab in batches[:3]:
        net.train_step(x, lab)
    for kind, run in (("muon", batches[3:6]), ("adam", batches[6:])):
        before = net.get_optimizer_state()
        assert np.abs(before[0][hidden]).max() > 0
        fresh = _like(net, cfg, kind)
        net.set_optimizer(kind)
        after = net.get_optimizer_state()
        for old, new in zip(before[:2], after[:2]):
            assert not new[hidden].any()
            np.testing.assert_array_equal(new[~hidden], old[~hidden])
        assert before[2:] == after[2:]
        for x, lab in run:
            net.train_step(x, lab)
            fresh.train_step(x, lab)
            np.testing.assert_array_equal(net.get_params(), fresh.get_params())
            for a, b in zip(net.get_optimizer_state(), fresh.get_optimizer_state()):
                np.testing.assert_array_equal(a, b)


def test_new_arguments_keep_the_momentum():
    cfg = make_cfg(F=64, L=1, knn=1)
    net = make_network(cfg, max_batch=64)
    net.set_params(O.flatten(cfg, perturbed_params(cfg, seed=12)))
    net.set_optimizer("muon")
    net.train_step(*synthetic_batch(64, 2, seed=0))
    before = net.get_optimizer_state()[0]
    net.set_optimizer("muon", momentum=0.5, weight_decay=0.01)
    np.testing.assert_array_equal(net.get_optimizer_state()[0], before)
    with pytest.raises(Exception, match="Muon"):
        net.set_optimizer("muon", steps=0)       # a refused call changes nothing
    np.testing.assert_array_equal(net.get_optimizer_state()[0], before)
    assert before[_hidden(net)].any()
