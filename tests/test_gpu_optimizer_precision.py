"""Muon in the training step (lcn_set_optimizer) and 8-bit predictions (lcn_set_precision) of the
network handle, against 64-bit arithmetic on the handle's own tensors."""
import math
import os
import shutil

import numpy as np
import pytest
import torch

import lcn_oracle as O
from lcn_testutil import make_cfg, make_network, perturbed_params, synthetic_batch
from test_gpu_multirank import ThreadAllReduce, run_ranks

pytestmark = pytest.mark.gpu

MUON = (3.4445, -4.775, 2.0315)


def newton_schulz(u, steps=5):
    x = torch.from_numpy(np.asarray(u, np.float64))
    x = x / torch.linalg.norm(x)
    for _ in range(steps):
        a = x @ x.T
        x = MUON[0] * x + (MUON[1] * a + MUON[2] * a @ a) @ x
    return x.numpy()


def hidden(net):
    return [(n, off, shape) for n, off, shape in net.param_layout() if n[:3] in ("w2_", "w3_")]


@pytest.mark.parametrize("graphs", ["0", "1"])
def test_muon_step_updates_the_hidden_weights_and_adam_the_rest(graphs, monkeypatch):
    monkeypatch.setenv("LCN_GRAPHS", graphs)
    cfg = make_cfg(F=64, L=1, knn=2)
    theta = O.flatten(cfg, perturbed_params(cfg, seed=2))
    adam, muon = make_network(cfg, max_batch=96), make_network(cfg, max_batch=96)
    muon.set_optimizer("muon", momentum=0.9, weight_decay=0.1)
    adam.set_params(theta)
    muon.set_params(theta)
    names = hidden(muon)
    assert len(names) == 2
    buf = {n: np.zeros(s) for n, _, s in names}
    for step in range(3):
        x, lab = synthetic_batch(96, 2, seed=step)
        before = muon.get_params().astype(np.float64)
        adam.set_params(muon.get_params())      # the same weights: Adam's own variables move alike
        _, lr = muon.train_step(x, lab, update=False, keep_grads=True)
        grads = muon.get_grads().astype(np.float64)
        muon.train_step(x, lab)
        adam.train_step(x, lab)
        after, other = muon.get_params().astype(np.float64), adam.get_params()
        m = muon.get_optimizer_state()[0]
        rest = np.ones(after.size, bool)
        for n, off, shape in names:
            sl = slice(off, off + shape[0] * shape[1])
            rest[sl] = False
            g = grads[sl].reshape(shape)
            buf[n] = 0.9 * buf[n] + g
            o = newton_schulz(g + 0.9 * buf[n])
            scale = 0.2 * math.sqrt(1088)
            want = (1 - lr * 0.1) * before[sl].reshape(shape) - lr * scale * o
            got = after[sl].reshape(shape)
            # the gradients of two runs of the step are equal bits; a momentum takes one rounding a step, the
            # direction's error (2^-20 |a|^5 of its norm, the momentum's roundings below that) times the step,
            # and three roundings of the parameter
            bound = lr * scale * np.linalg.norm(o) * 2.0 ** -20 * MUON[0] ** 5 + 3 * 2.0 ** -24 * np.linalg.norm(want)
            assert np.linalg.norm(got - want) <= bound
            assert np.abs(m[sl].reshape(shape) - buf[n]).max() <= (2 + step) * 2.0 ** -24 * 2 * np.abs(buf[n]).max()
            buf[n] = m[sl].reshape(shape).astype(np.float64)
        np.testing.assert_array_equal(after[rest].astype(np.float32), other[rest])
    with pytest.raises(Exception):
        muon.get_grads()                          # the last step kept none, and used their buffer


def test_back_to_adam_is_adam():
    cfg = make_cfg(F=64, L=1, knn=1)
    theta = O.flatten(cfg, perturbed_params(cfg, seed=3))
    a, b = make_network(cfg, max_batch=64), make_network(cfg, max_batch=64)
    b.set_optimizer("muon")
    b.set_optimizer("adam")
    for net in (a, b):
        net.set_params(theta)
        for step in range(2):
            net.train_step(*synthetic_batch(64, 2, seed=step))
    np.testing.assert_array_equal(a.get_params(), b.get_params())


def test_refusals():
    net = make_network(make_cfg(F=64, L=1, knn=1), max_batch=32)
    for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(weight_decay=float("inf")), dict(steps=0),
               dict(steps=65), dict(momentum=float("nan"))):
        with pytest.raises(Exception, match="Muon"):
            net.set_optimizer("muon", **kw)
    assert net.optimizer == "adam"
    with pytest.raises(ValueError):
        net.set_optimizer("sgd")
    with pytest.raises(ValueError):
        net.set_precision("int4")
    flat = make_network(make_cfg(F=64, L=0, knn=1), max_batch=32)
    with pytest.raises(Exception, match="hidden layer"):
        flat.set_optimizer("muon")
    flat.set_precision("int8")                    # nothing to do, and nothing breaks
    x, _ = synthetic_batch(32, 2, seed=0)
    out = flat.forward(x)
    flat.set_precision("fp32")
    np.testing.assert_array_equal(out, flat.forward(x))


def effective_weight(cfg, params, name):
    """W_e = clip(W) (.) M of a hidden layer, 64-bit (oracle)."""
    M, _ = O.mask_value(cfg, params, np.float64)
    w = np.asarray(params[name], np.float64)
    if cfg.max_norm:
        w = w / max(np.linalg.norm(w), 1.0)
    return w * np.kron(M, np.ones((cfg.F, cfg.F)))


def check_layer(z, a, we, bias):
    """z of the device against a . We: each 8-bit rounding moves a factor by at most half a step."""
    s, t = np.abs(a).max(1, keepdims=True) / 127, np.abs(we).max(0, keepdims=True) / 127
    exact = a @ we + bias
    bound = 0.5 * s * np.abs(we).sum(0) + 0.5 * t * np.abs(a).sum(1, keepdims=True) + 0.25 * s * t * a.shape[1]
    err = np.abs(z - exact)
    # roundings of fp32 on the way (factors, sums, scales): 2^-20 of the sum of magnitudes covers them
    assert (err <= bound * (1 + 1e-3) + 2.0 ** -20 * (np.abs(a) @ np.abs(we) + np.abs(bias))).all()
    # and it is 8-bit arithmetic that comes out.  A factor's rounding has a root mean square of s / sqrt(12)
    # with s >= rms / 127: 2.3e-3 of the factor, and, the signs being independent, of the product; 1e-4 of the
    # product (without the bias, which is not rounded) is a twentieth of that and a thousand float32 roundings
    assert err.mean() > 1e-4 * np.abs(exact - bias).mean()


@pytest.mark.parametrize("kw", [dict(F=64, L=2, knn=3), dict(F=64, L=1, knn=1, residual=False),
                                dict(F=128, L=1, knn=2, in_F=3), dict(F=64, L=1, mask="exponential"),
                                dict(F=64, L=1, knn=2, batch_norm=False)])
@pytest.mark.parametrize("batch", [1, 33, 130, 300])
def test_int8_hidden_layers(kw, batch):
    cfg = make_cfg(**kw)
    params = perturbed_params(cfg, seed=4)
    net = make_network(cfg, max_batch=300)
    net.set_params(O.flatten(cfg, params))
    net.set_precision("int8")
    x, _ = synthetic_batch(batch, cfg.in_F, seed=batch)
    out = net.forward(x)
    assert np.isfinite(out).all()
    H = 17 * cfg.F
    for l in range(cfg.num_layers):
        k1, k2 = 2 * l + 1, 2 * l + 2
        h = net.debug_tensor(1, l, batch * H).reshape(batch, H).astype(np.float64)
        z1 = net.debug_tensor(0, k1, batch * H).reshape(batch, H).astype(np.float64)
        z2 = net.debug_tensor(0, k2, batch * H).reshape(batch, H).astype(np.float64)
        check_layer(z1, h, effective_weight(cfg, params, f"w2_{l}"), np.asarray(params[f"b2_{l}"], np.float64).ravel())
        if cfg.batch_norm:
            st = net.debug_tensor(2, k1, 2 * cfg.F).astype(np.float64)
            mean, rstd = np.tile(st[:cfg.F], 17), np.tile(st[cfg.F:], 17)
            # the statistics of the 8-bit z
            zc = z1.reshape(batch * 17, cfg.F)
            np.testing.assert_allclose(st[:cfg.F], zc.mean(0), rtol=0, atol=2.0 ** -18 * np.abs(zc).max())
            u = (z1 - mean) * rstd * np.tile(params[f"bn1{l}_gamma"].ravel(), 17) + np.tile(params[f"bn1{l}_beta"].ravel(), 17)
        else:
            u = z1
        check_layer(z2, np.where(u > 0, u, 0.2 * u), effective_weight(cfg, params, f"w3_{l}"),
                    np.asarray(params[f"b3_{l}"], np.float64).ravel())
    # training steps are float32 whatever the precision
    other = make_network(cfg, max_batch=300)
    other.set_params(O.flatten(cfg, params))
    xt, lab = synthetic_batch(max(batch, 2), cfg.in_F, seed=9)
    assert net.train_step(xt, lab) == other.train_step(xt, lab)
    np.testing.assert_array_equal(net.get_params(), other.get_params())
    net.set_precision("fp32")
    np.testing.assert_array_equal(net.forward(x), other.forward(x))


def test_muon_replicas_of_two_ranks_stay_equal():
    """The update follows the all-reduced gradients: both ranks' weights and momenta are the same bits, and the
    hidden weights move by the orthogonalised direction of the gradient the ranks report."""
    cfg = make_cfg(F=64, L=1, knn=2)
    theta = O.flatten(cfg, perturbed_params(cfg, seed=7))
    x, lab = synthetic_batch(96, 2, seed=3)
    ar = ThreadAllReduce(2)

    def rank(r):
        net = make_network(cfg, max_batch=64)
        net.comm_init_host(r, 2, ar.for_rank(r))
        net.set_optimizer("muon", momentum=0.9)
        net.set_params(theta)
        part = slice(0, 40) if r == 0 else slice(40, 96)
        lr = net.train_step(x[part], lab[part], update=False, keep_grads=True)[1]
        grads = net.get_grads()
        net.train_step(x[part], lab[part])
        first = net.get_params()
        net.train_step(x[part], lab[part])
        out = grads, first, net.get_params(), net.get_optimizer_state()[0], lr, hidden(net)
        net.close()
        return out

    one, two = run_ranks(2, rank)
    for a, b in zip(one[:4], two[:4]):
        np.testing.assert_array_equal(a, b)
    grads, first, _, _, lr, names = one
    for n, off, shape in names:
        sl = slice(off, off + shape[0] * shape[1])
        o = newton_schulz(1.9 * grads[sl].reshape(shape).astype(np.float64))   # g + 0.9 g, at any scale
        want = theta[sl].reshape(shape) - lr * 0.2 * math.sqrt(1088) * o
        # as above: the direction's error, then the parameter's roundings
        bound = lr * 0.2 * math.sqrt(1088) * np.linalg.norm(o) * 2.0 ** -20 * MUON[0] ** 5 + 3 * 2.0 ** -24 * np.linalg.norm(want)
        assert np.linalg.norm(first[sl].reshape(shape) - want) <= bound


def test_int8_poses_of_two_ranks():
    """Without batch statistics a pose's prediction depends on nothing but the pose."""
    cfg = make_cfg(F=64, L=1, knn=2, batch_norm=False)
    theta = O.flatten(cfg, perturbed_params(cfg, seed=8))
    x, _ = synthetic_batch(96, 2, seed=4)
    ar = ThreadAllReduce(2)

    def rank(r):
        net = make_network(cfg, max_batch=64)
        net.comm_init_host(r, 2, ar.for_rank(r))
        net.set_params(theta)
        net.set_precision("int8")
        out = net.forward(x[:40] if r == 0 else x[40:])
        net.close()
        return out

    parts = run_ranks(2, rank)
    whole = make_network(cfg, max_batch=96)
    whole.set_params(theta)
    whole.set_precision("int8")
    np.testing.assert_array_equal(np.concatenate(parts), whole.forward(x))


def test_int8_predict_dataset_and_repeats():
    cfg = make_cfg(F=64, L=2, knn=3)
    net = make_network(cfg, max_batch=128)
    net.set_params(O.flatten(cfg, perturbed_params(cfg, seed=5)))
    x, lab = synthetic_batch(200, 2, seed=1)
    net.dataset_upload(0, x)
    net.dataset_upload(1, lab)
    fp = net.predict_dataset(0, 200, 128)
    net.set_precision("int8")
    a, loss = net.predict_dataset(0, 200, 128, lab_slot=1)
    b = net.predict_dataset(0, 200, 128)
    np.testing.assert_array_equal(a, b)
    assert len(loss) == 2 and np.isfinite(loss).all()
    assert not np.array_equal(a, fp)
    one = net.forward(x[:128])
    np.testing.assert_array_equal(a[:128].astype(np.float32), one)   # the same kernels behind both entries


def test_int8_nan_stays_in_its_pose_without_batch_statistics():
    cfg = make_cfg(F=64, L=1, knn=1, batch_norm=False)
    net = make_network(cfg, max_batch=64)
    net.set_params(O.flatten(cfg, perturbed_params(cfg, seed=6)))
    net.set_precision("int8")
    x, _ = synthetic_batch(64, 2, seed=2)
    want = net.forward(x)
    x[7, 3] = np.nan
    got = net.forward(x)
    assert np.isnan(got[7]).any()
    keep = np.arange(64) != 7
    np.testing.assert_array_equal(got[keep], want[keep])


@pytest.fixture
def model_dir():
    name = "pytest_gpu_muon"
    yield name
    from network import models_att
    shutil.rmtree(os.path.join(os.path.dirname(models_att.__file__), "..", "experiment", name), ignore_errors=True)


def test_cgcnn_trains_with_muon_and_predicts_in_8_bits(model_dir, monkeypatch):
    """One user's run: fit with Muon, its checkpoint, predictions of a second model in 8 bits."""
    from lcn_amd import checkpoint as ckpt
    from network.models_att import cgcnn
    from tools import filter_hub, params_help
    monkeypatch.setenv("LCN_INIT_SEED", "3")
    rng = np.random.default_rng(0)
    x = rng.uniform(-1, 1, size=(256, 34))
    y = np.concatenate([x.reshape(256, 17, 2), rng.uniform(-1, 1, (256, 17, 1))], 2).reshape(256, 51)
    p = params_help.get_params(is_training=True)
    p.update(dict(dir_name=model_dir, num_epochs=1, batch_size=64, F=64, num_layers=1, knn=2, init_type="same", dropout=0,
                  neighbour_matrix=params_help.get_neighbour_matrix_by_hand(filter_hub.neighbour_dict_set[0], knn=2),
                  optimizer="muon"))
    model = cgcnn(**p)
    assert model._net.optimizer == "muon"
    losses, _ = model.fit(x, y, x[:100], y[:100])
    assert len(losses) == 1 and np.isfinite(losses).all()
    prefix = ckpt.latest_checkpoint(os.path.join(model._get_path("checkpoints"), "final"))
    from lcn_amd import tf_bundle
    t = tf_bundle.read_bundle(prefix)
    key = "linear_model/two_linear_0/w2_0"
    m = model._net.get_optimizer_state()[0]
    off, shape = [(o, s) for n, o, s in model._net.param_layout() if n == "w2_0"][0]
    np.testing.assert_array_equal(t[key + "/Momentum"], m[off:off + shape[0] * shape[1]].reshape(shape))
    assert key + "/Adam" not in t and np.abs(t[key + "/Momentum"]).max() > 0
    # Adam does not take the momentum for its own state, Muon does
    fresh = cgcnn(**p)
    ckpt.restore(fresh._net, prefix)
    np.testing.assert_array_equal(fresh._net.get_optimizer_state()[0], m)
    plain = cgcnn(**dict(p, optimizer="adam"))
    ckpt.restore(plain._net, prefix)
    got = plain._net.get_optimizer_state()[0]
    assert not got[off:off + shape[0] * shape[1]].any() and got.any()

    eight = cgcnn(**dict(p, optimizer="adam", precision="int8"))
    fp, q = plain.predict(x[:100]), eight.predict(x[:100])
    assert q.shape == (100, 51) and np.isfinite(q).all() and not np.array_equal(q, fp)
    tta = eight.predict_tta(x[:100], flip=True)
    assert tta.shape == (100, 51) and np.isfinite(tta).all()
