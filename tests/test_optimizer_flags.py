"""The flags and parameters of the additions to the reference's CLIs, without a GPU."""
import numpy as np
import pytest

from lcn_amd import checkpoint as ckpt


def test_flags_are_absent_unless_given():
    from tools import cli_flags, params_help
    base = ["--train_set", "h36m", "--validation_set", "h36m"]
    assert not hasattr(cli_flags.parse("train", base), "optimizer")
    args = cli_flags.parse("train", base + ["--optimizer", "muon"])
    params = params_help.get_params(is_training=True)
    assert "optimizer" not in params
    params_help.update_parameters(args, params)
    assert params["optimizer"] == "muon" and "precision" not in params
    inf = ["--train_set", "h36m", "--test_set", "h36m"]
    args = cli_flags.parse("inference", inf + ["--precision", "int8"])
    params = params_help.get_params(is_training=True)
    params_help.update_parameters(args, params)
    assert params["precision"] == "int8"
    for prog, argv in (("train", base + ["--optimizer", "sgd"]), ("inference", inf + ["--precision", "int4"]),
                       ("train", base + ["--precision", "int8"]), ("inference", inf + ["--optimizer", "muon"])):
        with pytest.raises(SystemExit):
            cli_flags.parse(prog, argv)


class _Net:
    """What checkpoint.py asks of a network: two hidden weights and a bias."""
    def __init__(self, optimizer):
        self.optimizer = optimizer
        self.n_params = 4 + 4 + 2
        self.p, self.m, self.v = (np.arange(10, dtype=np.float32) + 10 * i for i in range(3))

    def param_layout(self):
        return [("w2_0", 0, (2, 2)), ("w3_0", 4, (2, 2)), ("b1", 8, (2,))]

    def get_params(self):
        return self.p

    def get_optimizer_state(self):
        return self.m, self.v, 7, 0.5, 0.25

    def set_params(self, p):
        self.p = p

    def set_optimizer_state(self, m, v, *rest):
        self.m, self.v, self.rest = m, v, rest


def test_momentum_has_a_slot_of_its_own(tmp_path):
    muon = _Net("muon")
    prefix = ckpt.save(muon, str(tmp_path / "model"), 7)
    t = ckpt.to_tensors(muon)
    assert "linear_model/two_linear_0/w2_0/Momentum" in t and "linear_model/two_linear_0/w2_0/Adam" not in t
    assert "linear_model/b1/Adam" in t and "linear_model/b1/Adam_1" in t
    back = _Net("muon")
    ckpt.restore(back, prefix)
    np.testing.assert_array_equal(back.m, muon.m)
    np.testing.assert_array_equal(back.v[8:], muon.v[8:])
    assert not back.v[:8].any()
    adam = _Net("adam")
    ckpt.restore(adam, prefix)
    assert not adam.m[:8].any() and not adam.v[:8].any()
    np.testing.assert_array_equal(adam.m[8:], muon.m[8:])
    prefix = ckpt.save(_Net("adam"), str(tmp_path / "adam" / "model"), 7)
    back = _Net("muon")
    ckpt.restore(back, prefix)
    assert not back.m[:8].any()
    np.testing.assert_array_equal(back.m[8:], _Net("adam").m[8:])
