"""An error of an earlier call does not become the operators' own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from lcn_amd import native, ops  # noqa: E402

NO_DEVICE = 99


def _calls(lib):
    """The four operators through the C ABI as functions of the device."""
    stream = torch.cuda.current_stream().cuda_stream
    a, b, c = (torch.randn(2, 80, 100, device="cuda") for _ in range(3))
    q, s = torch.empty(80, 100, dtype=torch.int8, device="cuda"), torch.empty(80, device="cuda")
    y = torch.empty(100, 80, device="cuda")
    ws = torch.empty(lib.lcn_orthogonalize_workspace(2, 80, 100), dtype=torch.uint8, device="cuda")
    coef = ops._triple(ops.MUON_COEFFICIENTS)
    x = torch.randn(100, 100, device="cuda")
    return [
        lambda d: lib.lcn_orthogonalize(d, stream, 0, 2, 80, 100, a.data_ptr(), 8000, 100, b.data_ptr(), 8000, 100, 5, coef, 1e-7,
                                        ws.data_ptr(), ws.numel()),
        lambda d: lib.lcn_muon_update(d, stream, 0, 2, 80, 100, a.data_ptr(), 8000, 100, b.data_ptr(), 8000, 100, c.data_ptr(), 8000,
                                      100, 0.1, None, 1.0, 0.9, 1, 0.0, 5, coef, 1e-7, ws.data_ptr(), ws.numel()),
        lambda d: lib.lcn_int8_quantize_weight(d, stream, 0, 80, 100, a.data_ptr(), 100, 1, q.data_ptr(), s.data_ptr()),
        lambda d: lib.lcn_int8_linear(d, stream, 0, 100, 100, 80, x.data_ptr(), 100, q.data_ptr(), 100, s.data_ptr(), None, y.data_ptr(),
                                      80, None, 0),
    ]


def test_a_refused_device_leaves_nothing_behind():
    lib = native.load_library()
    calls = _calls(lib)
    for call in calls:
        assert call(0) == 0
        assert call(NO_DEVICE) < 0 and lib.lcn_last_error(None)
        for other in calls:
            assert other(0) == 0, lib.lcn_last_error(None)
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize()


def test_a_failed_create_leaves_nothing_behind():
    from lcn_testutil import make_cfg, make_network
    lib = native.load_library()
    for call in _calls(lib):
        with pytest.raises(native.LcnNativeError):
            make_network(make_cfg(F=64, L=1, knn=1), max_batch=32, device=NO_DEVICE)
        assert call(0) == 0, lib.lcn_last_error(None)
    torch.cuda.synchronize()
