"""The scratch memory that the operators ask for (without a GPU)."""
import pytest

from lcn_amd import native


def up(v, to):
    return (v + to - 1) // to * to


@pytest.mark.parametrize("t,k,n", [(65536, 1088, 1088), (16384, 1216, 4352), (1 << 20, 64, 64), (1 << 24, 1088, 16), (16384, 1, 1)])
def test_tokens_that_stay_on_the_chip_take_no_memory(t, k, n):
    """Many tokens of moderate length are quantised into LDS: the weights, laid out once, are all there is."""
    assert native.load_library().lcn_int8_linear_workspace(t, k, n) == up(up(n, 64) * up(k, 64), 256)


@pytest.mark.parametrize("t,k,n", [(1, 1088, 1088), (16, 64, 64), (200, 1088, 1088), (777, 1003, 333)])
def test_few_tokens_take_none(t, k, n):
    assert native.load_library().lcn_int8_linear_workspace(t, k, n) == 0


@pytest.mark.parametrize("t,k,n", [(16384, 4352, 4352), (16383, 1088, 1088), (16384, 1217, 64)])
def test_other_tokens_go_through_memory(t, k, n):
    want = up(4 * t, 256) + up(t * up(k, 64), 256) + up(up(n, 64) * up(k, 64), 256)
    assert native.load_library().lcn_int8_linear_workspace(t, k, n) == want
