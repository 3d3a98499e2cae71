"""Boundaries that do not ascend from 0 to the number of rows: the kernels clamp them, touch nothing else and report."""
import pytest
import torch

from test_recurrence_gpu import delta_inputs, scan_inputs
from test_recurrence_use_gpu import OPS, both_ways, boundaries, call, inputs, same

pytestmark = pytest.mark.gpu

BAD = {"behind the rows": [0, 70, 301], "first behind the rows": [301, 301, 301], "before the rows": [-1, 70, 300], "down": [0, 200, 100],
       "down to the first": [100, 300, 0], "far": [0, 2 ** 31 - 1, 2 ** 31 - 1], "alone": [301], "alone, before": [-5]}


def reported():
    from xorl_b200.ops import _lib
    status = _lib.read_status()
    assert status[:2] in ([0, 0], [3, 13]), status            # an argument, the recurrences
    return status[0] == 3


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("cuts", BAD.values(), ids=BAD.keys())
def test_bad_boundaries_are_reported(op, cuts):
    good = boundaries([0, 100, 300])
    ts, ok = inputs(op, docs=len(cuts) - 1, state=len(cuts) > 1), inputs(op, docs=2)
    want = both_ways(op, ok, good)
    assert not reported()
    with torch.no_grad():
        call(op, ts, boundaries(cuts))
    assert reported()
    if ts[-1] is not None:
        both_ways(op, ts, boundaries(cuts))
        assert reported()
    same(want, both_ways(op, ok, good))
    assert not reported()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T", [16, 48])
@pytest.mark.parametrize("cuts", [[0, 1, 2, 9], [0, 5, 4, 8], [-1, 1, 2, 8], [9, 9, 9, 9]])
def test_bad_boundaries_of_few_tokens_are_reported(op, T, cuts):
    """With and without a plan behind the token-by-token kernels."""
    cuts = [c + T - 8 if c > 2 else c for c in cuts]
    ts = list((delta_inputs if op == "delta" else scan_inputs)(T, 2, 4, 16, 24, 3, state=True))
    with torch.no_grad():
        call(op, ts, boundaries([0, 1, 2, T]))
        assert not reported()
        call(op, ts, boundaries(cuts))
    assert reported()
    both_ways(op, ts, boundaries(cuts))
    assert reported()
