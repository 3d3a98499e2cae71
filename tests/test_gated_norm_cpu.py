"""Host side of the gated RMS norm's kernels, without a GPU."""
import contextlib

import torch

from xorl_b200.ops import _lib, norm


def test_partial_sums_are_sized_for_the_tensors_device(monkeypatch):
    """Two devices of different sizes, neither of them twice asked the same for the other's."""
    now = [0]

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    class Lib:
        def xb_gated_norm_partial(self, T, groups, d, shared):
            return (100, 148)[now[0]] * d

    monkeypatch.setattr(_lib, "cuda_lib", Lib)
    monkeypatch.setattr(torch.cuda, "device", device)
    norm._gated_norm_partial.cache_clear()
    try:
        assert [norm._gated_norm_partial(64, 2, 8, 1, i) for i in (0, 1, 0)] == [800, 1184, 800]
        assert now == [0]
    finally:
        norm._gated_norm_partial.cache_clear()
