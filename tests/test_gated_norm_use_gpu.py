"""The gated RMS norm as programs use it: its entry points' refusals, an engine's gradient buffer.  Tolerances as in
test_gated_norm_gpu.py."""
import pytest
import torch

from test_gated_norm_gpu import _need_cuda, make  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [True, False])
def test_partial_sums_that_do_not_fit_are_refused(shared):
    """A buffer that is too small for the launch's blocks is refused before anything is launched."""
    from xorl_b200.ops import _lib
    T, group, groups = 300, 128, 4
    x, z, w, dy = make(T, group * groups, group if shared else group * groups)
    rstd = torch.ones(T, groups, device="cuda")
    dx, dz, dw = torch.empty_like(x), torch.empty_like(z), torch.empty_like(w)
    need = _lib.cuda_lib().xb_gated_norm_partial(T, groups, group, int(shared))
    part = torch.empty(need, device="cuda")

    def run(size):
        _lib.call_on(x.device, "xb_gated_norm_bwd", dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0),
                     w.data_ptr(), 0, int(shared), rstd.data_ptr(), dx.data_ptr(), dz.data_ptr(), part.data_ptr(), size,
                     dw.data_ptr(), 0, T, groups, group, 1)

    run(need)
    for size in (need - 1, 1, 0):
        with pytest.raises(RuntimeError, match="xb_gated_norm_bwd failed with code -1"):
            run(size)
