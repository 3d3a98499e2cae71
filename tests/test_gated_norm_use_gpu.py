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


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_weight_gradient_into_an_engines_buffer(first, shared, wdtype):
    """fp32 sums in the buffer: the first pass writes over what lies there, the second adds, autograd gets none."""
    from xorl_b200.ops.norm import gated_rms_norm
    T, group, groups = 300, 72, 5
    x, z, w, dy = make(T, group * groups, group if shared else group * groups, wdtype)
    plain = w.detach().requires_grad_()
    xi, zi = x.detach().requires_grad_(), z.detach().requires_grad_()
    want = torch.autograd.grad(gated_rms_norm(xi, zi, plain, group, norm_first=first), [xi, zi, plain], dy)
    p = torch.nn.Parameter(w.detach().clone())
    p._xb_grad_buf, p._xb_grad_fresh = torch.full(w.shape, 7.0, device="cuda"), True
    X, Z, W, D = x.double(), z.double(), w.double().requires_grad_(), dy.double()
    act = Z / (1 + torch.exp(-Z))
    h = (X if first else X * act).unflatten(-1, (-1, group))
    n = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)).flatten(-2) * (act if first else 1)
    terms = (D * n).reshape(-1, w.numel())
    for k in (1, 2):
        xi, zi = x.detach().requires_grad_(), z.detach().requires_grad_()
        gated_rms_norm(xi, zi, p, group, norm_first=first).backward(dy)
        assert p.grad is None and not p._xb_grad_fresh
        assert torch.equal(xi.grad, want[0]) and torch.equal(zi.grad, want[1])
        err = (p._xb_grad_buf.double() - k * terms.sum(0)).abs()
        # the kernel's sum, its rounding, and that of the addition
        assert bool((err <= 2 * 2.0 ** -24 * k * terms.sum(0).abs() + k * 2.0 ** -15 * terms.abs().sum(0)).all())
