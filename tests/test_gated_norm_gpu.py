"""The gated RMS norm and its gradients against the formula in 64 bits.

Tolerances: x, gate and dy are bf16; outputs are rounded once (2^-8 of the value at most for bf16).  What is computed
before is fp32: the sum of d squares in a tree is off by at most (d / 256 + 10) * 2^-24 of it, exp and its quotient by
2^-20; ten such factors in a row stay below 2^-16 of the terms, whose largest stands for them here.  A weight's gradient
adds T * groups terms of that error in fp32 and stays below 2^-15 of the sum of their sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from xorl_b200.ops import _lib
    _lib.cuda_lib()
    yield
    assert all(v == 0 for v in _lib.read_status()[:4]), _lib.read_status()


def oracle(x, z, w, group, eps, first):
    act = z / (1 + torch.exp(-z))
    h = (x if first else x * act).unflatten(-1, (-1, group))
    h = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.view(-1, group)).flatten(-2)
    return h * act if first else h


def run(x, z, w, dy, group, first, eps=1e-6):
    from xorl_b200.ops.norm import gated_rms_norm
    a = [t.detach().requires_grad_() for t in (x, z, w)]
    b = [t.detach().double().requires_grad_() for t in (x, z, w)]
    y, r = gated_rms_norm(*a, group, eps, norm_first=first), oracle(*b, group, eps, first)
    y.backward(dy)
    r.backward(dy.double())
    for name, got, ref in (("y", y.detach(), r.detach()), ("x", a[0].grad, b[0].grad), ("gate", a[1].grad, b[1].grad)):
        assert got.dtype == torch.bfloat16 and got.shape == ref.shape and torch.isfinite(got).all(), name
        err, most = (got.double() - ref).abs(), ref.abs().max() if ref.numel() else 0
        assert bool((err <= 2.0 ** -8 * ref.abs() + 2.0 ** -16 * most + 1e-30).all()), (name, err.max())
    # the sum of the sizes of a weight gradient's terms
    act = b[1].detach() / (1 + torch.exp(-b[1].detach()))
    h = (b[0].detach() if first else b[0].detach() * act).unflatten(-1, (-1, group))
    n = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)).flatten(-2)
    size = (dy.double() * n * (act if first else 1)).abs()
    size = size.reshape(-1, group).sum(0) if w.numel() == group else size.reshape(-1, w.numel()).sum(0)
    got, ref = a[2].grad, b[2].grad
    assert got.dtype == w.dtype
    step = 2.0 ** -8 if w.dtype == torch.bfloat16 else 2.0 ** -24
    assert bool(((got.double() - ref).abs() <= step * ref.abs() + 2.0 ** -15 * size + 1e-30).all())


def make(T, W, n, wdtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return r(T, W).bfloat16(), r(T, W).bfloat16(), (1 + 0.3 * r(n)).to(wdtype), r(T, W).bfloat16()


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("T,group,groups", [(1, 8, 1), (3, 64, 3), (37, 72, 5), (130, 128, 32), (65, 256, 2), (33, 264, 3),
                                            (17, 512, 4), (19, 1000, 2), (40, 1024, 8), (9, 1032, 3), (21, 4096, 2),
                                            (5, 8192, 1), (1000, 8, 2)])
@pytest.mark.parametrize("shared", [True, False])
def test_gated_norm(T, group, groups, first, shared):
    x, z, w, dy = make(T, group * groups, group if shared else group * groups)
    run(x, z, w, dy, group, first)


@pytest.mark.parametrize("first", [True, False])
def test_fp32_weight_and_strided_rows(first):
    x, z, w, dy = make(50, 512, 512, torch.float32, seed=3)
    wide = torch.cat([z, x, dy, z[:, :8]], 1)
    run(wide[:, 512:1024], wide[:, :512], w, wide[:, 1024:1536], 128, first)          # rows of a wider matrix
    run(wide[:, 4:516], wide[:, 5:517], w, dy, 128, first)                            # rows that start off 16 bytes
    run(x.t().contiguous().t(), z, w, dy, 128, first)                                 # columns contiguous


@pytest.mark.parametrize("first", [True, False])
def test_extreme_values(first):
    """Zero rows, rows of one sign, gates far from zero: nothing but finite numbers, and the formula's."""
    x, z, w, dy = make(16, 256, 128, seed=4)
    x[0] = 0
    z[1], z[2] = 80.0, -80.0
    x[3] = 1e-18
    x[4] *= 1e4
    run(x, z, w, dy, 128, first)


def test_batch_dimensions_and_no_rows():
    from xorl_b200.ops.norm import gated_rms_norm
    x, z, w, dy = make(12, 256, 256, seed=5)
    y = gated_rms_norm(x.view(3, 4, 256), z.view(3, 4, 256), w, 128)
    assert torch.equal(y.view(12, 256), gated_rms_norm(x, z, w, 128))
    e = x[:0].detach().requires_grad_()
    wl = w.detach().requires_grad_()
    gated_rms_norm(e, z[:0], wl, 128).sum().backward()
    assert e.grad.shape == (0, 256) and bool((wl.grad == 0).all())


def test_same_bits_twice_and_in_a_graph():
    from xorl_b200.ops.norm import gated_rms_norm
    x, z, w, dy = make(777, 1024, 128, seed=6)

    def both():
        leaves = [t.detach().requires_grad_() for t in (x, z, w)]
        y = gated_rms_norm(*leaves, 128, norm_first=True)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    first = [t.clone() for t in both()]
    for a, b in zip(first, both()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    x.mul_(0.5)
    graph.replay()
    for a, b in zip([t.clone() for t in outs], both()):
        assert torch.equal(a, b)
