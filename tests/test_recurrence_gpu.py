"""The gated linear recurrences (gated delta rule, state-space scan) and their gradients against the token-by-token
definition in 64 bits.

Tolerances: an output in bf16 is rounded once (2^-8 of the value at most).  Before that, every computed operand of a
product is held as two bf16 values, off by at most 2^-17 of it, and low x low (2^-18) is left out; a result passes at
most four such products in a row with two operands each, so its error stays below 4 * 2 * (2^-17 + 2^-18) = 9.2e-5 of
what the sums add up (their largest value stands for it here), and below that fraction of the norm on average."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HELD = 4 * 2 * (2.0 ** -17 + 2.0 ** -18)


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from xorl_b200.ops import _lib
    _lib.cuda_lib()
    yield
    assert all(v == 0 for v in _lib.read_status()[:4]), _lib.read_status()


def oracle_delta(q, k, v, g, beta, cuts, scale, l2norm, s_in):
    """fp64, differentiable; rows outside the documents give zeros."""
    if l2norm:
        q, k = torch.nn.functional.normalize(q, dim=-1), torch.nn.functional.normalize(k, dim=-1)
    rep = v.shape[1] // q.shape[1]
    q, k = (scale * q).repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    rows, states = {}, []
    for d in range(len(cuts) - 1):
        S = s_in[d] if s_in is not None else q.new_zeros(v.shape[1], q.shape[2], v.shape[2]) + 0.0 * v.sum()
        for t in range(cuts[d], cuts[d + 1]):
            S = torch.exp(g[t]).view(-1, 1, 1) * S
            u = beta[t].unsqueeze(-1) * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
            S = S + k[t].unsqueeze(-1) * u.unsqueeze(1)
            rows[t] = torch.einsum("hkv,hk->hv", S, q[t])
        states.append(S)
    zero = 0.0 * v[0]                                                   # in the graph even where no row is
    return torch.stack([rows.get(t, zero) for t in range(v.shape[0])]), torch.stack(states) if states else None


def oracle_scan(x, dt, A, B, C, D, cuts, s_in):
    rep = x.shape[1] // B.shape[1]
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    rows, states = [], []
    T = x.shape[0]
    docs = [(0, cuts[0], None)] + [(cuts[i], cuts[i + 1], i) for i in range(len(cuts) - 1)] + [(cuts[-1], T, None)]
    for s, e, d in docs:
        S = s_in[d] if s_in is not None and d is not None else x.new_zeros(x.shape[1], x.shape[2], B.shape[2]) + 0.0 * x.sum()
        for t in range(s, e):
            S = torch.exp(dt[t] * A).view(-1, 1, 1) * S + (dt[t].unsqueeze(-1) * x[t]).unsqueeze(-1) * B[t].unsqueeze(1)
            rows.append(torch.einsum("hpn,hn->hp", S, C[t]) + D.unsqueeze(-1) * x[t])
        if d is not None:
            states.append(S)
    return torch.stack(rows), torch.stack(states) if states else None


def near(got, ref, name):
    assert got.shape == ref.shape and torch.isfinite(got).all(), name
    got, ref = got.double(), ref.detach()
    most = ref.abs().max().item() if ref.numel() else 0.0
    return got, ref, most


def check(got, ref, name):
    bf = got.dtype == torch.bfloat16
    g, r, most = near(got, ref, name)
    err = (g - r).abs()
    allowed = (2.0 ** -8 if bf else 2.0 ** -24) * r.abs() + HELD * most + 1e-30
    worst = (err - allowed).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{name}: off by {err.max().item():.3g} of {most:.3g}"
    if not bf and r.numel():
        assert (g - r).norm() <= HELD * r.norm() + 1e-30, f"{name}: norm off by {((g - r).norm() / r.norm()).item():.3g}"


def delta_inputs(T, hk, hv, dk, dv, docs, seed=0, state=False, strength=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    q, k, v = r(T, hk, dk).bfloat16(), r(T, hk, dk).bfloat16(), r(T, hv, dv).bfloat16()
    g = -strength * torch.nn.functional.softplus(r(T, hv))
    beta = torch.sigmoid(r(T, hv))
    return q, k, v, g, beta, (0.3 * r(docs, hv, dk, dv) if state else None)


def scan_inputs(T, groups, heads, N, P, docs, seed=0, state=False, strength=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, B, C = r(T, heads, P).bfloat16(), r(T, groups, N).bfloat16(), r(T, groups, N).bfloat16()
    dt = 0.1 * torch.nn.functional.softplus(r(T, heads))
    A, D = -strength * (1 + torch.arange(heads, device="cuda", dtype=torch.float32)), r(heads)
    return x, dt, A, B, C, D, (0.3 * r(docs, heads, P, N) if state else None)


def leaves(ts):
    return ([None if t is None else t.detach().requires_grad_() for t in ts],
            [None if t is None else t.detach().double().requires_grad_() for t in ts])


def run_delta(ins, cuts, scale=1.0, l2norm=True, final=True):
    from xorl_b200.ops.recurrence import gated_delta_rule
    a, b = leaves(ins)
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    o, S = gated_delta_rule(*a[:5], cu, scale=scale, qk_l2norm=l2norm, initial_state=a[5], return_final_state=True)
    ro, rS = oracle_delta(*b[:5], cuts, scale, l2norm, b[5])
    finish(a, b, o, S, ro, rS, ("q", "k", "v", "g", "beta", "initial_state"), final)


def run_scan(ins, cuts, final=True):
    from xorl_b200.ops.recurrence import ssd_scan
    a, b = leaves(ins)
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    y, S = ssd_scan(*a[:6], cu, initial_state=a[6], return_final_state=True)
    ry, rS = oracle_scan(*b[:6], cuts, b[6])
    finish(a, b, y, S, ry, rS, ("x", "dt", "A", "B", "C", "D", "initial_state"), final)


def finish(a, b, o, S, ro, rS, names, final):
    check(o.detach(), ro, "output")
    if rS is not None:
        check(S.detach(), rS, "final state")
    gen = torch.Generator(device="cuda").manual_seed(99)
    do = torch.randn(o.shape, generator=gen, device="cuda").bfloat16()
    outs, grads = [o], [do]
    routs, rgrads = [ro], [do.double()]
    if final and rS is not None:
        dS = torch.randn(S.shape, generator=gen, device="cuda")
        outs, grads, routs, rgrads = [o, S], [do, dS], [ro, rS], [do.double(), dS.double()]
    torch.autograd.backward(outs, grads)
    torch.autograd.backward(routs, rgrads)
    for x, y, n in zip(a, b, names):
        if x is not None:
            check(x.grad, y.grad if y.grad is not None else torch.zeros_like(y), "d" + n)


SHAPES = [  # T, shared heads, heads, state rows, state columns
    (1, 1, 1, 8, 8), (5, 2, 4, 8, 8), (63, 1, 2, 16, 24), (64, 2, 2, 64, 64), (65, 1, 3, 128, 128),
    (130, 2, 4, 72, 40), (200, 1, 2, 96, 80), (257, 2, 4, 128, 64), (129, 1, 2, 32, 136),
]


@pytest.mark.parametrize("T,hk,hv,dk,dv", SHAPES)
def test_delta_one_document(T, hk, hv, dk, dv):
    run_delta(delta_inputs(T, hk, hv, dk, dv, 1), [0, T], scale=dk ** -0.5)


@pytest.mark.parametrize("T,groups,heads,N,P", SHAPES)
def test_scan_one_document(T, groups, heads, N, P):
    run_scan(scan_inputs(T, groups, heads, N, P, 1), [0, T])


CUTS = [  # documents of one token, without tokens, rows before the first and behind the last
    [0, 1, 1, 2, 66, 130, 190], [3, 3, 70, 70, 71, 180], list(range(0, 191)), [0], [190], [0, 0, 0], [0, 64, 128, 190],
]


@pytest.mark.parametrize("cuts", CUTS, ids=["mixed", "outside", "tokens", "none", "tail", "empty", "aligned"])
@pytest.mark.parametrize("state", [False, True])
def test_delta_documents_and_states(cuts, state):
    run_delta(delta_inputs(190, 2, 4, 16, 24, len(cuts) - 1, seed=1, state=state and len(cuts) > 1), cuts, scale=0.25)


@pytest.mark.parametrize("cuts", CUTS, ids=["mixed", "outside", "tokens", "none", "tail", "empty", "aligned"])
@pytest.mark.parametrize("state", [False, True])
def test_scan_documents_and_states(cuts, state):
    run_scan(scan_inputs(190, 2, 4, 16, 24, len(cuts) - 1, seed=1, state=state and len(cuts) > 1), cuts)
