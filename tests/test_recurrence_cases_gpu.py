"""Documents of a few tokens beside others' infinities and with decays that leave nothing, and heads shared by many.
Tolerances as in test_recurrence_gpu.py."""
import pytest
import torch

from test_recurrence_gpu import _need_cuda, check, delta_inputs, oracle_delta, run_delta, run_scan, scan_inputs  # noqa: F401
from test_recurrence_use_gpu import NAMES, OPS, both_ways, boundaries, call, inputs, same

pytestmark = pytest.mark.gpu

SHORT = [0, 3, 4, 20, 21, 33, 34]                # documents of 3, 1, 16, 1, 12 and 1 tokens


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("doc", [0, 1, 2, 5])
def test_short_documents_keep_their_neighbours_values_out(op, value, doc):
    """A document of Inf or NaN, state and gradients included: the others' bits stay, with and without gradients."""
    cu, n = boundaries(SHORT), len(SHORT) - 1
    s, e = SHORT[doc], SHORT[doc + 1]
    ts = inputs(op, T=36, docs=n, seed=5)
    rows = [i for i, name in enumerate(NAMES[op]) if name not in ("A", "D", "initial_state")]
    bad = [t.clone() for t in ts]
    for i in rows:
        bad[i][s:e] = value
    bad[-1][doc] = value
    gen = torch.Generator(device="cuda").manual_seed(4)
    do, dS = torch.randn(bad[0].shape[0], 4, 64, generator=gen, device="cuda").bfloat16(), torch.randn(bad[-1].shape, generator=gen, device="cuda")
    bad_do, bad_dS = do.clone(), dS.clone()
    bad_do[s:e], bad_dS[doc] = value, value

    def run(us, d):
        leaves = [t.detach().requires_grad_() for t in us]
        o, S = call(op, leaves, cu)
        return o.detach(), S.detach(), torch.autograd.grad([o, S], leaves, d)

    (o, S, g), (o2, S2, g2) = run(ts, [do, dS]), run(bad, [bad_do, bad_dS])
    keep, docs = [t for t in range(36) if not s <= t < e], [d for d in range(n) if d != doc]
    assert torch.equal(o[keep], o2[keep]) and torch.equal(S[docs], S2[docs])
    for i in rows:
        assert torch.equal(g[i][keep], g2[i][keep]), NAMES[op][i]
    assert torch.equal(g[-1][docs], g2[-1][docs])
    with torch.no_grad():
        o3, S3 = call(op, bad, cu)
    assert torch.equal(o[keep], o3[keep]) and torch.equal(S[docs], S3[docs])


def test_delta_strong_decays_of_few_tokens():
    ts = delta_inputs(36, 1, 2, 32, 32, len(SHORT) - 1, seed=3, state=True)
    g = ts[3]
    g[0], g[3], g[10], g[11], g[20], g[34] = -float("inf"), -1e4, -130.0, 0.0, -float("inf"), -float("inf")
    ts[4][5], ts[4][6] = 0.0, 1.0
    live, ref = [t.detach().requires_grad_() for t in ts], [t.detach().double().requires_grad_() for t in ts]
    from xorl_b200.ops.recurrence import gated_delta_rule
    o, S = gated_delta_rule(*live[:5], boundaries(SHORT), scale=0.2, qk_l2norm=True, initial_state=live[5], return_final_state=True)
    ro, rS = oracle_delta(*ref[:5], SHORT, 0.2, True, ref[5])
    check(o.detach(), ro, "o")
    check(S.detach(), rS, "S")
    do, dS = torch.randn_like(ro).bfloat16(), torch.randn_like(rS).float()
    got = torch.autograd.grad([o, S], live, [do, dS])
    want = torch.autograd.grad([ro, rS], ref, [do.double(), dS.double()])
    for name, x, y in zip(NAMES["delta"], got, want):
        check(x, y, "d" + name)


def test_scan_strong_decays_of_few_tokens():
    x, dt, A, B, C, D, s = scan_inputs(36, 1, 4, 32, 32, len(SHORT) - 1, seed=3, state=True)
    dt[0], dt[3], dt[10], dt[21:25] = 1e3, 60.0, 1e3, 0.0
    A[0], A[1] = 0.0, -1e4
    run_scan((x, dt, A, B, C, D, s), SHORT)


@pytest.mark.parametrize("hk,hv", [(1, 5), (1, 16), (2, 16)])
@pytest.mark.parametrize("cuts", [[0, 40, 130], SHORT], ids=["chunks", "few tokens"])
def test_heads_shared_by_many(hk, hv, cuts):
    T, docs = cuts[-1] + 2, len(cuts) - 1
    run_delta(delta_inputs(T, hk, hv, 64, 72, docs, seed=7, state=True), cuts, scale=0.125)
    run_scan(scan_inputs(T, hk, hv, 72, 64, docs, seed=7, state=True), cuts)


@pytest.mark.parametrize("op", OPS)
def test_one_shared_head_is_read_in_place(op):
    """One of the heads of a wider tensor, for all heads of v (x): as it lies, with the bits of a copy."""
    from xorl_b200.ops import recurrence as R
    cu, ts = boundaries([0, 70, 71, 300]), inputs(op)
    one = (0, 1) if op == "delta" else (3, 4)
    views, copies = list(ts), list(ts)
    for i in one:
        views[i] = ts[i][:, 1:]
        assert R._rows(views[i]) is views[i]
        copies[i] = views[i].clone(memory_format=torch.contiguous_format)
    same(both_ways(op, copies, cu), both_ways(op, views, cu))
