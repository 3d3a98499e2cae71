"""Calls of the gated linear recurrences that have to give the same bits: repeated beside other work on the GPU, with and
without gradients, and whatever a call keeps for its backward pass."""
import pytest
import torch

from test_recurrence_gpu import _need_cuda, delta_inputs, run_delta, run_scan, scan_inputs  # noqa: F401
from test_recurrence_use_gpu import OPS, both_ways, boundaries, call, inputs, layer, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op,hk,hv,dk,dv", [("delta", 2, 2, 128, 32), ("delta", 1, 3, 128, 64), ("delta", 1, 8, 64, 128),
                                            ("scan", 2, 2, 128, 64), ("scan", 1, 3, 128, 64), ("scan", 1, 16, 64, 96)])
def test_gradients_repeat_beside_other_work(op, hk, hv, dk, dv):
    """Few slices and few heads, so that the gradient kernel's last head is soon behind its first, and products on another
    stream that take issue slots and memory from its warps in ever different places."""
    cuts = [0, 70, 71, 135, 700]
    ts = list((delta_inputs if op == "delta" else scan_inputs)(700, hk, hv, dk, dv, len(cuts) - 1, seed=11, state=True))
    cu = boundaries(cuts)
    want = both_ways(op, ts, cu)
    side, m = torch.cuda.Stream(), torch.randn(1024, 1024, device="cuda").bfloat16()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(40):
        with torch.cuda.stream(side):
            for _ in range(i % 4):
                m @ m
        same(want, both_ways(op, ts, cu))
    torch.cuda.current_stream().wait_stream(side)


def test_long_walks_without_gradients_beside_other_work():
    """Several hundred chunks in a row through the two-stage walk that keeps nothing, with products on another stream that
    hold up its warps: the bits of the first call, and no wait that ran out (the fixture reads the status words)."""
    from xorl_b200.ops.recurrence import gated_delta_rule
    q, k, v, g, beta, s = delta_inputs(20000, 1, 2, 64, 64, 1, seed=13, state=True)
    cu = boundaries([0, 20000])
    side, m = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda").bfloat16()
    with torch.no_grad():
        run = lambda: gated_delta_rule(q, k, v, g, beta, cu, scale=0.125, qk_l2norm=True, initial_state=s,  # noqa: E731
                                       return_final_state=True)
        want = run()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(10):
            with torch.cuda.stream(side):
                for _ in range(8):
                    m @ m
            same(want, run())
    torch.cuda.current_stream().wait_stream(side)


def call_both(op, ts, cu):
    """The call with gradients and without: outputs and states."""
    with torch.no_grad():
        plain = call(op, ts, cu)
    return plain, [t.detach() for t in call(op, [None if t is None else t.detach().requires_grad_() for t in ts], cu)]


CUTS = {"one": [0, 300], "two chunks": [0, 128], "long and short": [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 300], "outside": [40, 40, 101, 250],
        "many": list(range(0, 2001, 50)), "tokens": list(range(0, 120)), "short and long": [5, 6, 7, 8, 9, 9, 10, 30, 31, 47, 48, 112],
        "padded": [0, 100, 290] + [300] * 30, "short and outside": [20, 21, 22, 37, 54, 55, 55, 56, 57]}


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("cuts", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 4, 64, 64), (1, 4, 128, 128), (4, 8, 32, 40)])
@pytest.mark.parametrize("state", [False, True])
def test_calls_with_and_without_gradients(op, cuts, hk, hv, dk, dv, state):
    """A pass without gradients that is repeated with them (recomputed activations), or whose scores are compared with those of
    training, has the same bits."""
    T = max(cuts[-1] + 3, 128)
    ts = list((delta_inputs if op == "delta" else scan_inputs)(T, hk, hv, dk, dv, len(cuts) - 1, seed=17, state=state))
    same(*call_both(op, ts, boundaries(cuts)))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("cuts", [[0, 1, 2, 3, 40, 41, 41, 57, 70], [18, 19, 20, 36, 53, 60, 61, 62], list(range(0, 65))],
                         ids=["mixed", "outside", "ones"])
@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 4, 64, 64), (1, 3, 128, 72), (4, 4, 24, 8)])
def test_gradients_behind_documents_of_few_tokens(op, cuts, hk, hv, dk, dv, monkeypatch):
    """The forward pass goes token by token, the backward pass works on chunks, from kept tiles or from ones that it makes itself,
    twice in a row with the same bits."""
    T, docs = cuts[-1] + 5, len(cuts) - 1
    if op == "delta":
        run_delta(delta_inputs(T, hk, hv, dk, dv, docs, seed=19, state=True), cuts, scale=dk ** -0.5)
        ts = list(delta_inputs(T, hk, hv, dk, dv, docs, seed=19, state=True))
    else:
        run_scan(scan_inputs(T, hk, hv, dk, dv, docs, seed=19, state=True), cuts)
        ts = list(scan_inputs(T, hk, hv, dk, dv, docs, seed=19, state=True))
    leaves = [t.detach().requires_grad_() for t in ts]
    o, S = call(op, leaves, boundaries(cuts))
    d = [torch.randn_like(o), torch.randn_like(S)]
    want = torch.autograd.grad([o, S], leaves, d, retain_graph=True)
    same(want, torch.autograd.grad([o, S], leaves, d))
    from xorl_b200.ops import recurrence as R
    monkeypatch.setattr(R, "KEEP_BYTES", 0)
    again = call(op, leaves, boundaries(cuts))
    same([o, S], again)
    same(want, torch.autograd.grad(again, leaves, d))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("cuts", [[0, 70, 71, 300], list(range(0, 301, 10))], ids=["chunks", "few tokens"])
@pytest.mark.parametrize("keep", [True, False])
def test_boundaries_are_the_callers_again_behind_the_forward_pass(op, cuts, keep, monkeypatch):
    """A buffer of boundaries that takes the next batch's before the backward pass of this one, whatever the call keeps."""
    from xorl_b200.ops import recurrence as R
    if not keep:
        monkeypatch.setattr(R, "KEEP_BYTES", 0)
        R._layout.cache_clear()
    try:
        ts, cu = inputs(op, docs=len(cuts) - 1), boundaries(cuts)
        want = both_ways(op, ts, cu)
        leaves = [t.detach().requires_grad_() for t in ts]
        o, S = call(op, leaves, cu)
        cu.copy_(torch.arange(len(cuts)))
        gen = torch.Generator(device="cuda").manual_seed(9)
        do, dS = torch.randn(o.shape, generator=gen, device="cuda").bfloat16(), torch.randn(S.shape, generator=gen, device="cuda")
        same(want, [o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [do, dS])])
    finally:
        R._layout.cache_clear()


@pytest.mark.parametrize("op", OPS)
def test_what_a_call_keeps_is_bounded(op, monkeypatch):
    """Nothing, the operands, or the tiles too: within the bound, which a program may set at any time, with the same bits."""
    from xorl_b200.ops import recurrence as R
    ts, cu = inputs(op, T=2000, docs=2), boundaries([0, 700, 2000])
    want = both_ways(op, ts, cu)
    hk, hv, d = 2, 4, 64
    full = R._layout(2000, 2, hk, hv, d, d, op == "delta", True, 0, 1 << 40)
    part = R._layout(2000, 2, hk, hv, d, d, op == "delta", True, 0, full[1] - 1)
    assert (full[3], part[3]) == (2, 1) and part[1] < full[1]
    out = ts[2 if op == "delta" else 0].numel() * 2 + ts[-1].numel() * 4          # outputs and states
    # what was asked for: of a cached block that is up to 1 MB larger the allocator hands out all
    held = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731
    for limit, bound in ((full[1], full[1]), (full[1] - 1, part[1]), (part[1], part[1]), (part[1] - 1, 0), (0, 0)):
        monkeypatch.setattr(R, "KEEP_BYTES", limit)
        leaves = [t.detach().requires_grad_() for t in ts]
        torch.cuda.synchronize()
        before = held()
        o, S = call(op, leaves, cu)
        assert held() - before <= out + bound + 8192
        gen = torch.Generator(device="cuda").manual_seed(9)
        do, dS = torch.randn(o.shape, generator=gen, device="cuda").bfloat16(), torch.randn(S.shape, generator=gen, device="cuda")
        same(want, [o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [do, dS])])
        del o, S, do, dS, leaves


@pytest.mark.parametrize("docs,length", [(1, 100), (2, 256), (3, 520), (40, 64), (10, 300), (3, 700)])
@pytest.mark.parametrize("heads", [2, 20])
def test_stages_of_the_walk(docs, length, heads):
    """Few and many CTAs, short and long documents, on both sides of the walk's choice: without gradients the bits of the call
    with them, which always has two stages."""
    T = docs * length
    ts = list(delta_inputs(T, heads // 2, heads, 128, 128, docs, seed=23, state=True))
    same(*call_both("delta", ts, boundaries(list(range(0, T + 1, length)))))


@pytest.mark.parametrize("kind", OPS)
@pytest.mark.parametrize("cuts", [[0, 33, 34, 200], list(range(0, 201, 8))], ids=["chunks", "few tokens"])
def test_layers_recomputed(kind, cuts):
    """A layer's first pass without gradients and the one that is run again for them."""
    from xorl_b200.models.context import StepContext
    m = layer(kind)
    ctx = StepContext(cu_seqlens=boundaries(cuts), position_ids=torch.cat([torch.arange(b - a) for a, b in zip(cuts, cuts[1:])]).cuda(),
                      max_seqlen=max(b - a for a, b in zip(cuts, cuts[1:])))
    x = torch.randn(200, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    with torch.no_grad():
        first = m(x, ctx)
    assert torch.equal(first, m(x.requires_grad_(), ctx).detach())
