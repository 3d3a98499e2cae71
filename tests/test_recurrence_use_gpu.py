"""The gated linear recurrences as programs use them: strided inputs, streams, graphs, neighbouring documents, strong
decays, states carried from call to call, many and long documents, and the layers that call them.  Tolerances as in
test_recurrence_gpu.py; where two calls do the same arithmetic their bits are equal."""
import pytest
import torch

from test_recurrence_gpu import (HELD, _need_cuda, check, delta_inputs, oracle_delta, oracle_scan, run_delta,  # noqa: F401
                                 run_scan, scan_inputs)

pytestmark = pytest.mark.gpu

NAMES = {"delta": ("q", "k", "v", "g", "beta", "initial_state"), "scan": ("x", "dt", "A", "B", "C", "D", "initial_state")}
OPS = ["delta", "scan"]


def boundaries(cuts):
    return torch.tensor(cuts, dtype=torch.int32, device="cuda")


def inputs(op, T=300, docs=3, state=True, seed=0, **kw):
    if op == "delta":
        return list(delta_inputs(T, 2, 4, 64, 64, docs, seed=seed, state=state, **kw))
    return list(scan_inputs(T, 2, 4, 64, 64, docs, seed=seed, state=state, **kw))


def call(op, ts, cu, **kw):
    from xorl_b200.ops.recurrence import gated_delta_rule, ssd_scan
    if op == "delta":
        return gated_delta_rule(*ts[:5], cu, scale=0.125, qk_l2norm=True, initial_state=ts[5], return_final_state=True, **kw)
    return ssd_scan(*ts[:6], cu, initial_state=ts[6], return_final_state=True, **kw)


def both_ways(op, ts, cu, seed=9):
    """(output, states, gradients ...) of one forward and backward pass."""
    leaves = [None if t is None else t.detach().requires_grad_() for t in ts]
    o, S = call(op, leaves, cu)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    do, dS = torch.randn(o.shape, generator=gen, device="cuda").bfloat16(), torch.randn(S.shape, generator=gen, device="cuda")
    grads = torch.autograd.grad([o, S], [t for t in leaves if t is not None], [do, dS])
    return [o.detach(), S.detach(), *grads]


def same(a, b):
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("op", OPS)
def test_same_bits_twice_and_on_another_stream(op):
    ts, cu = inputs(op), boundaries([0, 70, 71, 300])
    first = both_ways(op, ts, cu)
    same(first, both_ways(op, ts, cu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both_ways(op, ts, cu)
    torch.cuda.current_stream().wait_stream(side)
    same(first, again)


@pytest.mark.parametrize("op", OPS)
def test_two_calls_at_once_and_two_backward_passes(op):
    """Two graphs alive at the same time, each walked through twice."""
    cu = boundaries([0, 70, 71, 300])
    a, b = inputs(op, seed=1), inputs(op, seed=2)
    la, lb = ([t.detach().requires_grad_() for t in ts] for ts in (a, b))
    (oa, _), (ob, _) = call(op, la, cu), call(op, lb, cu)
    do = torch.randn(oa.shape, device="cuda").bfloat16()
    gb = torch.autograd.grad(ob, lb, do, retain_graph=True)
    ga = torch.autograd.grad(oa, la, do, retain_graph=True)
    same(gb, torch.autograd.grad(ob, lb, do))
    same(ga, torch.autograd.grad(oa, la, do))


def test_both_operators_on_two_streams():
    """Passes of both, of different lengths, side by side on two streams: the bits of one after the other."""
    cases = [(op, inputs(op, T=T, docs=3, seed=T), boundaries([0, 70, 71, T])) for T in (300, 1500) for op in OPS]
    want = [both_ways(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append(both_ways(*cases[(i * 3 + i // 2) % len(cases)]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        same(g, want[(i * 3 + i // 2) % len(cases)])


@pytest.mark.parametrize("op", OPS)
def test_captured_and_replayed(op):
    """Two captured passes over the same buffers, replayed in turn with new values in them (boundaries too)."""
    ts, cu = inputs(op), boundaries([0, 70, 71, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both_ways(op, ts, cu)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        leaves = [t.detach().requires_grad_() for t in ts]
        do, dS = torch.zeros_like(ts[2 if op == "delta" else 0]), torch.zeros_like(ts[-1])
        with torch.cuda.graph(graph):
            o, S = call(op, leaves, cu)
            grads = torch.autograd.grad([o, S], leaves, [do, dS])
        graphs.append((graph, do, dS, [o, S, *grads]))
    for step in range(3):
        new = inputs(op, seed=10 + step)
        cu.copy_(boundaries([[0, 64, 128, 300], [0, 0, 299, 300], [5, 6, 200, 200]][step]))
        for t, n in zip(ts, new):
            t.copy_(n)
        want = both_ways(op, new, cu.clone(), seed=step)
        gen = torch.Generator(device="cuda").manual_seed(step)
        d0 = torch.randn(graphs[0][1].shape, generator=gen, device="cuda").bfloat16()
        d1 = torch.randn(graphs[0][2].shape, generator=gen, device="cuda")
        for graph, do, dS, outs in graphs:
            do.copy_(d0), dS.copy_(d1)
            graph.replay()
        for _, _, _, outs in graphs:
            same([t.detach() for t in outs], want)


@pytest.mark.parametrize("op", OPS)
def test_captured_without_gradients(op):
    """A captured call of short documents, replayed with boundaries that make long ones too."""
    ts = inputs(op, T=128, docs=8)
    cu = boundaries(list(range(0, 129, 16)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            call(op, ts, cu)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(op, ts, cu)
        for cuts in ([0, 1, 2, 3, 100, 101, 102, 103, 128], [0, 0, 128, 128, 128, 128, 128, 128, 128], [5, 6, 7, 8, 9, 10, 11, 12, 90]):
            cu.copy_(boundaries(cuts))
            graph.replay()
            got = [t.clone() for t in out]
            same(got, call(op, ts, boundaries(cuts)))
            us = [t.double() for t in ts]
            ref = oracle_delta(*us[:5], cuts, 0.125, True, us[5]) if op == "delta" else oracle_scan(*us[:6], cuts, us[6])
            check(got[0], ref[0], "o")
            check(got[1], ref[1], "S")


@pytest.mark.parametrize("op", OPS)
def test_entry_points_refuse(op):
    """What the Python side never hands over is refused before anything is launched: pointers and strides off 16 bytes, sizes
    beyond the kernels', too few chunks."""
    from xorl_b200.ops import _lib, recurrence as R
    ts, cu = inputs(op, T=64, docs=1, state=False), boundaries([0, 64])
    q, k, v = ts[:3] if op == "delta" else (ts[4], ts[3], ts[0])
    g, b = (ts[3], ts[4]) if op == "delta" else (None, ts[1])
    A, D = (None, None) if op == "delta" else (ts[2], ts[5])
    lay = R._layout(64, 1, 2, 4, 64, 64, op == "delta", False, 0)
    ws, o = torch.empty(lay[1], dtype=torch.uint8, device="cuda"), torch.empty_like(v)

    def run(q=q, k=k, v=v, lay=lay, step=0, s_in=None):
        words = R._words(q, k, v, g, b, A, D, cu, s_in, None, None, None, None, (o.data_ptr(), 0, 0, 0, 0, 0, 0, 0), ws, None, lay,
                         op == "delta", 0, step)
        _lib.call_on(v.device, "xb_recurrence_fwd", words, 1.0, op == "delta")

    run()
    wide = torch.zeros(64, 2, 80, dtype=torch.bfloat16, device="cuda")
    odd = torch.zeros(64 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")[1:1 + 64 * 4 * 64].view(64, 4, 64)
    flat = torch.zeros(64 * 4 * 64 + 4, device="cuda")
    for bad in (dict(q=wide[:, :, 1:65]), dict(k=torch.zeros(64, 2, 65, device="cuda").bfloat16()[:, :, :64]), dict(v=odd),
                dict(q=wide[:, :, :60]), dict(lay=(lay[0] - 3, *lay[1:])), dict(step=64), dict(step=-1),
                dict(s_in=flat[1:1 + 4 * 64 * 64].view(1, 4, 64, 64))):
        with pytest.raises(RuntimeError, match="xb_recurrence_fwd failed with code -1"):
            run(**bad)


@pytest.mark.parametrize("op", OPS)
def test_strides_and_alignment(op):
    """Slices of a fused projection, rows off 16 bytes, shared (expanded) heads, other orders, states off 16 bytes."""
    cu = boundaries([0, 70, 71, 300])
    ts = inputs(op)
    want = both_ways(op, ts, cu)

    def fused(t, pad):                       # the middle of wider rows
        wide = torch.randn(t.shape[0], t.shape[1] * t.shape[2] + 2 * pad, device="cuda").bfloat16()
        view = wide[:, pad:pad + t.shape[1] * t.shape[2]].view(t.shape) if pad % 8 == 0 else \
            wide.as_strided(t.shape, (wide.stride(0), t.shape[2], 1), pad)
        view.copy_(t)
        return view

    def shifted(t):                          # contiguous, four bytes off
        flat = torch.empty(t.numel() + 4, device="cuda")[1:1 + t.numel()].view(t.shape)
        return flat.copy_(t)

    turn = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for change in (lambda t: fused(t, 16), lambda t: fused(t, 3), turn, lambda t: t.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        same(want, both_ways(op, [change(t) if t.dtype == torch.bfloat16 else t for t in ts], cu))
    per_head = [turn(t) if t.dim() == 2 else shifted(t) if t.dim() == 4 else t for t in ts]
    same(want, both_ways(op, per_head, cu))
    one = 0 if op == "delta" else 3          # one head for all, without a copy
    wide = list(ts)
    wide[one] = ts[one][:, :1].expand(-1, 2, -1)
    full = list(ts)
    full[one] = wide[one].contiguous()
    same(both_ways(op, full, cu), both_ways(op, wide, cu))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_documents_keep_their_neighbours_values_out(op, value):
    """A document of Inf or NaN, its gradient included: the others' bits stay."""
    cu = boundaries([0, 70, 101, 300])
    ts = inputs(op)
    rows = [i for i, n in enumerate(NAMES[op]) if n not in ("A", "D", "initial_state")]
    bad = [t.clone() for t in ts]
    for i in rows:
        bad[i][70:101] = value
    bad[-1][1] = value

    def run(us):
        leaves = [t.detach().requires_grad_() for t in us]
        o, S = call(op, leaves, cu)
        gen = torch.Generator(device="cuda").manual_seed(4)
        do, dS = torch.randn(o.shape, generator=gen, device="cuda").bfloat16(), torch.randn(S.shape, generator=gen, device="cuda")
        if us is bad:
            do[70:101], dS[1] = value, value
        grads = torch.autograd.grad([o, S], leaves, [do, dS])
        return o, S, grads

    (o, S, g), (o2, S2, g2) = run(ts), run(bad)
    keep, docs = [*range(70), *range(101, 300)], [0, 2]
    assert torch.equal(o[keep], o2[keep]) and torch.equal(S[docs], S2[docs])
    for i in rows:
        assert torch.equal(g[i][keep], g2[i][keep]), NAMES[op][i]
    assert torch.equal(g[-1][docs], g2[-1][docs])


def test_delta_strong_decays_and_zero_rows():
    """Decays that leave nothing (down to -inf) beside none at all, betas of 0 and 1, rows of zeros under the norm."""
    ts = delta_inputs(150, 1, 2, 32, 32, 2, seed=3, state=True)
    g = ts[3]
    g[10], g[11], g[40], g[70:80], g[100] = -1e4, 0.0, -float("inf"), 0.0, -130.0
    ts[4][20], ts[4][21] = 0.0, 1.0
    ts[0][5], ts[1][6], ts[1][100] = 0, 0, 0
    from xorl_b200.ops.recurrence import gated_delta_rule
    live = [t.detach().requires_grad_() for t in ts]
    ref = [t.detach().double().requires_grad_() for t in ts]
    o, S = gated_delta_rule(*live[:5], boundaries([0, 100, 150]), scale=0.2, qk_l2norm=True, initial_state=live[5],
                            return_final_state=True)
    ro, rS = oracle_delta(*ref[:5], [0, 100, 150], 0.2, True, ref[5])
    check(o.detach(), ro, "o")
    check(S.detach(), rS, "S")
    do, dS = torch.randn_like(ro).bfloat16(), torch.randn_like(rS).float()
    got = torch.autograd.grad([o, S], live, [do, dS])
    want = torch.autograd.grad([ro, rS], ref, [do.double(), dS.double()])
    for name, x, y in zip(NAMES["delta"], got, want):
        if name in ("q", "k"):               # at a row of zeros the norm has no derivative: 1e12 there, by its lower limit
            rows = [t for t in range(150) if t not in (5, 6, 100)]
            assert torch.isfinite(x).all()
            x, y = x[rows], y[rows]
        check(x, y, "d" + name)


def test_scan_strong_decays():
    """Steps of zero, and steps that forget everything before them."""
    x, dt, A, B, C, D, s = scan_inputs(150, 1, 4, 32, 32, 2, seed=3, state=True)
    dt[10], dt[11:20], dt[70] = 1e3, 0.0, 60.0
    A[0], A[1] = 0.0, -1e4
    run_scan((x, dt, A, B, C, D, s), [0, 100, 150])


@pytest.mark.parametrize("op", OPS)
def test_states_made_again(op, monkeypatch):
    """A call whose tiles are not kept gives the same gradients."""
    from xorl_b200.ops import recurrence as R
    ts, cu = inputs(op), boundaries([0, 70, 71, 300])
    want = both_ways(op, ts, cu)
    monkeypatch.setattr(R, "KEEP_BYTES", 0)
    R._layout.cache_clear()
    try:
        same(want, both_ways(op, ts, cu))
    finally:
        R._layout.cache_clear()


@pytest.mark.parametrize("op", OPS)
def test_calls_without_gradients(op):
    """Many short documents beside a long one, and an ordinary batch, in every kind of boundaries.  The scan's bits are those of
    the call that keeps its tiles; the delta rule's call with gradients carries more bits inside."""
    for cuts in ([0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 300], [0, 300]):
        ts, cu = inputs(op, docs=len(cuts) - 1), boundaries(cuts)
        want = both_ways(op, ts, cu)
        with torch.no_grad():
            got = call(op, ts, cu)
            if op == "scan":
                same(want[:2], got)
            check(got[1], want[1].double(), "S")
            o, most = want[0].double(), want[0].abs().max().item()          # two roundings to bf16 apart
            assert ((got[0].double() - o).abs() <= 2 * 2.0 ** -8 * o.abs() + HELD * most).all()
            same(got, call(op, ts, cu.long()))
            same(got, call(op, ts, cu.cpu()))


@pytest.mark.parametrize("op", OPS)
def test_only_some_outputs_and_inputs_count(op):
    ts, cu = inputs(op), boundaries([0, 70, 71, 300])
    fn = oracle_delta if op == "delta" else oracle_scan
    cuts = [0, 70, 71, 300]
    for which in (0, 1):
        a = [t.detach().requires_grad_() for t in ts]
        b = [t.detach().double().requires_grad_() for t in ts]
        out = call(op, a, cu)[which]
        ref = (fn(*b[:5], cuts, 0.125, True, b[5]) if op == "delta" else fn(*b[:6], cuts, b[6]))[which]
        d = torch.randn_like(ref).to(out.dtype)
        got = torch.autograd.grad(out, a, d)
        want = torch.autograd.grad(ref, b, d.double(), allow_unused=True)
        for n, x, y, z in zip(NAMES[op], got, want, b):
            check(x, torch.zeros_like(z) if y is None else y, "d" + n)
    a = [t.detach().requires_grad_(i == 2) for i, t in enumerate(ts)]
    o, S = call(op, a, cu)
    o.float().sum().backward()               # an expanded gradient
    assert a[2].grad is not None and torch.isfinite(a[2].grad).all() and all(t.grad is None for i, t in enumerate(a) if i != 2)


def test_one_tensor_as_q_and_k():
    q, _, v, g, beta, _ = delta_inputs(100, 2, 2, 32, 32, 1, seed=6)
    from xorl_b200.ops.recurrence import gated_delta_rule
    a, b = [t.detach().requires_grad_() for t in (q, v, g, beta)], [t.detach().double().requires_grad_() for t in (q, v, g, beta)]
    o = gated_delta_rule(a[0], a[0], *a[1:], boundaries([0, 100]), scale=0.2, qk_l2norm=True)
    ro, _ = oracle_delta(b[0], b[0], *b[1:], [0, 100], 0.2, True, None)
    do = torch.randn_like(ro).bfloat16()
    got, want = torch.autograd.grad(o, a, do), torch.autograd.grad(ro, b, do.double())
    # autograd adds two rounded gradients and rounds again: three roundings of at most 2^-8 of the larger part
    most = want[0].abs().max()
    assert ((got[0].double() - want[0]).abs() <= 3 * 2.0 ** -8 * 2 * most + HELD * most).all()
    for x, y, n in zip(got[1:], want[1:], "vgb"):
        check(x, y, n)


@pytest.mark.parametrize("op", OPS)
def test_no_rows(op):
    """A call without rows hands the states through, their gradients too."""
    ts = [t[:0] if t is not None and t.dim() > 1 and i < 5 else t for i, t in enumerate(inputs(op, docs=2))]
    cu = boundaries([0, 0, 0])
    leaves = [t.detach().requires_grad_() for t in ts]
    o, S = call(op, leaves, cu)
    assert o.shape[0] == 0 and torch.equal(S, ts[-1])
    dS = torch.randn_like(S)
    grads = torch.autograd.grad([o, S], leaves, [o.detach(), dS])
    assert torch.equal(grads[-1], dS)
    if op == "scan":
        assert not grads[2].any() and not grads[5].any()


@pytest.mark.parametrize("op", OPS)
def test_serving(op):
    """Prompts of several lengths in one call, then single tokens with the states carried, against one call over all."""
    lens, more = [1, 64, 131], 4
    total = sum(lens) + more * len(lens)
    ts = inputs(op, T=total, docs=len(lens), state=False, seed=8)
    rows = [i for i, n in enumerate(NAMES[op]) if n not in ("A", "D", "initial_state")]
    cuts = [0]
    for n in lens:
        cuts.append(cuts[-1] + n + more)
    with torch.no_grad():
        whole, last = call(op, ts, boundaries(cuts))

        def part(at, state):                 # `at`: the rows of each document
            idx = torch.cat([torch.arange(cuts[d] + s, cuts[d] + e) for d, (s, e) in enumerate(at)]).cuda()
            us = [t[idx] if i in rows else t for i, t in enumerate(ts)]
            us[-1] = state
            c = [0]
            for s, e in at:
                c.append(c[-1] + e - s)
            o, S = call(op, us, boundaries(c))
            got[idx] = o
            return S

        got = torch.empty_like(whole)
        state = part([(0, n) for n in lens], None)
        for i in range(more):
            state = part([(n + i, n + i + 1) for n in lens], state)
    check(state, last.double(), "state")
    most = whole.double().abs().max()        # two roundings to bf16 apart
    assert ((got.double() - whole.double()).abs() <= 2 * 2.0 ** -8 * whole.double().abs() + HELD * most).all()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("hk,hv,dk,dv", [(1, 1, 8, 8), (2, 4, 64, 64), (1, 3, 128, 128), (2, 4, 72, 40), (1, 2, 32, 136)])
@pytest.mark.parametrize("lens", [[1] * 7, [0, 1, 5, 0, 16, 3], [1, 16, 17, 0, 64, 2, 65, 1, 1, 200, 16] + [1] * 20, [1, 0]],
                         ids=["ones", "short", "mixed", "two"])
@pytest.mark.parametrize("outside", [(0, 0), (3, 20), (18, 2)])
def test_few_tokens_per_document(op, hk, hv, dk, dv, lens, outside):
    """Documents around the length up to which they go token by token, rows outside them on both sides of it too."""
    from xorl_b200.ops.recurrence import gated_delta_rule, ssd_scan
    cuts = [outside[0]]
    for n in lens:
        cuts.append(cuts[-1] + n)
    T = cuts[-1] + outside[1]
    for state in (False, True):
        if op == "delta":
            ts = delta_inputs(T, hk, hv, dk, dv, len(lens), seed=4, state=state)
            o, S = gated_delta_rule(*ts[:5], boundaries(cuts), scale=0.3, qk_l2norm=state, initial_state=ts[5], return_final_state=True)
            bits = lambda t: t.view(torch.int16)  # noqa: E731  (long keys: what grows without bound ends as NaN in both)
            assert torch.equal(bits(o), bits(gated_delta_rule(*ts[:5], boundaries(cuts), scale=0.3, qk_l2norm=state, initial_state=ts[5])))
            ds = [None if t is None else t.double() for t in ts]
            if not state:                        # short keys
                ts[1].div_(dk), ts[0].div_(dk)
                o, S = gated_delta_rule(*ts[:5], boundaries(cuts), scale=0.3, return_final_state=True)
                ds = [None if t is None else t.double() for t in ts]
            ro, rS = oracle_delta(*ds[:5], cuts, 0.3, state, ds[5])
        else:
            ts = scan_inputs(T, hk, hv, dk, dv, len(lens), seed=4, state=state)
            o, S = ssd_scan(*ts[:6], boundaries(cuts), initial_state=ts[6], return_final_state=True)
            assert torch.equal(o, ssd_scan(*ts[:6], boundaries(cuts), initial_state=ts[6]))
            ds = [None if t is None else t.double() for t in ts]
            ro, rS = oracle_scan(*ds[:6], cuts, ds[6])
        check(o, ro, "o")
        check(S, rS, "S")


@pytest.mark.parametrize("op", OPS)
def test_long_document_in_two_halves(op):
    ts = inputs(op, T=6000, docs=1, state=False, seed=12)
    rows = [i for i, n in enumerate(NAMES[op]) if n not in ("A", "D", "initial_state")]
    with torch.no_grad():
        whole, last = call(op, ts, boundaries([0, 6000]))
        first = [t[:3001] if i in rows else t for i, t in enumerate(ts)]
        o1, S = call(op, first, boundaries([0, 3001]))
        second = [t[3001:] if i in rows else t for i, t in enumerate(ts)]
        second[-1] = S
        o2, S = call(op, second, boundaries([0, 2999]))
    check(S, last.double(), "state")
    most = whole.double().abs().max()
    assert ((torch.cat([o1, o2]).double() - whole.double()).abs() <= 2 * 2.0 ** -8 * whole.double().abs() + HELD * most).all()


def test_delta_many_documents_of_one_token():
    """4200 documents of one token and 32 heads: the operand tiles (4.3 GB) and the kept states (8.7 GB) pass 32 bits of
    bytes.  With S = 0 the output is beta (scale k.q) v."""
    from xorl_b200.ops.recurrence import gated_delta_rule
    T = 4200
    q, k, v, g, beta, _ = delta_inputs(T, 16, 32, 128, 128, 1, seed=2)
    a, b = [t.detach().requires_grad_() for t in (q, k, v, g, beta)], [t.detach().double().requires_grad_() for t in (q, k, v, g, beta)]
    o = gated_delta_rule(*a, torch.arange(T + 1, device="cuda"), scale=0.1)
    dot = 0.1 * (b[0] * b[1]).sum(-1).repeat_interleave(2, 1)
    ro = (b[4] * dot).unsqueeze(-1) * b[2]
    do = torch.randn_like(ro).bfloat16()
    check(o.detach(), ro, "o")
    got = torch.autograd.grad(o, a, do)
    want = torch.autograd.grad(ro, [b[i] for i in (0, 1, 2, 4)], do.double())
    assert not got[3].any()                  # nothing enters that could decay
    for name, x, y in zip(("q", "k", "v", "beta"), [got[0], got[1], got[2], got[4]], want):
        check(x, y, "d" + name)


@pytest.mark.parametrize("op", OPS)
def test_rows_behind_32_bits_of_elements(op):
    """Rows so far apart that the last start behind 2^31 elements."""
    T, far = 70, (1 << 31) // 69 // 8 * 8 + 8
    ts = inputs(op, T=T, docs=1, seed=3)
    cu = boundaries([0, T])
    with torch.no_grad():
        want = call(op, ts, cu)
    i = 2 if op == "delta" else 0
    store = torch.empty(far * (T - 1) + ts[i][0].numel(), dtype=torch.bfloat16, device="cuda")
    ts[i] = store.as_strided(ts[i].shape, (far, ts[i].shape[2], 1)).copy_(ts[i])
    with torch.no_grad():
        same(want, call(op, ts, cu))


@pytest.mark.parametrize("op", OPS)
def test_gradients_against_differences(op):
    """Along a random direction, the gradient's product with it is the definition's (64 bits) difference quotient."""
    ts, cuts = inputs(op, T=100, docs=2, seed=5), [0, 30, 100]
    fn = (lambda us: oracle_delta(*us[:5], cuts, 0.125, True, us[5])) if op == "delta" else (lambda us: oracle_scan(*us[:6], cuts, us[6]))
    got = both_ways(op, ts, boundaries(cuts), seed=9)[2:]
    gen = torch.Generator(device="cuda").manual_seed(9)
    base = [t.double() for t in ts]
    o, S = fn(base)
    do, dS = torch.randn(o.shape, generator=gen, device="cuda").bfloat16().double(), torch.randn(S.shape, generator=gen, device="cuda").double()
    loss = lambda us: sum((x * y).sum() for x, y in zip(fn(us), (do, dS)))  # noqa: E731
    h = 1e-5
    for i, name in enumerate(NAMES[op]):
        way = torch.randn(ts[i].shape, generator=gen, device="cuda").double()
        up, down = ([t + s * h * way if j == i else t for j, t in enumerate(base)] for s in (1, -1))
        quotient = (loss(up) - loss(down)) / (2 * h)
        terms = got[i].double() * way
        # half a step of the gradient's type on every term, what the kernels hold, and the quotient's own error (h^2 of the
        # third derivative and 2^-53 / h of the loss's terms: below 1e-6 of the terms' size)
        size = terms.abs().sum()
        step = 2.0 ** -8 if got[i].dtype == torch.bfloat16 else 2.0 ** -24
        room = (step + 1e-6) * size + HELD * got[i].double().abs().max() * way.abs().sum()
        assert (terms.sum() - quotient).abs() <= room, name


def test_other_types_and_sizes_run_as_tensor_ops():
    from xorl_b200.ops import recurrence as R
    for dk, dv, dtype in ((20, 16, torch.bfloat16), (16, 12, torch.bfloat16), (136, 16, torch.bfloat16), (16, 16, torch.float32),
                          (16, 16, torch.float16)):
        q, k, v, g, beta, _ = delta_inputs(50, 1, 2, dk, dv, 1)
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        n = R.launch_count()
        o = R.gated_delta_rule(q, k, v, g, beta, boundaries([0, 20, 50]), qk_l2norm=True)
        ro, _ = oracle_delta(*(t.double() for t in (q, k, v, g, beta)), [0, 20, 50], 1.0, True, None)
        assert R.launch_count() == n and o.shape == v.shape
        assert (o.double() - ro).abs().max() <= 2.0 ** -8 * 2 * ro.abs().max()
        x, dt, A, B, C, D, _ = scan_inputs(50, 1, 2, dk, dv, 1)
        x, B, C = x.to(dtype), B.to(dtype), C.to(dtype)
        y = R.ssd_scan(x, dt, A, B, C, D, boundaries([0, 20, 50]))
        ry, _ = oracle_scan(*(t.double() for t in (x, dt, A, B, C, D)), [0, 20, 50], None)
        assert R.launch_count() == n and (y.double() - ry).abs().max() <= 2.0 ** -8 * 2 * ry.abs().max()


# ---- the layers ------------------------------------------------------------------------------------------------------
def layer(kind):
    from xorl_b200.models.config import ModelConfig
    extra = dict(linear_num_key_heads=2, linear_num_value_heads=4, linear_key_head_dim=64, linear_value_head_dim=64,
                 linear_conv_kernel_dim=4) if kind == "delta" else \
        dict(mamba_num_heads=8, mamba_head_dim=64, n_groups=2, ssm_state_size=64, conv_kernel=4)
    cfg = ModelConfig(hidden_size=256, extra=extra)
    torch.manual_seed(0)
    if kind == "delta":
        from xorl_b200.models.gated_deltanet import GatedDeltaNet as Layer
    else:
        from xorl_b200.models.mamba2 import Mamba2Mixer as Layer
    m = Layer(cfg, 0, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith("norm_weight") or n == "D":
                p.copy_(1 + 0.1 * torch.randn_like(p))
            elif n in ("A_log", "dt_bias"):
                p.copy_(torch.randn_like(p) - 1)
            elif "bias" in n:
                p.zero_()
            else:
                p.copy_(torch.randn_like(p) * (0.3 if "conv" in n else p.shape[-1] ** -0.5))
    return m


@pytest.mark.parametrize("kind", OPS)
def test_layers(kind, monkeypatch):
    """Recurrence and gated norm together in the layer, forward and backward, against the layer on tensor ops.

    Both sides round to bf16 behind the recurrence, the norm and each projection, apart by at most 2^-8 there: five such
    places forward, and as many again on the way back, where each meets the rounded gradient of the one behind it.
    Gradients of a few sums over all rows (one number per head) are left to the operators' own tests: what cancels in them
    has no such bound."""
    from xorl_b200.models import gated_deltanet, mamba2
    from xorl_b200.models.context import StepContext
    from xorl_b200.ops import norm, recurrence as R
    m = layer(kind)
    cuts = [0, 33, 34, 200]
    ctx = StepContext(cu_seqlens=boundaries(cuts), position_ids=torch.cat([torch.arange(b - a) for a, b in zip(cuts, cuts[1:])]).cuda(),
                      max_seqlen=166)
    x = torch.randn(200, 256, device="cuda").bfloat16()
    dy = torch.randn(200, 256, device="cuda").bfloat16()

    def run():
        xi = x.detach().requires_grad_()
        y = m(xi, ctx)
        return [y.detach(), *torch.autograd.grad(y, [xi, *m.parameters()], dy)]

    before = R.launch_count()
    got = run()
    assert R.launch_count() > before
    monkeypatch.setattr(R, "_kernel_ok", lambda *a: False)
    plain = lambda x, gate, w, group, eps, norm_first=True: norm._gated_rms_norm_ref(x, gate, w, group, eps, norm_first)  # noqa: E731
    monkeypatch.setattr(gated_deltanet, "gated_rms_norm", plain)
    monkeypatch.setattr(mamba2, "gated_rms_norm", plain)
    before = R.launch_count()
    want = run()
    assert R.launch_count() == before
    for i, (a, b) in enumerate(zip(got, want)):
        if a.numel() >= 64:
            assert (a.double() - b.double()).norm() <= (5 if i == 0 else 10) * 2.0 ** -8 * b.double().norm(), i
