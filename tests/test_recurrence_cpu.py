"""The gated linear recurrences and the gated norm without a GPU: what they refuse, and their tensor-op forms against the
token-by-token definition in 64 bits.

Tolerances: the tensor-op forms are fp32; a result passes at most four products in a row that add up at most 128 terms
of 2^-24 each with two operands, and factors e^G with |G| <= 8 from sums of at most 128 terms: 4 * 2 * 128 * 2^-24 +
128 * 8 * 2^-24 = 1.3e-4 of what the sums add up, for which the largest value stands."""
import pytest
import torch

from test_recurrence_gpu import oracle_delta, oracle_scan
from xorl_b200.ops.norm import gated_rms_norm
from xorl_b200.ops.recurrence import gated_delta_rule, ssd_scan

HELD = 4 * 2 * 128 * 2.0 ** -24 + 128 * 8 * 2.0 ** -24


def delta_inputs(T=70, hk=2, hv=4, dk=8, dv=16, docs=1, state=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return [r(T, hk, dk), r(T, hk, dk), r(T, hv, dv), -0.1 * torch.nn.functional.softplus(r(T, hv)), torch.sigmoid(r(T, hv)),
            0.3 * r(docs, hv, dk, dv) if state else None]


def scan_inputs(T=70, groups=2, heads=4, N=8, P=16, docs=1, state=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return [r(T, heads, P), 0.1 * torch.nn.functional.softplus(r(T, heads)), -0.1 * (1 + torch.arange(heads, dtype=torch.float32)),
            r(T, groups, N), r(T, groups, N), r(heads), 0.3 * r(docs, heads, P, N) if state else None]


def cu(*cuts):
    return torch.tensor(cuts, dtype=torch.int32)


def without(ts, i, value):
    return [value if j == i else t for j, t in enumerate(ts)]


def test_refusals_of_the_delta_rule():
    ins = delta_inputs()
    call = lambda ts, c=cu(0, 70), **kw: gated_delta_rule(*ts[:5], c, **kw)  # noqa: E731
    call(ins)
    for i, bad in ((0, ins[0][:, 0]), (1, ins[1][:69]), (1, ins[1][..., :4]), (2, ins[2][:69]), (2, ins[2][:, :3]), (2, ins[2][..., :0]),
                   (3, ins[3][:, :2]), (4, ins[4][:69]), (3, ins[3].to("meta")), (1, ins[1].to("meta"))):
        with pytest.raises(ValueError, match="gated_delta_rule"):
            call(without(ins, i, bad))
    for c in (torch.tensor([[0, 70]]), torch.tensor([0.0, 70.0]), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="cu_seqlens"):
            call(ins, c)
    for scale in (0.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            call(ins, scale=scale)
    for s in (torch.zeros(2, 4, 8, 16), torch.zeros(1, 4, 16, 8), torch.zeros(1, 4, 8, 16, device="meta")):
        with pytest.raises(ValueError, match="initial_state"):
            call(ins, initial_state=s)


def test_refusals_of_the_scan():
    ins = scan_inputs()
    call = lambda ts, c=cu(0, 70), **kw: ssd_scan(*ts[:6], c, **kw)  # noqa: E731
    call(ins)
    for i, bad in ((0, ins[0][:69]), (0, ins[0][:, :3]), (1, ins[1][:, :2]), (2, ins[2][:3]), (3, ins[3][..., :4]), (4, ins[4][:, :1]),
                   (5, ins[5].view(4, 1)), (5, ins[5].to("meta"))):
        with pytest.raises(ValueError, match="ssd_scan"):
            call(without(ins, i, bad))
    with pytest.raises(ValueError, match="cu_seqlens"):
        call(ins, torch.tensor([0.0, 70.0]))
    with pytest.raises(ValueError, match="initial_state"):
        call(ins, initial_state=torch.zeros(1, 4, 8, 16))


def test_refusals_of_the_norm():
    x = torch.randn(4, 32)
    for args in ((x, x[:3], torch.ones(8), 8), (x, x, torch.ones(8), 5), (x, x, torch.ones(16), 8), (x, x, torch.ones(8), 0),
                 (x, x.to("meta"), torch.ones(8), 8), (x, x, torch.ones(8, device="meta"), 8), (x[:, :0], x[:, :0], torch.ones(8), 8)):
        with pytest.raises(ValueError, match="gated_rms_norm"):
            gated_rms_norm(*args)


def close(got, ref, name):
    got, ref = got.double(), ref.detach()
    assert got.shape == ref.shape, name
    if ref.numel():
        assert (got - ref).abs().max() <= HELD * ref.abs().max() + 1e-30, (name, (got - ref).abs().max(), ref.abs().max())


@pytest.mark.parametrize("cuts", [(0, 70), (0, 1, 1, 40, 70), (3, 30, 60)])
@pytest.mark.parametrize("op", ["delta", "scan"])
def test_tensor_op_forms(op, cuts):
    docs = len(cuts) - 1
    ins = (delta_inputs if op == "delta" else scan_inputs)(docs=docs, state=True)
    a, b = [t.clone().requires_grad_() for t in ins], [t.double().requires_grad_() for t in ins]
    if op == "delta":
        o, S = gated_delta_rule(*a[:5], cu(*cuts), scale=0.5, qk_l2norm=True, initial_state=a[5], return_final_state=True)
        ro, rS = oracle_delta(*b[:5], list(cuts), 0.5, True, b[5])
    else:
        o, S = ssd_scan(*a[:6], cu(*cuts), initial_state=a[6], return_final_state=True, chunk=16)
        ro, rS = oracle_scan(*b[:6], list(cuts), b[6])
    close(o.detach(), ro, "o")
    close(S.detach(), rS, "state")
    gen = torch.Generator().manual_seed(5)
    do, dS = torch.randn(o.shape, generator=gen), torch.randn(S.shape, generator=gen)
    torch.autograd.backward([o, S], [do, dS])
    torch.autograd.backward([ro, rS], [do.double(), dS.double()])
    for i, (x, y) in enumerate(zip(a, b)):
        close(x.grad, y.grad, i)


@pytest.mark.parametrize("op", ["delta", "scan"])
def test_states_carry_from_call_to_call(op):
    """A document in pieces, each with the state that the piece before it left."""
    ins = (delta_inputs if op == "delta" else scan_inputs)()

    def call(s, e, state):
        part = [t[s:e] if t.dim() > 1 else t for t in ins if t is not None]
        fn = gated_delta_rule if op == "delta" else ssd_scan
        return fn(*part, cu(0, e - s), initial_state=state, return_final_state=True)

    whole, last = call(0, 70, None)
    state, rows = None, []
    for s, e in ((0, 1), (1, 33), (33, 33), (33, 70)):
        o, state = call(s, e, state)
        rows.append(o)
    close(torch.cat(rows), whole.double(), "o")
    close(state, last.double(), "state")
