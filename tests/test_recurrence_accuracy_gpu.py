"""What the third bf16 parts of operands buy in the gated linear recurrences, in cases where two parts show.

Tolerances, of the norm of an output against 64 bits.  With three parts an operand keeps its 24 bits, and what is left are
roundings of fp32 values and of the accumulators.

Scan: at most eight roundings of 2^-24 after one another lie between the inputs and a state or its gradient: 2^-21.  A gradient of
dt is a difference of two such sums: 2^-20.

Delta rule inside a chunk: the tensor core cuts its sum to 24 bits after every step of 16 terms, always towards zero, so that
the errors add up: half a unit in the last place on average, 0.75 * 2^-24 of the partial sum, whose size grows as the root of
the steps and is 2/3 of the final one on average.  T R and T^T Y have 16 steps each, dR U^T has 24 for 64 columns: 28 * 2^-24
if all of them stood behind the whole result.  Three quarters of it do in the gradient of beta, half of which is dR.v without
dR U^T: 21 * 2^-24 = 1.25e-6.  (The same products with such sums, in 64 bits on the host: 0.9e-6 to 1.1e-6; with sums that are
rounded to the nearest: 2.5e-7.)  The gradient of the decay is a difference of two such sums: 42 * 2^-24 = 2.5e-6 (host: 1.5e-6
to 1.8e-6).

An operand of two parts is off by up to 2^-18 of itself.  Left out one at a time, the third parts of T and R in T R, of T and Y
in T^T Y, of dR and of U in dR U^T bring the gradient of beta to 1.8e-6, 2.8e-6, 3.5e-6, 2.1e-6, 1.5e-6, 3.6e-6 at least, those
of U in dO U^T the decay's to 1.5e-5; of the scan's added operands its states and their gradients to 2.3e-6, of the kept
gradients dt's to 2.1e-6, of the kept states dt's to 2.5e-6."""
import pytest
import torch

from test_recurrence_gpu import _need_cuda, leaves, oracle_delta, oracle_scan, scan_inputs  # noqa: F401

pytestmark = pytest.mark.gpu


def off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("seed", range(4))
def test_delta_products_inside_a_chunk(seed):
    """Documents of one chunk without states or decay: Q K^T, K K^T and P are exact, and T, R, Y, U and dR are all that rounds."""
    from xorl_b200.ops.recurrence import gated_delta_rule
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    T, cuts = 256, [0, 64, 128, 192, 256]
    sign = lambda: torch.cat([0.5 * torch.sign(r(T, 2, 4)), torch.zeros(T, 2, 4, device="cuda")], -1).bfloat16()  # noqa: E731
    ins = [sign(), sign(), r(T, 4, 64).bfloat16(), torch.zeros(T, 4, device="cuda"), torch.sigmoid(r(T, 4))]
    a, b = leaves(ins)
    o = gated_delta_rule(*a, torch.tensor(cuts, dtype=torch.int32, device="cuda"))
    ro, _ = oracle_delta(*b, cuts, 1.0, False, None)
    do = r(T, 4, 64).bfloat16()
    got, want = torch.autograd.grad(o, a[3:], do), torch.autograd.grad(ro, b[3:], do.double())
    assert off(got[1], want[1]) <= 21 * 2.0 ** -24, off(got[1], want[1])
    assert off(got[0], want[0]) <= 42 * 2.0 ** -24, off(got[0], want[0])


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("strength", [0.01, 1.0])
def test_scan_states_and_decay(seed, strength):
    """Several chunks: the states and their gradients, and the gradients of dt and A that read both."""
    from xorl_b200.ops.recurrence import ssd_scan
    cuts = [0, 320]
    a, b = leaves(scan_inputs(320, 1, 4, 128, 64, 1, seed=seed, state=True, strength=strength))
    y, S = ssd_scan(*a[:6], torch.tensor(cuts, dtype=torch.int32, device="cuda"), initial_state=a[6], return_final_state=True)
    ry, rS = oracle_scan(*b[:6], cuts, b[6])
    assert off(S.detach(), rS.detach()) <= 2.0 ** -21
    gen = torch.Generator(device="cuda").manual_seed(99)
    do, dS = torch.randn(y.shape, generator=gen, device="cuda").bfloat16(), torch.randn(S.shape, generator=gen, device="cuda")
    pick = (1, 2, 6)
    got = torch.autograd.grad([y, S], [a[i] for i in pick], [do, dS])
    want = torch.autograd.grad([ry, rS], [b[i] for i in pick], [do.double(), dS.double()])
    err = {n: off(x, z) for n, x, z in zip(("dt", "A", "state"), got, want)}
    assert err["state"] <= 2.0 ** -21 and err["dt"] <= 2.0 ** -20, err


@pytest.mark.parametrize("seed", range(4))
def test_scan_entering_state(seed):
    """Nothing is added to the state, so that dt's gradient is A times sums of C.(S dy): the kept state is all that rounds."""
    from xorl_b200.ops.recurrence import ssd_scan
    ins = list(scan_inputs(64, 1, 2, 128, 64, 1, seed=seed, state=True, strength=1.0))
    ins[0] = torch.zeros_like(ins[0])
    a, b = leaves(ins)
    y = ssd_scan(*a[:6], torch.tensor([0, 64], dtype=torch.int32, device="cuda"), initial_state=a[6])
    ry, _ = oracle_scan(*b[:6], [0, 64], b[6])
    dy = torch.randn(y.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
    got, want = torch.autograd.grad(y, a[1], dy)[0], torch.autograd.grad(ry, b[1], dy.double())[0]
    assert off(got, want) <= 2.0 ** -20, off(got, want)
