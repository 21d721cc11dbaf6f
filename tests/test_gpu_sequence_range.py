"""The sequence operators at the ends of their numbers' range: large logits, infinities, values too small to be normal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ds_splat_b200 as ds  # noqa: E402

U = 2.0 ** -24
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("channels", [4, 2, 1])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_both_decays_keep_their_relative_precision_for_large_logits(dtype, channels, single):
    """f and 1 - f by themselves: one row from the state 1 with the input 0, and one coupled row from 0 with the input 1, whose
    products and sums are exact; the last state is 32-bit.  In units of U = 2^-24, with e = exp(-g): the exponential 4 (2 ulp),
    its argument's correction 1, the sum 1 + e 1, the reciprocal 2 (1 ulp), the product e f 1, so 8 for f and 9 for 1 - f.
    A 16-bit gate's argument is rounded: 1.22 |g| (half a step of the product, 0.22 by the constant's own rounding) more."""
    g = torch.linspace(-80, 80, 20004, dtype=torch.float64).to(DTYPES[dtype])
    gate = g.cuda().view(-1, channels)
    n = gate.shape[0]
    exact = g.double().numpy().reshape(n, channels)
    bound = 9 + (1.22 * np.abs(exact) if dtype != "fp32" else 0)
    for coupled, x, state, want in ((False, 0.0, 1.0, 1 / (1 + np.exp(-exact))), (True, 1.0, 0.0, 1 / (1 + np.exp(exact)))):
        x = torch.full_like(gate, x)
        last = torch.full((n, channels), state, device="cuda")
        if single:
            ds.gated_recurrence_step(x, gate, last, coupled=coupled)
        else:
            _, last = ds.gated_recurrence(x[:, None], gate[:, None], last, coupled=coupled)
        off = np.abs(last.double().cpu().numpy() - want) / want / U
        worst = (off / bound).argmax()
        assert (off <= bound).all(), f"coupled {coupled}: off by {off.flat[worst]:.1f} U at the logit {exact.flat[worst]:.2f}"


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_what_is_not_finite_stays_so_to_the_end_of_its_sequence_and_nowhere_else(dtype, reverse, value):
    """One input of one channel.  From its row on the channel holds infinities or NaN: an infinity may have become a NaN where the
    decays between have a product below 2^-126.  Rows before, other channels, other sequences keep their bits, as do their gradients,
    except where the sum of a gradient takes the row in: the gate's of the same channel and the inputs' of no row."""
    t = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(t)  # noqa: E731
    rows, at, c = 3000, 1234, 5
    clean, gate, v_h = rand(3, rows, 16), rand(3, rows, 16) - 1, rand(3, rows, 16)
    bad = clean.clone()
    bad[1, at, c] = value
    out = []
    for x in (clean, bad):
        leaves = [x.requires_grad_(), gate.detach().requires_grad_()]
        h, last = ds.gated_recurrence(*leaves, reverse=reverse)
        out.append((h.detach(), last.detach(), *torch.autograd.grad(h, leaves, v_h)))
    (h0, last0, dx0, dg0), (h1, last1, dx1, dg1) = out
    reached = torch.zeros(3, rows, 16, dtype=torch.bool, device="cuda")
    reached[1, :at + 1, c] = reverse
    reached[1, at:, c] |= not reverse
    assert torch.equal(torch.isfinite(h1), ~reached) and torch.equal(h1[~reached], h0[~reached])
    ends = torch.zeros(3, 16, dtype=torch.bool, device="cuda")
    ends[1, c] = True
    assert torch.equal(torch.isfinite(last1), ~ends) and torch.equal(last1[~ends], last0[~ends])
    assert torch.equal(dx1, dx0)                               # h_t is linear in x: nothing of x is in its gradient
    assert torch.equal(dg1[~reached], dg0[~reached])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_values_too_small_to_be_normal_may_count_as_zero(dtype):
    small = torch.tensor([1e-39, -1e-40, 2.0 ** -24, 0.0], device="cuda").to(DTYPES[dtype]).view(1, 1, 4)
    out = ds.dropout(small, 0.0, (1, 2))
    assert ((out.double() - small.double()).abs() < 2.0 ** -126).all()
    h, last = ds.gated_recurrence(small, torch.zeros_like(small), form="decay")
    assert ((h.double() - small.double()).abs() < 2.0 ** -126).all() and ((last[:, None].double() - small.double()).abs() < 2.0 ** -126).all()
