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
