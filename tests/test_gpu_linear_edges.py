"""GPU: linear_act's activations in f32 over fine grids and at infinite arguments, and its products where operands are infinite.

e = 2^-24, half a step of f32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _of_bias(z, act, rows=1):
    """(y, d) of a layer whose products are 0: act(z) and act'(z) of its bias z, on the vector units (1 row) or the matrix cores"""
    from ppo_amd import ops
    x, w = torch.zeros(rows, 2, device="cuda", dtype=z.dtype), torch.zeros(z.numel(), 2, device="cuda", dtype=z.dtype)
    y, d = ops.linear_act_fwd(x, w, z, act, want_deriv=True)
    return y[-1], d[-1]


@pytest.mark.parametrize("low,high", [(-12.0, 12.0), (-80.0, 80.0)])
def test_silu_derivative_keeps_its_digits(low, high):
    """d = s (1 + z r), s = s(z), r = s(-z).  e^-|z| is good to 4 half steps (an exp2 of 2, its correction, a product), 1 / (1 + e) to 3,
    their product to 8.  z >= 0: s 3, z r <= 0.28 to 9, the sum 1, the product 1: below 8 d.  z < 0: s 8 of d (and 1 for the product),
    r 3 and z r 1 more of s |z| <= 0.28, the sum 1 of s max(1, |1 + z r|): below 9 d + 2.  Bound: e (9 |d| + 2)."""
    z = torch.linspace(low, high, 1 << 20, device="cuda")
    x = z.double()
    s, r = torch.sigmoid(x), torch.sigmoid(-x)
    want = s * (1 + x * r)
    for rows in (1, 40):
        d = _of_bias(z[:: 1 if rows == 1 else 64].contiguous(), "silu", rows)[1].double()
        w = want[:: 1 if rows == 1 else 64]
        assert bool(((d - w).abs() <= E * (9 * w.abs() + 2) + 1e-37).all()), float(((d - w).abs() / (9 * w.abs() + 2)).max() / E)
