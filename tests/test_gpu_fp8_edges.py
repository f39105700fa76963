"""The block-scaled e4m3 linears at the ends of their ranges, against the restatement in 64 bits
(oracle/fp8_oracle.py) with the bounds of test_gpu_fp8."""
import numpy as np
import pytest
import torch

from eredu_amd import fp8
from oracle import fp8_oracle as F
from tests.test_gpu_fp8 import BF, HF, SF, case, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("least,most", [(-87.3, -80.0), (-88.7, -87.4), (-96.0, -89.0), (-110.0, -97.0), (-160.0, -105.0)])
def test_silu_mul_of_far_gates(cuda, least, most, dtype):
    """Gates whose sigmoid is at f32's smallest normal value and below it, with factors that bring the product back: groups
    of such gates alone, and of those among larger ones.  Below 2^-126 a product is rounded by 2^-150,
    which is 2^-24 of a quotient at the most (scales are 2^-126 or more), in the value and in its group's largest."""
    case("far gates", least, most, dtype)
    factors = (1.0, 60000.0) if dtype is HF else (1.0, 1e4, 1e30, 3e38)
    g = torch.linspace(least, most, 128, device="cuda").repeat(2 * len(factors))
    u = torch.cat([torch.linspace(0.5, 1, 128, device="cuda") * f for f in factors for _ in range(2)])
    for i in range(len(factors)):
        g[256 * i + 128:256 * i + 256:9] = torch.linspace(-12, 0.5, 15, device="cuda")
    g, u = g[None].to(dtype), u[None].to(dtype)
    got = fp8.silu_mul(g, u)
    q, s = F.quotients(F.silu_mul(f64(g), f64(u)))
    assert np.isfinite(s).all()
    c, err = f64(got.codes), 8 * 2.0 ** -24
    assert np.all(np.abs(f64(got.scales) - s) <= (err + 2.0 ** -23) * s)
    assert np.all(np.abs(c - q) <= F.step(q) / 2 + 3 * err * np.abs(q) + 2.0 ** -23)


def test_silu_mul_of_infinite_far_gates(cuda):
    """-inf is NaN (its sigmoid is 0), an infinite factor stays infinite, the farthest finite gates give nothing."""
    case("infinite far gates")
    g = torch.full((4, 128), -88.0, device="cuda")
    u = torch.ones(4, 128, device="cuda")
    g[0, 5], u[1, 6], g[2], u[2], g[3], u[3, 7] = -float("inf"), float("inf"), torch.finfo(SF).min, torch.finfo(SF).max, -400.0, float("nan")
    got = fp8.silu_mul(g, u)
    assert np.array_equal(np.isnan(f64(got.scales))[:, 0], [True, True, False, True])
    assert not f64(got.codes).any() and float(got.scales[2, 0]) == 2.0 ** -126
