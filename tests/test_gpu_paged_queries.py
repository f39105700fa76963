"""Queries with channels far above the others over the paged cache: how many bits of a
row's largest magnitude a query is held in must not show in the output.

In the mean over many outputs, in units of what rounding the exact output costs:
  the output's rounding                    1
  f16 probabilities                        at most 1 (a probability is off as an f16 output is; less where few
                                           tokens weigh most, an eighth for bf16 outputs)
  the query's digits                       at most 1: two digits are taken where scale * log2 e * (a unit of the 16
                                           bits) * (the page's step) is at most 2^-15 / sqrt(D), so a score is off by
                                           0.29 * 2^-15 * 35 * ln 2 = 2.1e-4 with codes of a root mean square of
                                           35 (normal values, the largest of a page at 127), and rounding
                                           f16 costs 2.1e-4; bf16 four times and eight times as much
together sqrt(3) = 1.73 at most, and with a third digit, of 1/256, sqrt(2).
"""
import numpy as np
import pytest
import torch

from tests.test_gpu_paged import Both, f64

pytestmark = pytest.mark.gpu


def held(D, T, heads, r, dtype, spread=1.0, n=600):
    b = Both(heads=heads, D=D, T=T, seqs=1, width=-(-n // T), pages=-(-n // T), seed=int(r) + D)
    b.extend([0], [n])
    k = b.rng.standard_normal((n, heads, D)) * spread
    k[..., 5] /= r
    v = b.rng.standard_normal((n, heads, D))
    b.append([0], [n], k=torch.from_numpy(k).to(dtype).cuda(), v=torch.from_numpy(v).to(dtype).cuda())
    b.same_codes()
    return b


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [9, 60, 300])  # waves over runs of tiles, blocks of 64 rows and of 128
@pytest.mark.parametrize("r", [1, 8, 30, 100, 300])
def test_one_channel_above_the_others(cuda, r, rows, D, dtype):
    print(f"[case] channel r={r} rows={rows} D={D} {dtype}", flush=True)
    heads = 2
    b = held(D, 32, 2, r, dtype, spread=2.0 if r > 8 else 1.0)
    q = b.rng.standard_normal((rows, 2 * heads, D))
    q[..., 5] *= r
    q = torch.from_numpy(q).to(dtype).cuda()
    out = b.attend([0], [rows], 2 * heads, dtype=dtype, q=q, causal=False)
    exact = b.ref.attention(0, f64(q), [0], [rows], D ** -0.5, False, 0, None)[0]
    alone = np.sqrt(((f64(torch.from_numpy(exact).to(dtype)) - exact) ** 2).mean())
    off = np.sqrt(((f64(out) - exact) ** 2).mean()) / alone
    print(f"[off] {off:.2f} times a rounding", flush=True)
    assert off <= 1.75


@pytest.mark.parametrize("rows", [3, 70, 260])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_pages_on_both_sides_of_the_third_digit(cuda, rows, D):
    """Pages whose keys are 2^12 times as large as others', in one tile and in several, masked and windowed:
    every score is as near as its own page asks for, and causal rows see no more for it."""
    print(f"[case] mixed pages rows={rows} D={D}", flush=True)
    n, heads = 520, 2
    b = Both(heads=heads, D=D, T=16, seqs=1, width=-(-n // 16), pages=-(-n // 16), seed=D)
    b.extend([0], [n])
    k = b.rng.standard_normal((n, heads, D)) * 2.0 ** -8
    for first in (48, 160, 176, 400):
        k[first:first + 16] *= 2.0 ** 12
    v = b.rng.standard_normal((n, heads, D))
    b.append([0], [n], dtype=torch.float16, k=torch.from_numpy(k).half().cuda(), v=torch.from_numpy(v).half().cuda())
    b.same_codes()
    for kw in (dict(causal=False), dict(), dict(window=37), dict(rope=True)):
        b.attend([0], [rows], 3 * heads, dtype=torch.float16, **kw)
