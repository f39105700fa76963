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

from tests.test_gpu_paged import Both, f64, ints

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


def test_the_smallest_and_largest_queries(cuda):
    """Rows of one value, of the smallest numbers, and with one value that is all of the row."""
    print("[case] extreme queries", flush=True)
    for D in (64, 128):
        b = held(D, 64, 1, 1, torch.bfloat16)
        q = torch.zeros((40, 1, D), dtype=torch.bfloat16, device="cuda")
        q[0] = 1.0
        q[1] = -1.0
        q[2, 0, 3] = 50.0
        q[3] = 2.0 ** -133
        q[4, 0, :5] = torch.tensor([2.0 ** -126, -2.0 ** -130, 2.0 ** -133, 2.0 ** -110, 0.0])
        q[5, 0, 7] = -2.0 ** 40
        q[6] = torch.linspace(-3, 3, D).to(torch.bfloat16)
        for rows in (7, 40):
            b.attend([0], [rows], 1, q=q[:rows].contiguous(), causal=False)


@pytest.mark.parametrize("power", [10, 20, 26, 27, 28, 40, 90])
@pytest.mark.parametrize("rows", [2, 40, 200])
def test_scores_of_any_size(cuda, rows, power):
    """Scores about 2^power, whose spacing in f32 is far above the softmax's range: the tokens of the largest
    weigh all, and nothing overflows.  Keys are powers of two of both signs, so that scores are exact whatever
    their size.  How those tokens share the weight is right where one wave or workgroup sees them: parts of a
    row are joined by their sums' exponents, which f32 rounds by 2^-24 of the score, more than a sum is worth
    from 2^24 on.  So an output lies between the smallest and the largest of those tokens' values, once rounded."""
    print(f"[case] scores rows={rows} power={power}", flush=True)
    D, n, T = 128, 500, 16
    b = Both(heads=1, D=D, T=T, seqs=1, width=-(-n // T), pages=-(-n // T), seed=power)
    b.extend([0], [n])
    k = np.zeros((n, 1, D))
    k[:, 0, 3] = b.rng.choice([-1.0, -0.5, 0.25, 0.5, 1.0], n) * 2.0 ** (power // 2)
    v = torch.from_numpy(b.rng.standard_normal((n, 1, D))).to(torch.bfloat16).cuda()
    b.append([0], [n], k=torch.from_numpy(k).to(torch.bfloat16).cuda(), v=v)
    b.same_codes()
    q = torch.zeros((rows, 2, D), dtype=torch.bfloat16, device="cuda")
    q[..., 3] = 2.0 ** (power - power // 2)
    q[:, 1, 3] *= -1
    for kw in (dict(causal=False), dict(), dict(window=50)):
        out = b.attend([0], [rows], 2, q=q, scale=1.0, **kw)
        held = f64(b.dev.read(0, ints([0]), n, dtype=torch.float32)[1])[:, 0]
        for r in range(rows):
            p = n - rows + r
            last = p + 1 if kw.get("causal", True) else n
            first = max(0, last - kw["window"]) if "window" in kw else 0
            for h, sign in ((0, 1), (1, -1)):
                s = sign * k[first:last, 0, 3]
                best = held[first:last][s == s.max()]
                o = f64(out[r, h])
                near = 2.0 ** -8 * np.abs(o) + 2.0 ** -20  # its rounding, and the sums' in f32
                assert (o >= best.min(0) - near).all() and (o <= best.max(0) + near).all()
