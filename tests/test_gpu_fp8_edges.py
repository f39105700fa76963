"""The block-scaled e4m3 linears at the ends of their ranges, and in the tile shapes that the sizes of
test_gpu_fp8_tiles leave out, against the restatement in 64 bits (oracle/fp8_oracle.py) with the bounds of test_gpu_fp8."""
import numpy as np
import pytest
import torch

from eredu_amd import fp8
from oracle import fp8_oracle as F
from tests import test_gpu_fp8_tiles as tiles
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


def drawn_ids(rng, routes, experts):
    """The experts that test_shapes_of_routes draws."""
    ids = np.minimum((experts - 1) * rng.random(routes) ** 2.5, experts - 2).astype(np.int64) + (1 if experts > 2 else 0)
    ids[rng.random(routes) < 0.02] = -1
    return ids


@pytest.mark.parametrize("m,n,k,dtype", [
    (16549, 920, 2400, BF), (278, 12801, 15952, HF),      # 128 x 128 and 128 x 96, the last pass in parts of K behind a whole one
    (11130, 20, 15936, SF), (1694, 16, 7728, SF),         # 128 x 128 and 128 x 64 in parts
    (8342, 132, 16, SF), (8611, 20, 16, SF),              # 128 x 96 and 128 x 64, whole
])
def test_more_shapes(cuda, m, n, k, dtype):
    tiles.test_shapes(cuda, m, n, k, dtype)


@pytest.mark.parametrize("routes,experts,n,k,dtype", [
    (8720, 2, 473, 16048, BF), (21714, 2, 2321, 10128, BF),  # 256 x 256 in parts of K, the second behind whole passes
    (16018, 8, 414, 12864, HF),                              # 256 x 128 in parts behind whole passes
    (21850, 2, 271, 7904, BF), (22844, 3, 261, 7936, SF),    # the same of 128 x 128
    (146, 2, 11557, 13184, HF), (16903, 8, 134, 14240, SF),  # the same of 128 x 96
    (16437, 3, 129, 16, SF), (16401, 3, 16, 16, SF),         # 128 x 128 and 128 x 96, whole
    (66, 2, 16, 16, BF), (67, 2, 16, 16, SF),                # 128 x 32, whole
])
def test_more_shapes_of_routes(cuda, routes, experts, n, k, dtype):
    tiles.test_shapes_of_routes(cuda, routes, experts, n, k, dtype)


@pytest.mark.parametrize("routes,experts", [(65, 3), (256, 300), (257, 2), (16384, 5), (16385, 4)])
def test_routes_in_one_part_and_at_the_borders_of_parts(cuda, routes, experts):
    """A workgroup places 256 routes, or more where 64 workgroups would not do."""
    tiles.test_every_route_is_placed_once(cuda, routes, experts)


def bits(t):
    return t.view(torch.uint8) if t.dtype is fp8.CODE_DTYPE else t


def test_calls_give_the_same_bits_every_time(cuda):
    """Each operator, the products in each way they are done: few rows, whole tiles, tiles in parts of K."""
    g = torch.Generator(device="cuda").manual_seed(9)

    def rows(m, k):
        return torch.randn(m, k, generator=g, device="cuda").to(BF)

    w, s = fp8.quantize_weight(rows(4097, 14320))
    x, wide, gain = rows(300, 14320), rows(300, 2 * 2064), rows(1, 14320)[0]
    calls = [lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x), lambda: fp8.rms_norm(x.clone(), gain, 1e-5, x),
             lambda: fp8.silu_mul(wide[:, :2064], wide[:, 2064:])]
    calls += [lambda m=m, d=d: (fp8.matmul(x[:m], w, s, d),) for m in (1, 3, 16, 77, 300) for d in (BF, SF)]
    for i, call in enumerate(calls):
        case("repeated call", i)
        want = call()
        for _ in range(5):
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(call(), want))


def test_what_passes_the_range_of_f32(cuda):
    """Rows whose sum of squares is infinite become zeros, and where a block's two scales pass f32's range together the results
    are not finite, those of other rows being as they are."""
    case("past f32")
    x = torch.full((2, 256), 2.0, dtype=BF, device="cuda")
    x[0] = 1e25
    r = fp8.rms_norm(x, torch.ones(256, dtype=BF, device="cuda"), 1e-5)
    assert not f64(r.codes[0]).any() and np.all(f64(r.scales[0]) == 2.0 ** -126)
    assert np.all(f64(r.codes[1]) == 448)
    for m in (2, 40):
        rows = torch.full((m, 128), 1.0, dtype=SF, device="cuda")
        rows[0] = 1e30
        w, s = fp8.quantize_weight(torch.full((16, 128), 1e25, dtype=SF, device="cuda"))
        for dtype in (BF, SF):
            y = fp8.matmul(fp8.quantize(rows), w, s, dtype)
            # 128 products of 1 and 1e25: every code is 448 and every sum exact but for the scales' and the result's roundings
            assert not torch.isfinite(y[0]).any() and np.all(np.abs(f64(y[1:]) / 1.28e27 - 1) < 2.0 ** -8 + 2.0 ** -11)


def repeated(base, times):
    """[times * len(base), K] of the same rows again and again."""
    return base.expand(times, *base.shape).reshape(-1, base.shape[1])


def test_rows_past_2_32_values(cuda):
    """Values, codes and results whose offsets pass 32 bits: rows of the same values give the same codes and results wherever they lie."""
    case("large rows")
    g = torch.Generator(device="cuda").manual_seed(12)
    few, times, K = 1024, 264, 16384
    assert few * times * K > 1 << 32 and few * times * -(-K // 128) < 1 << 26
    base = torch.randn(few, K, generator=g, device="cuda").to(BF)
    gain = torch.randn(K, generator=g, device="cuda").to(BF)
    x = repeated(base, times)
    same = lambda got, want: all(torch.equal(bits(got[0][i:i + few]), bits(want[0])) and torch.equal(got[1][i:i + few], want[1])
                                 for i in range(0, few * times, few))
    codes = fp8.quantize(x)
    assert same(codes, fp8.quantize(base))
    assert same(fp8.silu_mul(x, x), fp8.silu_mul(base, base))
    w, s = fp8.quantize_weight(torch.randn(40, K, generator=g, device="cuda").to(BF))
    y = fp8.matmul(codes, w, s, BF)
    for i in (0, few * (times // 2), few * (times - 1)):  # (the last rows' tiles are in parts of K, summed in another order)
        tiles.check(y[i:i + few], fp8.Fp8Rows(codes.codes[i:i + few], codes.scales[i:i + few]), w, s, np.random.default_rng(1), BF)
    assert all(torch.equal(y[i:i + few], y[:few]) for i in range(0, few * (times // 2), few))
    assert torch.equal(fp8.matmul(x, w, s), y)
    want = base + base
    assert same(fp8.rms_norm(x, gain, 1e-5, x.clone()), fp8.rms_norm(want.clone(), gain, 1e-5))
    assert all(torch.equal(x[i:i + few], want) for i in range(0, few * times, few))


def test_results_past_2_32_values(cuda):
    """y of more than 2^32 values, of rows and of routes."""
    case("large results")
    g = torch.Generator(device="cuda").manual_seed(13)
    few, times, K, N = 1024, 264, 144, 16400
    assert few * times * N > 1 << 32
    base = torch.randn(few, K, generator=g, device="cuda").to(BF)
    w, s = fp8.quantize_weight(torch.randn(N, K, generator=g, device="cuda").to(BF))
    codes = fp8.quantize(repeated(base, times))
    y = fp8.matmul(codes, w, s, BF)
    tiles.check(y[:few], fp8.Fp8Rows(codes.codes[:few], codes.scales[:few]), w, s, np.random.default_rng(2), BF)
    assert all(torch.equal(y[i:i + few], y[:few]) for i in range(0, few * times, few))
    del y
    rows = torch.arange(few, dtype=torch.int32, device="cuda").repeat(times)
    z = fp8.grouped_matmul(fp8.quantize(base), w[None], s[None], torch.zeros_like(rows), rows, BF)
    assert all(torch.equal(z[i:i + few], z[:few]) for i in range(0, few * times, few))
    tiles.check(z[:few], fp8.quantize(base), w, s, np.random.default_rng(2), BF)
