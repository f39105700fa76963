"""Products large enough for each tile shape and for split K (the sizes are ones at which the
cost rule takes 256 x 256, 256 x 192, 256 x 128, 128 x 128, 128 x 96, 128 x 64 and 128 x 32 weight
by activation rows, whole and ragged, with K of whole blocks and with a short last one): every result against a
product in 64 bits on the GPU, and some rows and columns, the borders of tiles among them, against
the oracle, with the bounds of test_gpu_fp8."""
import numpy as np
import pytest
import torch

from eredu_amd import fp8
from oracle import fp8_oracle as F
from tests.test_gpu_fp8 import BF, HF, ROUND, SF, case, f64, ints, near

pytestmark = pytest.mark.gpu


def some(n, tile, rng):
    at = {0, n - 1, *(i for b in range(tile, n, tile) for i in (b - 1, b)), *rng.integers(0, n, 24)}
    return np.array(sorted(at))


def operands(seed, m, n, k, experts=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = fp8.quantize((torch.randn(m, k, generator=g, device="cuda") * torch.linspace(0.2, 3, k, device="cuda")).to(BF))
    shape = (n, k) if experts is None else (experts, n, k)
    return x, fp8.quantize_weight((torch.randn(shape, generator=g, device="cuda") * 0.05).to(BF))


def wide(codes, scales):
    """What a weight's codes and scales stand for, f64 on the GPU."""
    n, k = codes.shape
    s = scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return codes.double() * s


def check(y, x, w, s, rng, dtype):
    """y [m, n] = x . w^T of one weight."""
    m, n, k = y.shape[0], w.shape[0], w.shape[1]
    xd, wd = x.dequantize(torch.float64), wide(w, s)
    want, size = xd @ wd.T, xd.abs() @ wd.abs().T
    assert torch.isfinite(y).all()
    # (all of 8 products at the largest's place: 7 * 2^-13 of the sum of sizes at the most)
    bound = ((128 + k / 128 + 3) * 2.0 ** -23 + (0 if dtype is SF else 7 * 2.0 ** -13)) * size + ROUND[dtype] * want.abs() + 2.0 ** -25
    assert ((y.double() - want).abs() <= bound).all()
    r, c = some(m, 32, rng)[:400], some(n, 128, rng)[:400]
    rows, cols = torch.from_numpy(r).cuda(), torch.from_numpy(c).cuda()
    near(y[rows][:, cols], *F.matmul(f64(xd[rows]), f64(wd[cols])), k, dtype)


@pytest.mark.parametrize("m,n,k,dtype", [
    (1024, 14336, 4096, BF), (1150, 12800, 2064, HF),      # 256 x 256
    (1150, 8192, 2064, BF), (1151, 8195, 2064, BF),        # 256 x 192
    (512, 14336, 4096, BF), (380, 12799, 4112, HF),        # 256 x 128
    (700, 9001, 2000, BF), (1024, 14336, 1040, SF),        # 128 x 128
    (190, 14336, 2064, BF), (80, 4097, 14320, HF), (77, 4097, 14320, SF),  # 128 x 96, the second and third with K in 7 parts
    (250, 14000, 1040, BF),                                # 128 x 64
    (256, 4096, 8208, BF),
    (90, 130, 8208, BF), (97, 4097, 3088, HF), (90, 131, 8208, SF),        # 128 x 32, the first and last with split K
])
def test_shapes(cuda, m, n, k, dtype):
    case("tiles", m, n, k, dtype)
    x, (w, s) = operands(m + n, m, n, k)
    check(fp8.matmul(x, w, s, dtype), x, w, s, np.random.default_rng(n), dtype)


@pytest.mark.parametrize("routes,experts,n,k,dtype", [
    (1554, 8, 4096, 4112, BF), (900, 4, 4000, 4112, HF),  # 256 x 128
    (2300, 8, 4100, 2064, BF), (3000, 3, 2000, 272, BF),  # 128 x 128
    (800, 2, 3000, 4112, BF),    # 128 x 96
    (800, 2, 1500, 4112, SF), (4096, 128, 768, 2048, BF), (700, 20, 1000, 272, BF),  # 128 x 64
])
def test_shapes_of_routes(cuda, routes, experts, n, k, dtype):
    """Experts of very different numbers of routes (one has none), rows of x named twice, some routes without an expert."""
    case("tiles of routes", routes, experts, n, k, dtype)
    rng = np.random.default_rng(routes)
    rows = routes // 2 + 1
    x, (w, s) = operands(routes, rows, n, k, experts)
    ids = np.minimum((experts - 1) * rng.random(routes) ** 2.5, experts - 2).astype(np.int64) + (1 if experts > 2 else 0)
    ids[rng.random(routes) < 0.02] = -1
    at = rng.integers(0, rows, routes)
    y = fp8.grouped_matmul(x, w, s, ints(ids), ints(at), dtype)
    assert not y[torch.from_numpy(np.nonzero(ids < 0)[0]).cuda()].any()
    for e in np.unique(ids[ids >= 0]):
        mine = np.nonzero(ids == e)[0]
        src = torch.from_numpy(at[mine]).cuda()
        check(y[torch.from_numpy(mine).cuda()], fp8.Fp8Rows(x.codes.view(torch.uint8)[src].view(fp8.CODE_DTYPE), x.scales[src]),
              w[e], s[e], rng, dtype)


@pytest.mark.parametrize("m,n,k,dtype", [
    (466, 9729, 11744, BF), (2478, 6758, 3984, HF),   # 256 x 256, the second of each line behind whole passes
    (556, 6955, 13088, HF), (2579, 6894, 10000, BF),  # 256 x 192
    (1372, 1536, 12560, BF), (863, 9500, 9872, HF),   # 256 x 128
    (375, 10804, 12560, BF), (2195, 3857, 4784, SF),  # 128 x 128
    (66, 5554, 10288, HF),                            # 128 x 96
    (826, 134, 9280, BF), (2381, 1723, 4224, HF), (2571, 1766, 5472, SF),  # 128 x 64
    (29, 130, 4816, BF), (21, 236, 5040, SF),         # 128 x 32
])
def test_parts_of_the_last_pass(cuda, m, n, k, dtype):
    test_shapes(cuda, m, n, k, dtype)


@pytest.mark.parametrize("routes,experts,n,k,dtype", [
    (1660, 3, 7849, 1312, BF), (957, 5, 8098, 1232, HF),  # 256 x 256, 256 x 192, whole tiles
    (322, 2, 7487, 12864, BF), (1554, 8, 4096, 14336, BF),  # 256 x 128, the second with more tiles than workgroups at once
    (3010, 2, 391, 12160, HF), (577, 2, 2306, 14128, SF),  # 128 x 128
    (473, 2, 676, 11408, BF), (3838, 3, 191, 7984, SF),  # 128 x 96
    (1188, 2, 155, 7376, BF), (1075, 2, 198, 8800, SF),  # 128 x 64
    (84, 5, 201, 5472, HF), (115, 2, 130, 5552, SF),  # 128 x 32
])
def test_parts_of_the_last_pass_of_routes(cuda, routes, experts, n, k, dtype):
    test_shapes_of_routes(cuda, routes, experts, n, k, dtype)


def test_a_bank_of_over_2_31_bytes(cuda):
    """Offsets of the last experts pass 32 bits, few and many routes."""
    case("large bank")
    experts, n, k = 9, 16384, 16384
    assert experts * n * k > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.empty(experts, n, k, dtype=fp8.CODE_DTYPE, device="cuda")
    for e in range(experts):
        w[e] = (torch.randn(n, k, generator=g, device="cuda") * 100).clamp_(-448, 448).to(fp8.CODE_DTYPE)
    s = torch.rand(experts, n // 128, k // 128, generator=g, device="cuda") + 0.5
    x = fp8.quantize(torch.randn(70, k, generator=g, device="cuda").to(BF))
    rng = np.random.default_rng(4)
    for routes in (3, 70):
        ids = ints([experts - 1] * routes)
        y = fp8.grouped_matmul(x, w, s, ids, ints(range(routes)), BF)
        check(y, fp8.Fp8Rows(x.codes[:routes], x.scales[:routes]), w[-1], s[-1], rng, BF)


def test_more_routes_than_a_workgroup_keeps(cuda):
    """Over 4096 routes, whose expert ids are read a second time, and over 1024 experts."""
    case("many routes")
    rng = np.random.default_rng(5)
    for routes, experts in ((9001, 7), (5000, 2000)):
        x, (w, s) = operands(routes, 300, 130, 144, experts)
        ids, at = rng.integers(-1, experts + 1, routes), rng.integers(0, 300, routes)
        y = f64(fp8.grouped_matmul(x, w, s, ints(ids), ints(at), SF))
        xd = f64(x.dequantize(torch.float64))
        real = (ids >= 0) & (ids < experts)
        assert not y[~real].any()
        wd = F.weight_of(f64(w), f64(s))
        for r in np.nonzero(real)[0][::37]:
            want, size, _ = F.matmul(xd[at[r]:at[r] + 1], wd[ids[r]])
            assert np.all(np.abs(y[r] - want[0]) <= (128 + 2 + 3) * 2.0 ** -23 * size[0] + 2.0 ** -24 * np.abs(want[0]))
        assert np.all(np.abs(y[real]).max(1) > 0)


@pytest.mark.parametrize("routes,experts", [(1023, 5), (1025, 300), (16385, 1), (65536, 6), (65537, 1100), (200003, 3)])
def test_every_route_is_placed_once(cuda, routes, experts):
    """Routes in one and in several parts, up to more than 64 parts of 1024: each gets its own expert's product of its own row."""
    case("parts of routes", routes, experts)
    rng = np.random.default_rng(routes)
    x, (w, s) = operands(routes, 40, 16, 16, experts)
    ids, at = rng.integers(-1, experts + 1, routes), rng.integers(-1, 41, routes)
    y = f64(fp8.grouped_matmul(x, w, s, ints(ids), ints(at), SF))
    xd, wd = f64(x.dequantize(torch.float64)), F.weight_of(f64(w), f64(s))
    real = (ids >= 0) & (ids < experts) & (at >= 0) & (at < 40)
    assert not y[~real].any()
    e, r = ids[real], at[real]
    want, size = np.einsum("rk,rnk->rn", xd[r], wd[e]), np.einsum("rk,rnk->rn", np.abs(xd[r]), np.abs(wd[e]))
    # 16 exact products, summed in f32 with 2^-23 of the sizes a sum, the scales' product and two more roundings
    assert np.all(np.abs(y[real] - want) <= (16 + 2 + 3) * 2.0 ** -23 * size + 2.0 ** -24 * np.abs(want))


def test_routes_give_the_same_bits_every_time(cuda):
    """Unsorted routes of which some experts' last tiles are taken in parts of K: their places do not depend on who comes first."""
    case("repeated routes")
    x, (w, s) = operands(8, 300, 3000, 12864, 3)
    rng = np.random.default_rng(8)
    ids, at = ints(rng.integers(0, 3, 1100)), ints(rng.integers(0, 300, 1100))
    want = fp8.grouped_matmul(x, w, s, ids, at, BF)
    for _ in range(6):
        assert torch.equal(fp8.grouped_matmul(x, w, s, ids, at, BF), want)
    for e in range(3):
        mine = torch.nonzero(ids == e)[:, 0]
        xd, wd = x.dequantize(torch.float64)[at[mine].long()], wide(w[e], s[e])
        size = xd.abs() @ wd.abs().T
        bound = ((128 + 12864 / 128 + 3) * 2.0 ** -23 + 7 * 2.0 ** -13) * size + ROUND[BF] * (xd @ wd.T).abs() + 2.0 ** -25
        assert ((want[mine].double() - xd @ wd.T).abs() <= bound).all()
