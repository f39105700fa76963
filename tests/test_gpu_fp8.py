"""The block-scaled e4m3 linears on the GPU (include/eredu_fp8.h, through eredu_amd.fp8)
against their restatement in 64 bits (oracle/fp8_oracle.py).

Codes of 16-bit values and of weights are equal, ties included; scales are off by the
roundings of one division, 2^-23.  Codes of values that were computed in f32 (norm, silu,
and f32 rows, whose product with 448 is rounded) lie next to a quotient that is off by
3 u (the value, its group's largest, and their quotient): |code - q| <= step(q) / 2 + 3 u |q|.
  norm: sums of squares of at most 24 values a thread, 6 steps in the wave and 16 waves,
  halved by the root; root, quotient, inverse and two products: u = (46 / 2 + 8) 2^-24
  silu: 2^t a step (two halves), its correction, the sum, the reciprocal a step, two products: u = 8 * 2^-24
  f32 rows: u = 2^-24

Products, with A = sum |x| |w| over a row and a column: f32 sums of 128 products and of
K / 128 blocks, each at most a step of 2^-23 of what they add up, and three products with
scales: (128 + K / 128 + 3) 2^-23 A; the result is rounded once, h |y| (bf16 2^-8, f16 2^-11,
f32 2^-24) or half of f16's smallest step.  For results of 16 bits the matrix cores cut each of 8
neighbouring products off at 2^-13 of the power of two below the largest's factors, which is at most the largest: of
the 8 the largest itself loses nothing, so 7 * 2^-13 of it, summed over the eights.
"""
import numpy as np
import pytest
import torch

from eredu_amd import EreduError, fp8
from oracle import fp8_oracle as F

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF: 2.0 ** -8, HF: 2.0 ** -11, SF: 2.0 ** -24}


def f64(t):
    return t.detach().double().cpu().numpy()


def values(rng, shape, dtype=BF, spread=0.7):
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[-1]))
    return torch.from_numpy(x).to(dtype).cuda()


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def weights(rng, *shape):
    w = torch.from_numpy(rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal((shape[-2], 1)))).to(BF).cuda()
    return fp8.quantize_weight(w)


def near_codes(got, q, s, u, zero=None):
    """Fp8Rows `got` against quotients q and scales s that were computed with a relative error of u."""
    c, sc = f64(got.codes), f64(got.scales)
    assert c.shape == q.shape and sc.shape == s.shape
    nan = np.isnan(s)
    assert np.array_equal(np.isnan(sc), nan)
    assert np.all(np.abs(sc - s)[~nan] <= (u + 2.0 ** -23) * s[~nan])
    assert np.all(np.abs(c - q) <= F.step(q) / 2 + 3 * u * np.abs(q))


def near(y, want, size, eights, K, dtype):
    assert y.dtype == dtype
    got = f64(y)
    assert got.shape == want.shape
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    bound = (128 + K / 128 + 3) * 2.0 ** -23 * size + ROUND[dtype] * np.abs(want) + (2.0 ** -25 if dtype is HF else 0)
    if dtype is not SF:
        bound += 7 * 2.0 ** -13 * eights
    off = np.abs(got - want)[~bad]
    assert np.all(off <= bound[~bad]), float((off / bound[~bad]).max())


def case(*a):
    print("[case]", *a, flush=True)


# ------------------------------------------------------------ codes

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 4096), (3, 128), (5, 144), (17, 400), (130, 1040), (2, 20000)])
def test_quantize_is_exact(cuda, rows, cols, dtype):
    case("quantize", rows, cols, dtype)
    x = values(np.random.default_rng(rows + cols), (rows, cols), dtype)
    r = fp8.quantize(x)
    c, s = F.quantize(f64(x))
    assert np.array_equal(f64(r.codes), c) and np.array_equal(f64(r.scales), s)
    assert r.scales.stride() == (1, rows) or rows == 1


def test_quantize_ties(cuda):
    """Rows whose quotients are ties between two codes, of both signs."""
    case("ties")
    table = F.decode_table()
    codes = np.sort(np.unique(table[np.isfinite(table)]))
    ties = (codes[1:] + codes[:-1]) / 2
    for scale in (1.0, 2.0 ** -20, 7.0, 2.0 ** 100):
        x = np.zeros((2, 128))
        x[0, :126], x[1, :126] = ties[:126], ties[126:]
        x[:, 127] = 448
        t = torch.from_numpy(x * scale).to(SF).cuda()
        assert np.array_equal(f64(t), x * scale)
        r = fp8.quantize(t)
        assert np.array_equal(f64(r.codes), F.nearest(x)), scale


def test_quantize_f32(cuda):
    case("f32")
    x = values(np.random.default_rng(5), (33, 416), SF)
    near_codes(fp8.quantize(x), *F.quotients(f64(x)), 2.0 ** -24)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_quantize_of_rare_values(cuda, dtype):
    """Zeros, the smallest and the largest values, infinities and NaN, each in a group of its own."""
    case("rare", dtype)
    lim = torch.finfo(dtype)
    x = torch.zeros(1, 8 * 128, dtype=SF)
    x[0, 128:256] = lim.smallest_normal
    x[0, 256:384] = lim.max
    x[0, 256] = -lim.max
    x[0, 390] = float("inf")
    x[0, 600] = float("nan")
    x[0, 700] = -float("inf")
    x[0, 640:660] = 3.0
    x[0, 800] = lim.smallest_normal * 2.0 ** -6  # a subnormal value beside none
    x[0, 900:910] = lim.max
    x[0, 910] = lim.smallest_normal
    x = x.to(dtype).cuda()
    r = fp8.quantize(x)
    q, s = F.quotients(f64(x))
    assert np.array_equal(np.isnan(f64(r.scales)), np.isnan(s))
    if dtype is SF:
        near_codes(r, q, s, 2.0 ** -24)
    else:
        assert np.array_equal(f64(r.codes), F.nearest(q))
    assert np.array_equal(np.signbit(f64(r.codes)[0, 256:258]), [True, False])


def test_quantize_layouts(cuda):
    """Slices of a wider tensor, turned ones, more dimensions, one row, none."""
    case("layouts")
    x = values(np.random.default_rng(6), (6, 10, 320), BF)
    want = fp8.quantize(x.reshape(60, 320))
    for got, at in ((fp8.quantize(x), slice(0, 60)), (fp8.quantize(x[2]), slice(20, 30)), (fp8.quantize(x[3, 4]), slice(34, 35))):
        assert torch.equal(got.codes.view(torch.uint8).reshape(-1, 320), want.codes[at].view(torch.uint8))
        assert torch.equal(got.scales.reshape(-1, 3), want.scales[at])
    part = fp8.quantize(x.reshape(60, 320)[:, 128:304])
    assert torch.equal(part.codes[:, :128].view(torch.uint8), want.codes[:, 128:256].view(torch.uint8))
    odd = fp8.quantize(x.reshape(60, 320)[:, 1:129])  # not 16-byte aligned
    assert torch.equal(odd.codes.view(torch.uint8), fp8.quantize(x.reshape(60, 320)[:, 1:129].clone()).codes.view(torch.uint8))
    turned = x[:, :, :60].reshape(60, 60)[:48, :48].t()
    assert torch.equal(fp8.quantize(turned).codes.view(torch.uint8), fp8.quantize(turned.contiguous()).codes.view(torch.uint8))
    none = fp8.quantize(x[:, :0])
    assert none.codes.shape == (6, 0, 320) and none.scales.shape == (6, 0, 3)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (130, 400), (1, 144), (3, 64, 272), (2, 2, 257, 128)])
def test_quantize_weight(cuda, shape, dtype):
    case("weight", shape, dtype)
    w = values(np.random.default_rng(sum(shape)), shape, dtype)
    c, s = fp8.quantize_weight(w)
    want_c, want_s = F.quantize_weight(f64(w))
    assert np.array_equal(f64(s), want_s)
    if dtype is SF:
        assert np.mean(f64(c) != want_c) < 1e-3 and np.all(np.abs(f64(c) - want_c) <= F.step(want_c) * 1.001)
    else:
        assert np.array_equal(f64(c), want_c)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,dim,residual", [(1, 16, True), (1, 4096, True), (3, 144, False), (5, 4112, True), (2, 8192, True),
                                               (2, 8208, False), (2, 16384, True), (3, 20000, True), (300, 128, True)])
def test_rms_norm(cuda, rows, dim, residual, dtype):
    case("norm", rows, dim, residual, dtype)
    rng = np.random.default_rng(rows * dim)
    x, w = values(rng, (rows, dim), dtype), values(rng, (dim,), dtype, 0.0)
    r = values(rng, (rows, dim), dtype) if residual else None
    kept = x.clone()
    got = fp8.rms_norm(x, w, 1e-5, r)
    hidden = (kept.float() + r.float()).to(dtype) if residual else kept
    assert torch.equal(x, hidden)
    near_codes(got, *F.quotients(F.rms_norm(f64(hidden), f64(w), 1e-5)), 31 * 2.0 ** -24)


def test_rms_norm_of_zeros_and_unfinite_rows(cuda):
    case("norm rare")
    x = torch.zeros(4, 256, dtype=BF, device="cuda")
    x[1, 3], x[2, 200], x[3] = float("inf"), float("nan"), 2.0
    w = torch.ones(256, dtype=BF, device="cuda")
    r = fp8.rms_norm(x, w, 0.0)  # 0 * inf: NaN in the first row; beside an infinity what is finite becomes 0
    assert np.array_equal(np.isnan(f64(r.scales)), [[True, True], [True, False], [True, True], [False, False]])
    assert not f64(r.codes[:3]).any()
    assert np.array_equal(f64(r.codes[3]), np.full(256, 448.0))
    r = fp8.rms_norm(x[:1], w, 1e-5)
    assert not f64(r.codes).any() and np.all(f64(r.scales) == 2.0 ** -126)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 14336), (48, 14336), (5, 400), (33, 1296)])
def test_silu_mul(cuda, rows, cols, dtype):
    case("silu", rows, cols, dtype)
    both = values(np.random.default_rng(rows + cols), (rows, 2 * cols), dtype)
    got = fp8.silu_mul(both[:, :cols], both[:, cols:])
    near_codes(got, *F.quotients(F.silu_mul(f64(both[:, :cols]), f64(both[:, cols:]))), 8 * 2.0 ** -24)


def test_silu_mul_of_rare_values(cuda):
    case("silu rare")
    g = torch.tensor([[0.0, -200.0, 200.0, -60000.0] * 32, [float("inf")] + [1.0] * 127, [-float("inf")] + [1.0] * 127], device="cuda")
    got = fp8.silu_mul(g, torch.ones_like(g))
    assert np.array_equal(f64(got.codes[0])[:4], [0, 0, 448, 0]) and abs(float(got.scales[0]) - 200 / 448) < 1e-6
    assert torch.isnan(got.scales[1:]).all() and not f64(got.codes[1:]).any()  # inf, and -inf * 0


# ------------------------------------------------------------ products

SIZES = [(1, 16, 16), (1, 1, 128), (2, 130, 144), (1, 512, 4096), (5, 128, 640), (16, 256, 2048), (17, 129, 272), (33, 1000, 1040),
         (64, 64, 128), (65, 385, 400), (127, 257, 1152), (130, 128, 4112), (200, 300, 2064), (256, 768, 256), (300, 1, 16),
         (520, 520, 528)]


@pytest.mark.parametrize("out", [BF, HF, SF])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(cuda, m, n, k, out):
    case("matmul", m, n, k, out)
    rng = np.random.default_rng(m + n + k)
    x = fp8.quantize(values(rng, (m, k)))
    w, s = weights(rng, n, k)
    near(fp8.matmul(x, w, s, out), *F.matmul(F.rows_of(f64(x.codes), f64(x.scales)), F.weight_of(f64(w), f64(s))), k, out)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul_of_16_bit_rows(cuda, m, n, k, dtype):
    """As of the codes that quantize gives, in one call."""
    case("matmul", m, n, k, dtype)
    rng = np.random.default_rng(m + n + k)
    x = values(rng, (m, k), dtype)
    w, s = weights(rng, n, k)
    near(fp8.matmul(x, w, s), *F.matmul(F.rows_of(*F.quantize(f64(x))), F.weight_of(f64(w), f64(s))), k, dtype)


@pytest.mark.parametrize("m,n,k,given", [(1, 14336, 1040, "codes"), (8, 12290, 400, "codes"), (9, 12305, 528, "codes"),
                                         (16, 20001, 144, "codes"), (4, 9000, 11760, "values"), (3, 40, 14336, "values"),
                                         (2, 12300, 272, "values"), (1, 33, 46000, "values"), (5, 33, 46000, "codes")])
def test_matmul_of_few_rows(cuda, m, n, k, given):
    """64 weight rows to a workgroup, rows that fill what is quantized in the launch and that pass it."""
    case("few", m, n, k, given)
    rng = np.random.default_rng(n)
    x = values(rng, (m, k))
    w, s = weights(rng, n, k)
    want = F.matmul(F.rows_of(*F.quantize(f64(x))), F.weight_of(f64(w), f64(s)))
    near(fp8.matmul(fp8.quantize(x) if given == "codes" else x, w, s, BF), *want, k, BF)


@pytest.mark.parametrize("m", [1, 7, 40, 200])
def test_matmul_of_f32_rows(cuda, m):
    """The codes of f32 rows are those of quantize."""
    case("matmul f32", m)
    rng = np.random.default_rng(m)
    x = values(rng, (m, 656), SF)
    w, s = weights(rng, 200, 656)
    c = fp8.quantize(x)
    near(fp8.matmul(x, w, s), *F.matmul(F.rows_of(f64(c.codes), f64(c.scales)), F.weight_of(f64(w), f64(s))), 656, SF)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_matmul_keeps_nan_to_its_row_and_column(cuda, m):
    """A row with a value that is not finite, and a weight block with a NaN scale."""
    case("matmul nan", m)
    rng = np.random.default_rng(m)
    x = values(rng, (m, 400))
    x[m // 2, 300] = float("inf")
    w, s = weights(rng, 300, 400)
    whole = fp8.matmul(values(rng, (m, 400)), w, s)
    y = fp8.matmul(x, w, s)
    assert torch.isnan(y[m // 2]).all() and torch.isfinite(y[torch.arange(m, device="cuda") != m // 2]).all()
    s[1, 2] = float("nan")
    y = fp8.matmul(fp8.quantize(values(rng, (m, 400))), w, s, BF)
    assert torch.isnan(y[:, 128:256]).all() and torch.isfinite(y[:, :128]).all() and torch.isfinite(y[:, 256:]).all()
    assert torch.isfinite(whole).all()


@pytest.mark.parametrize("m", [1, 20, 300])
def test_matmul_keeps_nan_codes_to_their_rows_and_columns(cuda, m):
    """e4m3's NaN among the codes of the weight and of a row, the last column of K beside others."""
    case("matmul nan codes", m)
    rng = np.random.default_rng(m + 1)
    x = fp8.quantize(values(rng, (m, 400)))
    w, s = weights(rng, 300, 400)
    w.view(torch.uint8)[130, 399] = 0x7f
    x.codes.view(torch.uint8)[m - 1, 0] = 0xff
    for dtype in (BF, SF):
        nan = torch.isnan(fp8.matmul(x, w, s, dtype))
        want = torch.zeros_like(nan)
        want[:, 130], want[m - 1] = True, True
        assert torch.equal(nan, want)


@pytest.mark.parametrize("m,n,k", [(3, 50, 272), (40, 200, 528), (150, 129, 400)])
def test_matmul_layouts(cuda, m, n, k):
    """Rows and columns of wider codes, scales in either order, more dimensions; outputs beside others untouched."""
    case("matmul layouts", m, n, k)
    rng = np.random.default_rng(k)
    r = fp8.quantize(values(rng, (m + 9, k + 256)))
    w, s = weights(rng, n, k)
    part = fp8.Fp8Rows(r.codes[4:4 + m, 128:128 + k], r.scales[4:4 + m, 1:1 + -(-k // 128)])
    flat = fp8.Fp8Rows(part.codes.contiguous(), part.scales.t().contiguous().t())
    want = fp8.matmul(flat, w, s, BF)
    near(want, *F.matmul(F.rows_of(f64(flat.codes), f64(flat.scales)), F.weight_of(f64(w), f64(s))), k, BF)
    assert torch.equal(fp8.matmul(part, w, s, BF), want)
    assert torch.equal(fp8.matmul(fp8.Fp8Rows(flat.codes, flat.scales.contiguous()), w, s, BF), want)
    cube = fp8.Fp8Rows(flat.codes.view(m, 1, k), flat.scales.unflatten(0, (m, 1)))
    assert torch.equal(fp8.matmul(cube, w, s, BF), want.view(m, 1, n))
    assert torch.equal(fp8.matmul(fp8.Fp8Rows(flat.codes[0], flat.scales[0]), w, s, BF).view(1, n),
                       fp8.matmul(fp8.Fp8Rows(flat.codes[:1], flat.scales[:1]), w, s, BF))
    assert fp8.matmul(fp8.Fp8Rows(flat.codes[:0], flat.scales[:0]), w, s, BF).shape == (0, n)
    x = values(rng, (m, k + 64))
    assert torch.equal(fp8.matmul(x[:, 8:8 + k], w, s), fp8.matmul(x[:, 8:8 + k].contiguous(), w, s))


def test_matmul_writes_its_rows_alone(cuda):
    """Through the C ABI into the middle of a larger buffer, at an address that only its values align."""
    from eredu_amd import _native as n

    case("rows alone")
    rng = np.random.default_rng(11)
    for M, N, K in ((1, 33, 144), (20, 130, 272), (130, 127, 128)):
        x = fp8.quantize(values(rng, (M, K)))
        w, s = weights(rng, N, K)
        want = fp8.matmul(x, w, s, BF)
        buf = torch.full((M * N + 300,), 7.0, dtype=BF, device="cuda")
        n.check(n.lib().eq_fp8_matmul(buf.data_ptr() + 2 * 129, x.codes.data_ptr(), K, x.scales.data_ptr(), M, w.data_ptr(),
                                      s.data_ptr(), M, N, K, n.EQ_DTYPE_F8E4M3, n.EQ_DTYPE_BF16, None, 0,
                                      torch.cuda.current_stream().cuda_stream))
        assert torch.equal(buf[129:129 + M * N].view(M, N), want)
        assert (buf[:129] == 7).all() and (buf[129 + M * N:] == 7).all()


# ------------------------------------------------------------ experts

def routes_of(rng, count, experts, rows, how):
    ids = rng.integers(0, experts, count)
    if how == "sorted":
        ids = np.sort(ids)
    elif how == "one":
        ids[:] = experts - 1
    elif how == "lost":  # some without an expert or a row
        ids[rng.random(count) < 0.2] = -1
        ids[rng.random(count) < 0.1] = experts
    at = rng.integers(0, rows, count)
    if how == "lost":
        at[rng.random(count) < 0.1] = rows
        at[rng.random(count) < 0.1] = -5
    return ids, at


@pytest.mark.parametrize("how", ["any", "sorted", "one", "lost"])
@pytest.mark.parametrize("routes,experts,rows,n,k", [(1, 1, 1, 16, 16), (8, 32, 1, 130, 272), (7, 4, 3, 768, 640), (40, 5, 40, 129, 400),
                                                     (300, 128, 37, 64, 128), (515, 3, 200, 257, 528), (1500, 9, 1500, 136, 256)])
def test_grouped_matmul(cuda, routes, experts, rows, n, k, how):
    case("grouped", routes, experts, rows, n, k, how)
    rng = np.random.default_rng(routes + n)
    w, s = weights(rng, experts, n, k)
    wide = F.weight_of(f64(w), f64(s))
    ids, at = routes_of(rng, routes, experts, rows, how)
    x = values(rng, (rows, k))
    c = fp8.quantize(x)
    xd = F.rows_of(f64(c.codes), f64(c.scales))
    want = F.grouped_matmul(xd, wide, ids, at)
    near(fp8.grouped_matmul(c, w, s, ints(ids), ints(at), BF), *want, k, BF)
    near(fp8.grouped_matmul(x, w, s, ints(ids), ints(at), SF), *want, k, SF)
    if rows == routes:
        near(fp8.grouped_matmul(c, w, s, ints(ids), dtype=HF), *F.grouped_matmul(xd, wide, ids), k, HF)


def test_grouped_matmul_of_no_route(cuda):
    case("no route")
    rng = np.random.default_rng(1)
    w, s = weights(rng, 3, 40, 128)
    x = values(rng, (5, 128))
    assert fp8.grouped_matmul(x, w, s, ints([]), ints([])).shape == (0, 40)
    assert not fp8.grouped_matmul(x, w, s, ints([-1] * 200), ints([0] * 200)).any()
    assert not fp8.grouped_matmul(x, w, s, ints([-1, 3])[:2], ints([0, 0])).any()


def test_refusals_on_the_gpu(cuda):
    case("refusals")
    rng = np.random.default_rng(2)
    w, s = weights(rng, 3, 40, 128)
    x = values(rng, (5, 128))
    for call, words in ((lambda: fp8.grouped_matmul(x, w, s, ints([0, 1])), "without `rows`"),
                        (lambda: fp8.grouped_matmul(x, w, s, ints([0, 1]).long(), ints([0, 1])), "int32"),
                        (lambda: fp8.grouped_matmul(x, w, s, ints([0, 1]), ints([0])), "as long as ids"),
                        (lambda: fp8.grouped_matmul(x, w, s, ints([0, 1]).cpu(), ints([0, 1])), "current device"),
                        (lambda: fp8.matmul(x.cpu(), w[0], s[0]), "current device"),
                        (lambda: fp8.quantize(x[:, :120]), "multiple of 16"),
                        (lambda: fp8.rms_norm(x[:, :24].contiguous(), x[0, :24].contiguous(), 1e-5), "multiple of 16")):
        with pytest.raises(EreduError) as e:
            call()
        assert words in str(e.value), e.value


# ------------------------------------------------------------ streams, graphs, together

def mlp(hidden, residual, norm, gate_up, down):
    h = fp8.rms_norm(hidden, norm, 1e-5, residual)
    both = fp8.matmul(h, *gate_up, dtype=hidden.dtype)
    F2 = both.shape[-1] // 2
    return fp8.matmul(fp8.silu_mul(both[..., :F2], both[..., F2:]), *down, dtype=hidden.dtype)


def mlp_sizes(rng, dim=512, inner=1296):
    return values(rng, (dim,), BF, 0.1), weights(rng, 2 * inner, dim), weights(rng, dim, inner)


@pytest.mark.parametrize("m", [1, 12, 300])
def test_an_mlp(cuda, m):
    """Each step against the oracle's on what the step before gave."""
    case("mlp", m)
    rng = np.random.default_rng(m)
    norm, gu, down = mlp_sizes(rng)
    hidden, residual = values(rng, (m, 512)), values(rng, (m, 512))
    total = (hidden.float() + residual.float()).to(BF)
    y = mlp(hidden, residual, norm, gu, down)
    assert torch.equal(hidden, total)
    h = fp8.rms_norm(total.clone(), norm, 1e-5)
    near_codes(h, *F.quotients(F.rms_norm(f64(total), f64(norm), 1e-5)), 31 * 2.0 ** -24)
    both = fp8.matmul(h, *gu, dtype=BF)
    near(both, *F.matmul(F.rows_of(f64(h.codes), f64(h.scales)), F.weight_of(*map(f64, gu))), 512, BF)
    a = fp8.silu_mul(both[:, :1296], both[:, 1296:])
    near(y, *F.matmul(F.rows_of(f64(a.codes), f64(a.scales)), F.weight_of(*map(f64, down))), 1296, BF)


@pytest.mark.parametrize("tokens", [1, 90])
def test_routed_experts_together(cuda, tokens):
    """Two of six experts a token: up, gated activation and down products, weighted and added."""
    case("experts together", tokens)
    rng = np.random.default_rng(tokens)
    E, dim, inner = 6, 256, 208
    gu, down = weights(rng, E, 2 * inner, dim), weights(rng, E, dim, inner)
    x = values(rng, (tokens, dim))
    ids = np.stack([rng.permutation(E)[:2] for _ in range(tokens)]).reshape(-1)
    rows = np.repeat(np.arange(tokens), 2)
    c = fp8.quantize(x)
    both = fp8.grouped_matmul(c, *gu, ints(ids), ints(rows), BF)
    near(both, *F.grouped_matmul(F.rows_of(f64(c.codes), f64(c.scales)), F.weight_of(*map(f64, gu)), ids, rows), dim, BF)
    a = fp8.silu_mul(both[:, :inner], both[:, inner:])
    y = fp8.grouped_matmul(a, *down, ints(ids), dtype=SF)
    near(y, *F.grouped_matmul(F.rows_of(f64(a.codes), f64(a.scales)), F.weight_of(*map(f64, down)), ids), inner, SF)


@pytest.mark.parametrize("m", [1, 12, 300])
def test_captured(cuda, m):
    """A captured step, replayed on new inputs between eager work, and two graphs of one stream in turn."""
    case("captured", m)
    rng = np.random.default_rng(m)
    norm, gu, down = mlp_sizes(rng)
    bank, bank_scales = weights(rng, 4, 512, 512)
    ids = ints(rng.integers(0, 4, m))
    hidden, residual = values(rng, (m, 512)), values(rng, (m, 512))

    def step():
        y = mlp(hidden.clone(), residual, norm, gu, down)
        return y, fp8.grouped_matmul(y, bank, bank_scales, ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step()
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        hidden.copy_(values(rng, (m, 512)))
        ids.copy_(ints(rng.integers(0, 4, m)))
        want = step()
        for g, out in graphs[:: 1 if i % 2 else -1]:
            for t in out:
                t.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i


def test_a_capture_without_scratch_is_refused(cuda):
    """Where a stream's workspace would have to grow while it is captured, the C ABI says so and records nothing."""
    from eredu_amd import _native as n

    case("capture without scratch")
    L, rng = n.lib(), np.random.default_rng(10)
    w, s = weights(rng, 300, 1040)
    x = values(rng, (7000, 1040))
    y = torch.full((7000, 300), 3.0, dtype=BF, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y.add_(1.0)
        status = L.eq_fp8_matmul(y.data_ptr(), x.data_ptr(), 1040, None, 0, w.data_ptr(), s.data_ptr(), 7000, 300, 1040,
                                 n.EQ_DTYPE_BF16, n.EQ_DTYPE_BF16, None, 0, torch.cuda.current_stream().cuda_stream)
        said = L.eq_last_error().decode()
    assert status == 1 and "no workspace" in said
    g.replay()
    torch.cuda.synchronize()
    assert (y == 4).all()


def test_two_threads_on_one_stream(cuda):
    """What a call hands from one of its launches to the next lies in the stream's workspace, and stays its own."""
    import threading

    case("threads")
    rng = np.random.default_rng(11)
    w, s = weights(rng, 640, 2048)
    bank, bank_scales = weights(rng, 5, 256, 512)
    jobs = []
    for m in (90, 333):
        x, r = values(rng, (m, 2048)), values(rng, (m, 512))
        ids = ints(rng.integers(-1, 5, m))
        jobs.append((x, r, ids, fp8.matmul(x, w, s), fp8.grouped_matmul(r, bank, bank_scales, ids)))
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def work(x, r, ids, y, z):
        go.wait()
        for i in range(40):
            if not torch.equal(fp8.matmul(x, w, s), y) or not torch.equal(fp8.grouped_matmul(r, bank, bank_scales, ids), z):
                wrong.append(i)
                return

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_streams(cuda):
    """The same calls on two streams at once: float rows, whose codes lie in a stream's own workspace."""
    case("streams")
    rng = np.random.default_rng(9)
    w, s = weights(rng, 640, 2048)
    xs = [values(rng, (200, 2048)) for _ in range(2)]
    want = [fp8.matmul(x, w, s) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for st, x, g in zip(streams, xs, got):
            with torch.cuda.stream(st):
                g.append(fp8.matmul(x, w, s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
