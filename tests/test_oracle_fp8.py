"""The restatement of the block-scaled e4m3 linears (oracle/fp8_oracle.py) itself: the
codes against the bit fields and torch's own conversions, closed forms of the rest."""
import numpy as np
import pytest
import torch

from oracle import fp8_oracle as F


def test_decode_is_the_format_and_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(F.decode_table(), t, equal_nan=True)
    assert F.decode(0x7e) == 448 and F.decode(0x01) == 2.0 ** -9 and F.decode(0x38) == 1.0 and np.isnan(F.decode(0xff))


def test_nearest_is_torchs_rounding():
    rng = np.random.default_rng(0)
    v = np.concatenate((rng.uniform(-448, 448, 5000), rng.standard_normal(5000) * 2.0 ** rng.integers(-14, 6, 5000)))
    table = F.decode_table()
    codes = np.sort(table[np.isfinite(table)])
    v = np.concatenate((v, codes, (codes[1:] + codes[:-1]) / 2))  # the codes themselves and every tie
    want = torch.from_numpy(v).float().to(torch.float8_e4m3fn).double().numpy()
    at_f32 = v.astype(np.float32).astype(np.float64)
    assert np.array_equal(F.nearest(at_f32), want)


@pytest.mark.parametrize("shape", [(1, 16), (3, 128), (2, 144), (5, 400)])
def test_quantize_spans_the_range_and_comes_back(shape):
    rng = np.random.default_rng(1)
    x = rng.standard_normal(shape)
    c, s = F.quantize(x)
    for b in range(s.shape[1]):
        assert np.all(np.abs(c[:, 128 * b:128 * b + 128]).max(-1) == 448)
    back = F.rows_of(c, s)
    # half a step of 2^-4 relative, and of 2^-9 of a scale below the normal codes
    assert np.all(np.abs(back - x) <= 2.0 ** -4 * np.abs(x) + F.spread(s, shape[1], -1) * 2.0 ** -10 + 1e-7)


def test_groups_of_zeros_small_and_unfinite_values():
    x = np.zeros((1, 512))
    x[0, 128:256] = 1e-40
    x[0, 300] = np.inf
    x[0, 400] = np.nan
    c, s = F.quantize(x)
    assert s[0, 0] == 2.0 ** -126 and s[0, 1] == 2.0 ** -126 and np.isnan(s[0, 2]) and np.isnan(s[0, 3])
    assert np.all(c[0, :128] == 0) and np.all(c[0, 256:] == 0) and np.allclose(c[0, 128:256] * s[0, 1], 1e-40, rtol=2.0 ** -4)


def test_weights_have_square_blocks():
    rng = np.random.default_rng(2)
    w = rng.standard_normal((2, 130, 272))
    c, s = F.quantize_weight(w)
    assert s.shape == (2, 2, 3)
    assert np.abs(c[1, :128, 128:256]).max() == 448 and np.abs(c[0, 128:, 256:]).max() == 448
    assert np.abs(F.weight_of(c, s) - w).max() <= 2.0 ** -4 * np.abs(w).max()


def test_products_and_routes():
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((4, 32)), rng.standard_normal((3, 5, 32))
    y, size, eights = F.grouped_matmul(x, w, [2, -1, 0, 3, 1], [3, 0, 0, 1, 9])
    assert np.allclose(y[0], w[2] @ x[3]) and np.allclose(y[2], w[0] @ x[0])
    assert not y[[1, 3, 4]].any()
    p = np.abs(x[3] * w[2, 1])
    assert np.isclose(size[0, 1], p.sum()) and np.isclose(eights[0, 1], p.reshape(4, 8).max(1).sum())


def test_norm_and_silu_closed_forms():
    assert np.allclose(F.rms_norm(np.full((1, 8), 3.0), np.arange(8.0), 0.0), np.arange(8.0))
    assert np.allclose(F.silu_mul(np.array([0.0, 50.0, -800.0]), np.array([2.0, 2.0, 2.0])), [0, 100, 0])
