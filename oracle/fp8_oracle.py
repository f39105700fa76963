"""64-bit restatement of the linears in e4m3 codes with block scales
(include/eredu_fp8.h), in numpy.

e4m3: sign, four exponent bits with bias 7, three mantissa bits; exponent 0 is
subnormal (steps of 2^-9), 0x7f and 0xff are NaN, the largest value is 448 and
there are no infinities (the reference's block-FP8 linears,
eredu/src/backend/mlx/nn/fp8.rs, hold their weights so).
"""
import numpy as np

BLOCK, MOST, LEAST = 128, 448.0, 2.0 ** -126


def decode_table():
    """The value of each of the 256 codes."""
    b = np.arange(256)
    sign, exp, man = b >> 7, (b >> 3) & 15, b & 7
    v = np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(sign == 1, -v, v)


_TABLE = decode_table()


def decode(codes):
    return _TABLE[np.asarray(codes, dtype=np.uint8)]


def step(v):
    """The distance of the codes around |v| (of the smaller binade at a power of two's upper side)."""
    _, e = np.frexp(v)
    return np.ldexp(1.0, np.maximum(e - 1, -6) - 3)


def nearest(v):
    """The e4m3 value next to v (|v| <= 448), ties to even."""
    s = step(v)
    return np.rint(v / s) * s


def spread(scales, n, axis):
    """Block scales repeated for the n values of `axis`."""
    return np.take(np.repeat(scales, BLOCK, axis=axis), np.arange(n), axis=axis)


def _scale(top):
    fine = np.isfinite(top)
    a = np.maximum(np.where(fine, top, MOST), MOST * LEAST)
    return fine, a, np.where(fine, a / MOST, np.nan)


def _tops(v):
    K = v.shape[-1]
    pad = np.zeros((*v.shape[:-1], -K % BLOCK))
    return np.abs(np.concatenate((v, pad), -1)).reshape(*v.shape[:-1], -1, BLOCK).max(-1)  # (NaN stays NaN)


def quotients(v):
    """(448 v / max|v| not yet rounded, scales not yet rounded) of rows v [..., K]."""
    v = np.asarray(v, dtype=np.float64)
    fine, a, s = _scale(_tops(v))
    K = v.shape[-1]
    with np.errstate(invalid="ignore"):
        q = np.where(spread(fine, K, -1), v * MOST / spread(a, K, -1), 0.0)
    return q, s


def quantize(v):
    """(values of the codes, f32 scales as f64)."""
    q, s = quotients(v)
    return nearest(q), s.astype(np.float32).astype(np.float64)


def quantize_weight(w):
    w = np.asarray(w, dtype=np.float64)
    N, K = w.shape[-2:]
    tops = _tops(w)  # [.., N, blocks]
    pad = np.zeros((*tops.shape[:-2], -N % BLOCK, tops.shape[-1]))
    tops = np.concatenate((tops, pad), -2)
    tops = tops.reshape(*tops.shape[:-2], -1, BLOCK, tops.shape[-1]).max(-2)
    fine, a, s = _scale(tops)
    wide = lambda t: spread(spread(t, N, -2), K, -1)
    q = np.where(wide(fine), w * MOST / wide(a), 0.0)
    return nearest(q), s.astype(np.float32).astype(np.float64)


def rms_norm(hidden, weight, eps):
    """hidden / sqrt(mean(hidden^2) + eps) * weight, not in codes yet."""
    x = np.asarray(hidden, dtype=np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)


def silu_mul(gate, up):
    g = np.asarray(gate, dtype=np.float64)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * np.asarray(up, dtype=np.float64)


def rows_of(codes, scales):
    return codes * spread(scales, codes.shape[-1], -1)


def weight_of(codes, scales):
    N, K = codes.shape[-2:]
    return codes * spread(spread(scales, N, -2), K, -1)


def matmul(x, w):
    """(x . w^T, sum |x| |w|, the largest |x| |w| of each 8 neighbouring columns summed): the
    result and what its roundings are measured by."""
    a, b = np.abs(x), np.abs(w)
    eights = np.zeros((len(x), len(w)))
    for k in range(0, x.shape[1], 8):
        top = np.zeros_like(eights)
        for i in range(k, min(k + 8, x.shape[1])):
            np.maximum(top, np.outer(a[:, i], b[:, i]), out=top)
        eights += top
    return x @ w.T, a @ b.T, eights


def grouped_matmul(x, w, ids, rows=None):
    ids = np.asarray(ids)
    rows = np.arange(len(ids)) if rows is None else np.asarray(rows)
    out = [np.zeros((len(ids), w.shape[1])) for _ in range(3)]
    for e in range(len(w)):
        mine = np.nonzero((ids == e) & (rows >= 0) & (rows < len(x)))[0]
        if len(mine):
            for o, r in zip(out, matmul(x[rows[mine]], w[e])):
                o[mine] = r
    return out
