"""The restatement of the paged 8-bit cache against what its rules mean: every
sequence reads back its own tokens whatever happens to the pages, reference counts
are the tables' entries, codes are the nearest ones, attention is a dense softmax."""
import numpy as np
import pytest
import torch

from oracle.paged_oracle import Paged


def counted(p):
    ids = p.tables[p.tables >= 0]
    return np.array_equal(np.bincount(ids, minlength=len(p.refs)), p.refs)


def test_sequences_keep_their_tokens_whatever_the_pages_do():
    """Whole numbers up to 127 are stored exactly, so each sequence's tokens can be kept beside it."""
    rng = np.random.default_rng(0)
    T, D, S = 4, 8, 6
    p = Paged(2, 60, 2, D, S, 8, T)
    held = [np.zeros((0, 2, D)) for _ in range(S)]
    for step in range(300):
        op = rng.integers(0, 6)
        s = [int(x) for x in rng.permutation(S)[: rng.integers(1, S)]]
        if op <= 2:
            n = [int(min(x, 8 * T - len(held[i]))) for i, x in zip(s, rng.integers(0, 6, len(s)))]
            need = sum(-(-(len(held[i]) + c) // T) - len(held[i]) // T for i, c in zip(s, n))
            if need > (p.refs == 0).sum():
                continue
            new = rng.integers(-127, 128, (sum(n), 2, D)).astype(float)
            new[..., 0] = 127  # every page's step is 1
            p.extend(s, n)
            for layer in range(2):
                p.append(layer, new, -new, s, n)
            at = 0
            for i, c in zip(s, n):
                held[i] = np.concatenate((held[i], new[at : at + c]))
                at += c
        elif op == 3 and len(s) > 1:
            p.fork(s[:1] * (len(s) - 1), s[1:])
            for d in s[1:]:
                held[d] = held[s[0]]
        elif op == 4:
            n = [int(x) for x in rng.integers(0, 7, len(s))]
            p.shrink(s, n)
            for i, c in zip(s, n):
                held[i] = held[i][: max(len(held[i]) - c, 0)]
        else:
            p.free(s[:1])
            held[s[0]] = held[s[0]][:0]
            p.compact()
            live = int((p.refs > 0).sum())
            assert (p.refs[:live] > 0).all()
        assert counted(p) and p.missing == 0
        assert [int(x) for x in p.lengths] == [len(h) for h in held]
        for layer in range(2):
            k, v = p.read(layer, list(range(S)), [len(h) for h in held])
            want = np.concatenate(held)
            assert np.array_equal(k, want) and np.array_equal(v, -want), step


@pytest.mark.parametrize("size", [1e-30, 1.0, 3e4])
def test_codes_are_the_nearest_of_the_smallest_step(size):
    rng = np.random.default_rng(1)
    p = Paged(1, 2, 1, 64, 1, 2, 16)
    x = rng.standard_normal((16, 1, 64)) * size
    p.extend([0], [16])
    p.append(0, x, x, [0], [16])
    step = 2.0 ** (int(p.ks[0, 0, 0]) - 127)
    k, v = p.read(0, [0], [16])
    assert np.abs(k - x).max() <= step / 2 and np.array_equal(k, v)
    assert np.abs(x).max() <= 127 * step and np.abs(x).max() > 127 * step / 2
    y = 5 * x[:7]  # the step grows: old codes round once more, by less than half of the new one each time
    p.extend([0], [7])
    p.append(0, y, y, [0], [7])
    k, _ = p.read(0, [0], [23])
    assert np.abs(k[:16] - x).max() <= step / 2 and np.abs(k[16:] - y).max() <= 2.0 ** (int(p.ks[0, 1, 0]) - 128)


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 5), (True, 1), (False, 0)])
def test_attention_is_a_dense_softmax(causal, window):
    rng = np.random.default_rng(2)
    T, D, H, kv, n, c = 16, 64, 6, 2, 37, 9
    p = Paged(1, 4, kv, D, 2, 4, T)
    x = rng.standard_normal((n, kv, D))
    p.extend([1], [n])
    p.append(0, x, x[::-1].copy(), [1], [n])
    k, v = (torch.from_numpy(a).transpose(0, 1).repeat_interleave(H // kv, 0) for a in p.read(0, [1], [n]))
    q = rng.standard_normal((c, H, D))
    i, j = torch.arange(n - c, n)[:, None], torch.arange(n)[None]
    mask = (j <= i) & (j > i - window if window else j >= 0) if causal else torch.ones(c, n, dtype=torch.bool)
    s = torch.where(mask, torch.from_numpy(q).transpose(0, 1) @ k.transpose(1, 2).contiguous() * 0.125, -torch.inf)
    want = (torch.softmax(s, -1) @ v).transpose(0, 1).numpy()
    out, mag, unit, top = p.attention(0, q, [1], [c], 0.125, causal, window)
    assert np.abs(out - want).max() < 1e-13  # (37 products and sums of magnitude below 10 in 64 bits)
    assert (mag >= np.abs(out) - 1e-13).all() and (unit > 0).all() and (top > 0).all()


def test_rotation_is_a_complex_product():
    rng = np.random.default_rng(3)
    x, a = rng.standard_normal(64), rng.uniform(-9, 9, 32)
    z = (x[:32] + 1j * x[32:]) * np.exp(1j * a)
    got = Paged.turn(x, np.concatenate((np.cos(a), np.sin(a))))
    assert np.abs(got - np.concatenate((z.real, z.imag))).max() < 1e-14


def test_rows_that_see_nothing_are_zeros():
    p = Paged(1, 2, 1, 64, 1, 2, 16)
    p.extend([0], [2])
    x = np.ones((2, 1, 64))
    p.append(0, x, x, [0], [2])
    out, *_ = p.attention(0, np.ones((5, 1, 64)), [0, 7], [4, 1], 1.0)
    assert not out[:2].any() and (out[2:4] == 1).all() and not out[4].any()
