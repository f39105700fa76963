"""The paged 8-bit key/value cache on the GPU (include/eredu_kv.h, through
eredu_amd.PagedKVCache) against its restatement in 64 bits (oracle/paged_oracle.py).

Tables, lengths, reference counts, codes and scale bytes are equal, codes of
rotated keys but for roundings that f32 angles' products decide the other way:
u, the largest error of x1 cos - x2 sin in f32, is 3 * 2^-24 * max|x| (two products
and a difference), so a code may differ by one, and only where the value lies that near to a tie.

Attention, from the arithmetic that the header states.  With w the softmax's
weights, A = sum w |v| and S = scale * max|q| * max_j sum_d |k_j| over what a
row sees:
  out is rounded once                         h |out|,   h = 2^-8 bf16, 2^-11 f16
  q has 16 bits of its row's largest          2 * S / 65024 * A   (a score is off by at most
                                              S / 65024, w by twice that, relatively)
  q is rotated in f32                         2 * 3 * 2^-24 * S * A
  scores and exponents in f32                 2 * (|score| + 16) * 2^-23 * A
  probabilities in f16                        2^-11 * A
  sums in f32 over n tokens                   (n + D) * 2^-24 * A + n * 2^-30 * max A (f16's smallest values)
"""
import math

import numpy as np
import pytest
import torch

from eredu_amd import EreduError, PagedKVCache, rope_table
from eredu_amd.decode import llama3_rope_freqs
from oracle.paged_oracle import Paged

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def offsets(counts):
    return ints(np.concatenate(([0], np.cumsum(counts))))


def f64(t):
    return t.detach().double().cpu().numpy()


def values(rng, shape, dtype, spread=1.0):
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[-1]))
    return torch.from_numpy(x).to(dtype).cuda()


class Both:
    """A cache on the GPU and its restatement, driven together."""

    def __init__(self, layers=1, pages=24, heads=2, D=128, seqs=6, width=6, T=16, seed=0):
        self.dev = PagedKVCache(layers, pages, heads, D, seqs, width, page_size=T)
        self.ref = Paged(layers, pages, heads, D, seqs, width, T)
        self.rng = np.random.default_rng(seed)
        self.rope = rope_table(llama3_rope_freqs(D, 10000.0), width * T)

    def scramble(self):
        """Old bytes in every page, as pages that were used before have them."""
        for t, r in ((self.dev.k_codes, self.ref.k), (self.dev.v_codes, self.ref.v)):
            r[...] = self.rng.integers(-127, 128, r.shape)
            t.copy_(torch.from_numpy(r).to(torch.int8))
        for t, r in ((self.dev.k_scales, self.ref.ks), (self.dev.v_scales, self.ref.vs)):
            r[...] = self.rng.choice([1, 100, 140, 255], r.shape)
            t.copy_(torch.from_numpy(r).to(torch.uint8))

    def extend(self, seqs, counts):
        same = len(set(counts)) == 1
        self.dev.extend(ints(seqs), counts[0] if same else offsets(counts))
        self.ref.extend(seqs, counts)

    def append(self, seqs, counts, dtype=torch.bfloat16, rope=False, layer=0, spread=1.0, k=None, v=None):
        n = sum(counts)
        k = values(self.rng, (n, self.ref.heads, self.ref.D), dtype, spread) if k is None else k
        v = values(self.rng, (n, self.ref.heads, self.ref.D), dtype, spread) if v is None else v
        self.dev.append(layer, k, v, ints(seqs), offsets(counts) if len(set(counts)) > 1 else None,
                        rope=self.rope if rope else None)
        self.ref.append(layer, f64(k), f64(v), seqs, counts, f64(self.rope) if rope else None)
        return k, v

    def same_tables(self):
        for t, r in ((self.dev.tables, self.ref.tables), (self.dev.lengths, self.ref.lengths), (self.dev.refs, self.ref.refs)):
            assert np.array_equal(t.cpu().numpy(), r), (t.cpu().numpy(), r)
        assert int(self.dev.missing.item()) == self.ref.missing

    def same_codes(self, rotated=False):
        for t, r in ((self.dev.k_scales, self.ref.ks), (self.dev.v_scales, self.ref.vs), (self.dev.v_codes, self.ref.v)):
            assert np.array_equal(t.cpu().numpy(), r)
        d = np.abs(self.dev.k_codes.cpu().numpy().astype(np.int64) - self.ref.k)
        assert d.max() <= (1 if rotated else 0)
        # |x1 cos - x2 sin| <= 127 sqrt(2) steps: an error of 3 * 2^-24 * 180 steps on either side of a tie
        # is met by 6e-5 of evenly spread values; ten times that, and three for few values, is no chance
        assert (d > 0).sum() <= 6e-4 * d.size + 3
        self.ref.k[...] = self.dev.k_codes.cpu().numpy()

    def attend(self, seqs, counts, heads, dtype=torch.bfloat16, rope=False, layer=0, q=None, spread=0.7, **kw):
        n, D = sum(counts), self.ref.D
        q = values(self.rng, (n, heads, D), dtype, spread) if q is None else q
        got = self.dev.attention(layer, q, ints(seqs), offsets(counts) if len(set(counts)) > 1 else None,
                                 rope=self.rope if rope else None, **kw)
        assert got.shape == (n, heads, D) and got.dtype == dtype
        self.check_attention(f64(got), f64(q), seqs, counts, dtype, rope, layer, **kw)
        return got

    def check_attention(self, got, q, seqs, counts, dtype, rope=False, layer=0, scale=None, causal=True, window=0):
        D = self.ref.D
        ref, A, S, top = self.ref.attention(layer, q, seqs, counts, D ** -0.5 if scale is None else scale, causal,
                                            window, f64(self.rope) if rope else None)
        n = int(max(self.ref.lengths.max(), 1))
        fine = np.isfinite(ref)
        assert np.array_equal(fine, np.isfinite(got))
        rel = 2 * S / 65024 + 6 * 2.0 ** -24 * S + 2 * (top + 16) * 2.0 ** -23 + 2.0 ** -11 + (n + D) * 2.0 ** -24
        bound = HALF[dtype] * np.abs(ref) + rel * A + n * 2.0 ** -30 * np.nanmax(A) + 2.0 ** -24 * (A > 0)
        far = np.abs(got - ref)[fine] / np.maximum(bound[fine], 1e-300)
        far = np.where(np.abs(got - ref)[fine] == 0, 0, far)
        print(f"[far] {far.max() if far.size else 0:.3f} of the bound", flush=True)
        assert not far.size or far.max() <= 1


# ------------------------------------------------------------ tokens

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D,heads", [(16, 64, 3), (32, 128, 2), (64, 128, 1), (128, 256, 1), (16, 256, 2), (128, 64, 2)])
def test_append_and_read(cuda, T, D, heads, dtype):
    print(f"[case] append T={T} D={D} heads={heads} {dtype}", flush=True)
    b = Both(heads=heads, D=D, T=T, pages=30, width=5, seed=T + D)
    b.scramble()
    for counts in ([1, 1, 1], [T - 1, T, T + 1], [1, 1, 1], [2, 5, 1], [1, 2 * T + 3, T // 2]):
        b.extend([4, 0, 2], counts)
        b.append([4, 0, 2], counts, dtype, rope=True, spread=1.5)
        b.same_tables()
        b.same_codes(rotated=True)
    lens = [int(b.ref.lengths[s]) for s in (4, 0, 2)]
    for out in (torch.bfloat16, torch.float32):
        k, v = b.dev.read(0, ints([4, 0, 2]), offsets(lens), total=sum(lens), dtype=out)
        rk, rv = b.ref.read(0, [4, 0, 2], lens)
        assert np.array_equal(f64(k), rk, equal_nan=True) and np.array_equal(f64(v), rv, equal_nan=True)
    k, v = b.dev.read(0, ints([0]), 1)
    rk, rv = b.ref.read(0, [0], [1])
    assert np.array_equal(f64(k), rk) and np.array_equal(f64(v), rv)


def test_scales_grow_token_by_token(cuda):
    """A page whose values double with every token, one that shrinks, zeros,
    f16's smallest and largest, and values that are exactly 127 steps."""
    b = Both(T=16, D=64, heads=1, seqs=4, width=2, pages=8)
    b.scramble()
    for i in range(20):
        b.extend([0, 1, 2, 3], [1] * 4)
        rows = np.zeros((4, 1, 64))
        rows[0] = np.linspace(-1, 1, 64) * 2.0 ** i
        rows[1] = np.linspace(-1, 1, 64) * 2.0 ** -i
        rows[2] = 0 if i < 3 else 2.0 ** -24 * (i % 5)
        rows[3] = 127 * 2.0 ** (i % 3) / 128
        x = torch.from_numpy(rows).half().cuda()
        b.append([0, 1, 2, 3], [1] * 4, torch.float16, k=x, v=x.flip(2).contiguous())
        b.same_codes()
    # however often a scale grew, a value is off by less than a step of the last one
    k, _ = b.dev.read(0, ints([0]), 16, dtype=torch.float32)
    want = np.array([np.linspace(-1, 1, 64) * 2.0 ** i for i in range(4, 20)])
    want = torch.from_numpy(want).half().double().numpy()
    byte = f64(b.dev.k_scales)[0][b.ref.tables[0][(np.arange(4, 20) // 16)], 0]
    lost = byte == 255  # from 2^16 on the values are f16's infinities, and their page NaN
    assert lost.tolist() == [False] * 12 + [True] * 4 and np.isnan(f64(k)[lost]).all()
    assert (np.abs(f64(k)[:, 0] - want)[~lost] < 2.0 ** (byte[~lost, None] - 127)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(cuda, bad):
    """They make their page of that head NaN, for the rows that see the page, and nothing else."""
    b = Both(T=16, D=64, heads=2, seqs=2, width=4)
    b.extend([0, 1], [40, 40])
    k = values(b.rng, (80, 2, 64), torch.bfloat16)
    v = values(b.rng, (80, 2, 64), torch.bfloat16)
    k[20, 0, 5] = bad
    v[45, 1, 63] = bad
    b.append([0, 1], [40, 40], k=k, v=v)
    b.same_codes()
    b.attend([0, 1], [40, 40], 4)
    b.extend([0, 1], [1, 1])
    b.append([0, 1], [1, 1])
    b.same_codes()
    got = b.attend([0, 1], [1, 1], 4)
    assert torch.isnan(got[0, :2]).all() and not torch.isnan(got[0, 2:]).any()
    assert torch.isnan(got[1, 2:]).all() and not torch.isnan(got[1, :2]).any()
    q = values(b.rng, (2, 4, 64), torch.bfloat16)
    q[0, 3, 1] = bad
    b.attend([0, 1], [1, 1], 4, q=q)
    # the page is whole again for the sequence that takes it next
    b.dev.free(ints([0, 1]))
    b.ref.free([0, 1])
    b.extend([1], [48])
    b.append([1], [48])
    b.same_codes()
    assert not torch.isnan(b.attend([1], [48], 2)).any()


def test_rows_at_strides_and_offsets(cuda):
    """q, k and v as parts of one fused projection, and at addresses that are
    not 16-byte aligned (which are copied); out given by the caller."""
    b = Both(T=32, D=128, heads=2, width=3)
    b.extend([3, 1], [20, 20])
    fused = values(b.rng, (40, (4 + 2 + 2) * 128), torch.bfloat16)
    q, k, v = fused[:, :512], fused[:, 512:768], fused[:, 768:]
    b.append([3, 1], [20, 20], k=k.unflatten(1, (2, 128)), v=v.unflatten(1, (2, 128)))
    b.same_codes()
    out = torch.full((40, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = b.dev.attention(0, q, ints([3, 1]), out=out)
    assert got.data_ptr() == out.data_ptr()
    b.check_attention(f64(out), f64(q.unflatten(1, (4, 128))), [3, 1], [20, 20], torch.bfloat16)
    odd = torch.empty(40 * 512 + 3, dtype=torch.bfloat16, device="cuda")[3:].view(40, 4, 128)
    odd.copy_(q.unflatten(1, (4, 128)))
    assert torch.equal(b.dev.attention(0, odd, ints([3, 1])), out)
    turned = q.unflatten(1, (4, 128)).permute(1, 2, 0).contiguous().permute(2, 0, 1)
    assert torch.equal(b.dev.attention(0, turned, ints([3, 1])[torch.tensor([0, 1])]), out)


# ------------------------------------------------------------ attention

GEOMETRY = [(4, 2, 128), (16, 16, 64), (12, 4, 64), (8, 1, 128), (20, 1, 256), (6, 3, 256), (40, 8, 128), (71, 1, 64)]


@pytest.mark.parametrize("heads,kv,D", GEOMETRY)
@pytest.mark.parametrize("T", [16, 64])
def test_attention_one_token(cuda, heads, kv, D, T):
    """Sequences of 1 token to a few pages, in one batch."""
    print(f"[case] decode heads={heads}/{kv} D={D} T={T}", flush=True)
    lens = [1, 2, T - 1, T, T + 1, 63, 64, 65, 130]
    b = Both(heads=kv, D=D, T=T, seqs=len(lens) + 1, width=-(-130 // T) + 1, pages=2 * sum(-(-x // T) for x in lens))
    b.scramble()
    seqs = [int(s) for s in b.rng.permutation(len(lens) + 1)[: len(lens)]]
    b.extend(seqs, lens)
    b.append(seqs, lens, rope=True)
    b.same_codes(rotated=True)
    b.attend(seqs, [1] * len(lens), heads, rope=True)
    b.attend(seqs, [1] * len(lens), heads, torch.float16, scale=0.3)


@pytest.mark.parametrize("heads,kv,D", [(4, 2, 128), (3, 3, 64), (8, 1, 256), (24, 4, 64)])
@pytest.mark.parametrize("T", [16, 32, 128])
@pytest.mark.parametrize("counts", [[5, 5, 5], [1, 33, 150], [160, 1, 7], [70, 0, 129]])
def test_attention_several_tokens(cuda, heads, kv, D, T, counts):
    print(f"[case] tokens={counts} heads={heads}/{kv} D={D} T={T}", flush=True)
    lens = [c + x for c, x in zip(counts, (3, 0, 40))]
    b = Both(heads=kv, D=D, T=T, seqs=4, width=-(-200 // T) + 1, pages=60, seed=T)
    b.scramble()
    b.extend([2, 0, 3], lens)
    b.append([2, 0, 3], lens)
    b.attend([2, 0, 3], counts, heads, rope=True)
    b.attend([2, 0, 3], counts, heads, torch.float16, window=1)
    b.attend([2, 0, 3], counts, heads, window=37)
    b.attend([2, 0, 3], counts, heads, causal=False)


@pytest.mark.parametrize("n,heads,kv,D,T,dtype", [(1000, 8, 2, 128, 64, torch.bfloat16), (4093, 4, 4, 64, 16, torch.float16),
                                                   (2050, 2, 1, 256, 128, torch.bfloat16)])
def test_attention_long(cuda, n, heads, kv, D, T, dtype):
    """One token, a few, and a chunk of a prompt after thousands; a window far behind the start."""
    b = Both(heads=kv, D=D, T=T, seqs=2, width=-(-n // T), pages=-(-n // T) + 3)
    b.extend([1], [n])
    b.append([1], [n], rope=True, spread=0.5)
    for c, kw in ((1, {}), (6, dict(window=600)), (100, {}), (300, dict(window=511))):
        b.attend([1], [c], heads, dtype, rope=True, spread=0.5, **kw)


def test_rows_that_see_nothing(cuda):
    """More rows than tokens, an empty sequence, no sequence, missing pages: zeros."""
    b = Both(T=16, D=64, heads=1, seqs=4, width=3)
    b.scramble()
    b.extend([0, 2], [20, 40])
    b.append([0, 2], [20, 40])
    b.dev.tables[2, 0] = b.ref.tables[2, 0] = -1
    b.dev.tables[2, 2] = b.ref.tables[2, 2] = 1000  # no page of this cache
    seqs, counts = [0, 1, 2, 77, -1, 0], [25, 3, 45, 2, 1, 0]
    got = b.attend(seqs, counts, 2)
    assert not got[:5].any() and not got[25:28].any() and not got[73:76].any() and got[5:25].any(-1).all()  # (a value of code 0 is 0)
    b.attend(seqs, counts, 2, causal=False)
    b.attend([1, 77], [1, 1], 3)
    k, v = b.dev.read(0, ints(seqs), offsets(counts), total=sum(counts))
    rk, rv = b.ref.read(0, seqs, counts)
    assert np.array_equal(f64(k), rk, equal_nan=True) and np.array_equal(f64(v), rv, equal_nan=True)
    b.append([1, 0, 77], [2, 30, 1])  # positions before the first token and no sequence: nothing is written there
    b.same_codes()
    b.append([2], [40])  # what has no page is dropped
    b.same_codes()


def test_offsets_that_cover_less_or_are_wrong(cuda):
    """Rows that no entry covers stay; offsets are clamped, a decreasing pair is empty."""
    b = Both(T=16, D=64, heads=1, seqs=3, width=3)
    b.extend([0, 1], [20, 20])
    b.append([0, 1], [20, 20])
    q = values(b.rng, (12, 2, 64), torch.bfloat16)
    out = torch.full((12, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    b.dev.attention(0, q, ints([0, 1]), ints([2, 5, 8]), out=out)
    assert (out[:2] == 5).all() and (out[8:] == 5).all()
    b.check_attention(f64(out[2:8]), f64(q[2:8]), [0, 1], [3, 3], torch.bfloat16)
    out.fill_(5.0)
    b.dev.attention(0, q, ints([0, 1, 0]), ints([-4, 4, 1, 1 << 30]), out=out)
    ref = b.dev.attention(0, q[:4].contiguous(), ints([0]))
    assert torch.equal(out[:1], ref[:1]) or torch.equal(out[:4], ref)
    state = b.dev.k_codes.clone()
    k = values(b.rng, (12, 1, 64), torch.bfloat16)
    b.dev.append(0, k, k, ints([2, 2]), ints([9, 3, 3]))
    assert torch.equal(state, b.dev.k_codes)
    b.dev.extend(ints([2, 2]), ints([9, 3, 3]))
    assert int(b.dev.lengths[2].item()) == 0


def test_largest_and_smallest_magnitudes(cuda):
    """Scores far beyond exp's range, pages of zeros between pages of values,
    values 2^20 apart, one token that outweighs all, all-zero queries."""
    b = Both(T=16, D=64, heads=1, seqs=1, width=20, pages=20)
    b.extend([0], [300])
    k = values(b.rng, (300, 1, 64), torch.bfloat16)
    v = values(b.rng, (300, 1, 64), torch.bfloat16)
    k[16:48] = 0
    v[32:64] = 0
    v[64:80] *= 2.0 ** 20
    v[80:96] *= 2.0 ** -18
    k[200] *= 30
    b.append([0], [300], k=k, v=v)
    q = values(b.rng, (300, 2, 64), torch.bfloat16)
    q[10] = 0
    q[290] *= 100
    q[291] = k[200, 0] * 20
    q[292] *= 2.0 ** -60
    b.attend([0], [300], 2, q=q)
    b.attend([0], [3], 2, q=q[289:292].contiguous())
    b.attend([0], [1], 2, q=q[10:11].contiguous(), causal=False)


def test_offsets_past_32_bits(cuda):
    """Pages whose codes lie beyond 4 GiB."""
    c = PagedKVCache(1, 70000, 8, 128, 2, 3, page_size=64)
    assert c.k_codes.numel() > 1 << 32
    c.refs[:69990] = 1
    seq = ints([1])
    c.extend(seq, 100)
    assert c.tables[1].tolist() == [69990, 69991, -1]
    rng = np.random.default_rng(0)
    k, v = values(rng, (100, 8, 128), torch.bfloat16), values(rng, (100, 8, 128), torch.bfloat16)
    c.append(0, k, v, seq)
    low = PagedKVCache(1, 4, 8, 128, 2, 3, page_size=64)
    low.extend(seq, 100)
    low.append(0, k, v, seq)
    for a, b in zip(c.read(0, seq, 100), low.read(0, seq, 100)):
        assert torch.equal(a, b)
    q = values(rng, (100, 32, 128), torch.bfloat16)
    assert torch.equal(c.attention(0, q, seq), low.attention(0, q, seq))
    assert torch.equal(c.attention(0, q[99:], seq), low.attention(0, q[99:], seq))
    c.refs[:69990] = 0
    c.compact()
    assert c.tables[1].tolist() == [0, 1, -1]
    assert torch.equal(c.attention(0, q[99:], seq), low.attention(0, q[99:], seq))


# ------------------------------------------------------------ pages

def test_extend_takes_the_lowest_pages_and_counts_what_is_missing(cuda):
    b = Both(T=16, D=64, heads=1, pages=7, seqs=5, width=3)
    b.dev.refs[2] = b.ref.refs[2] = 1
    b.extend([3, 0], [17, 16])
    b.same_tables()
    b.extend([0, 3], [0, 5])
    b.extend([1, 1, 4, 9, -3], [3, 20, 33, 1, 1])  # the second of sequence 1's; no such sequences; no pages
    b.same_tables()
    with pytest.raises(EreduError, match="ran out"):
        b.dev.check()
    b.ref.missing = 0
    b.dev.check()
    b.extend([4, 2], [40, 1])  # no room in the table
    b.same_tables()
    assert b.dev.free_pages() == int((b.ref.refs <= 0).sum())


@pytest.mark.parametrize("layers", [1, 3])
def test_fork_extend_free_compact(cuda, layers):
    """Shared prefixes: who copies, who keeps, what is freed, what moves."""
    b = Both(layers=layers, T=16, D=64, heads=2, pages=40, seqs=8, width=4)
    b.scramble()
    b.extend([0, 1], [40, 16])
    for layer in range(layers):
        b.append([0, 1], [40, 16], layer=layer)
    steps = [
        lambda x, i: x.fork(i([0, 0, 0, 1]), i([2, 3, 4, 5])),
        lambda x, i: x.extend(i([2, 3]), *((1,) if x is b.dev else ([1, 1],))),  # others hold the page: both copy
        lambda x, i: x.extend(i([0, 4, 5]), *((1,) if x is b.dev else ([1, 1, 1],))),  # all who hold it: the last keeps it
        lambda x, i: x.fork(i([2, 3, 2, 99, 1]), i([3, 2, 6, 7, -1])),  # a permutation; pairs that name nothing
        lambda x, i: x.fork(i([0, 1]), i([7, 7])),  # one destination twice: the last pair
        lambda x, i: x.free(i([0, 3, 3, 50, 1])),
        lambda x, i: x.compact(),
        lambda x, i: x.compact(),
        lambda x, i: x.fork(i([2]), i([2])),
        lambda x, i: x.extend(i([6, 2, 4]), *((offsets([30, 9, 17]),) if x is b.dev else ([30, 9, 17],))),
        lambda x, i: x.free(i(range(8))),
        lambda x, i: x.compact(),
    ]
    for n, step in enumerate(steps):
        print(f"[step] {n}", flush=True)
        step(b.dev, ints)
        step(b.ref, list)
        b.same_tables()
        b.same_codes()
        if n == 6:
            b.attend([2, 4, 5], [3, 3, 3], 4, layer=layers - 1)
    assert not b.ref.refs.any()


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 3000])
def test_compact_random(cuda, pages):
    rng = np.random.default_rng(pages)
    for share in (0.0, 0.02, 0.5, 0.97, 1.0):
        b = Both(T=16, D=64, heads=1, pages=pages, seqs=3, width=max(1, pages // 2), seed=pages)
        b.scramble()
        live = rng.random(pages) < share
        ids = rng.permutation(np.nonzero(live)[0])[: 3 * b.ref.width]
        b.ref.refs[...] = 0
        b.ref.tables.reshape(-1)[: len(ids)] = ids
        b.ref.refs[ids] = rng.integers(1, 5, len(ids))
        b.dev.tables.copy_(torch.from_numpy(b.ref.tables).int())
        b.dev.refs.copy_(torch.from_numpy(b.ref.refs).int())
        b.dev.compact()
        b.ref.compact()
        b.same_tables()
        b.same_codes()


def test_many_entries(cuda):
    """More entries than the planning workgroup has threads."""
    n = 1500
    b = Both(T=16, D=64, heads=1, pages=3 * n, seqs=n, width=3)
    seqs = [int(s) for s in b.rng.permutation(n)]
    counts = [int(x) for x in b.rng.integers(0, 20, n)]
    b.extend(seqs, counts)
    b.same_tables()
    b.dev.fork(ints(seqs[:700]), ints(seqs[700:1400]))
    b.ref.fork(seqs[:700], seqs[700:1400])
    b.extend(seqs, [1] * n)
    b.same_tables()
    counts = [int(x) for x in b.rng.integers(0, 3, n)]
    b.extend(seqs, counts)  # (without it the tokens before the last may lie in shared pages, which append must not write)
    b.append(seqs, counts)
    b.same_codes()
    b.attend(seqs, counts, 1)


# ------------------------------------------------------------ as they are used

def test_a_service_of_sequences(cuda):
    """Prompts come, are sampled several times, grow token by token, end and
    make room; every step's attention against the restatement."""
    b = Both(layers=2, T=16, D=64, heads=2, pages=40, seqs=8, width=6, seed=5)
    def step(seqs, counts):
        b.extend(seqs, counts)
        for layer in range(2):
            b.append(seqs, counts, rope=True, layer=layer)
            b.same_codes(rotated=True)
            b.attend(seqs, counts, 6, rope=True, layer=layer)
        b.same_tables()
    step([0, 1, 2], [37, 5, 16])
    b.dev.fork(ints([0, 0, 2]), ints([3, 4, 5]))
    b.ref.fork([0, 0, 2], [3, 4, 5])
    for i in range(13):
        step([0, 3, 4, 5, 1], [1] * 5)
    b.dev.free(ints([0, 4]))
    b.ref.free([0, 4])
    b.dev.compact()
    b.ref.compact()
    step([6, 3, 5], [50, 1, 4])
    step([3, 5, 6, 1, 2], [1] * 5)
    b.dev.check()


def test_captured_steps_cross_page_borders(cuda):
    """One graph of a whole step (extend, append, attention) decodes successive tokens
    into new pages; a second graph of the same kind and eager calls run in between,
    and every replay equals the eager step."""
    def make():
        c = PagedKVCache(1, 30, 2, 128, 4, 8, page_size=16)
        c.extend(ints([0, 1, 2]), offsets([13, 30, 5]))
        g = np.random.default_rng(1)
        k = values(g, (48, 2, 128), torch.bfloat16)
        c.append(0, k, k.flip(2).contiguous(), ints([0, 1, 2]), offsets([13, 30, 5]))
        return c
    seqs, rope = ints([2, 0, 1]), rope_table(llama3_rope_freqs(128, 10000.0), 128)
    x = [values(np.random.default_rng(2), (3, 8, 128), torch.bfloat16), values(np.random.default_rng(3), (3, 2, 128), torch.bfloat16)]
    def step(c, x):
        c.extend(seqs, 1)
        c.append(0, x[1], x[1] * 2, seqs, rope=rope)
        return c.attention(0, x[0], seqs, rope=rope)
    want, a, b = make(), make(), make()
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        saved = [t.clone() for t in (c.tables, c.lengths, c.refs, c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
        with torch.cuda.graph(g):
            outs.append(step(c, x))
        for t, s in zip((c.tables, c.lengths, c.refs, c.k_codes, c.v_codes, c.k_scales, c.v_scales), saved):
            assert torch.equal(t, s)  # a capture runs nothing
        graphs.append(g)
    for i in range(40):
        for t in x:
            t.copy_(t.roll(1, 0) * (1.01 if i % 3 else 0.97))
        ref = step(want, x)
        graphs[0].replay()
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.current_stream().wait_stream(other)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref), i
        assert torch.equal(a.tables, want.tables) and torch.equal(b.lengths, want.lengths)
    want.check()


def test_calls_on_two_streams_share_nothing(cuda):
    """Attention over one cache from two streams at once, many times."""
    c = PagedKVCache(1, 200, 4, 128, 4, 64, page_size=64)
    c.extend(ints([0, 1]), offsets([4000, 3000]))
    rng = np.random.default_rng(0)
    k, v = values(rng, (7000, 4, 128), torch.bfloat16, 0.5), values(rng, (7000, 4, 128), torch.bfloat16, 0.5)
    c.append(0, k, v, ints([0, 1]), offsets([4000, 3000]))
    qs = [values(rng, (1, 16, 128), torch.bfloat16, 0.5), values(rng, (40, 16, 128), torch.bfloat16, 0.5)]
    want = [c.attention(0, qs[i], ints([i])) for i in range(2)]
    torch.cuda.synchronize()
    streams, seqs = [torch.cuda.Stream() for _ in range(2)], [ints([0]), ints([1])]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.attention(0, qs[i], seqs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_library_workspace_for_c_callers(cuda):
    """Scratch NULL: the stream's workspace, with the results of the given one."""
    import ctypes

    from eredu_amd import _native as n

    b = Both(T=16, D=64, heads=2, pages=60, seqs=4, width=30)
    b.extend([0, 1], [450, 3])
    b.append([0, 1], [450, 3])
    q = values(b.rng, (2, 8, 64), torch.bfloat16)
    want = b.dev.attention(0, q, ints([0, 1]))
    out, s = torch.empty_like(want), ints([0, 1])
    st = torch.cuda.current_stream().cuda_stream
    n.check(n.lib().eq_kv_attention(out.data_ptr(), q.data_ptr(), 512, 8, b.dev._ref, 0, s.data_ptr(), 2, None, 2, 0.125,
                                    True, 0, None, 0, n.EQ_DTYPE_BF16, None, 0, st))
    assert torch.equal(out, want)
    n.check(n.lib().eq_kv_extend(b.dev._ref, s.data_ptr(), 2, None, 20, None, 0, st))
    b.ref.extend([0, 1], [20, 20])
    n.check(n.lib().eq_kv_fork(b.dev._ref, s.data_ptr(), ints([2, 3]).data_ptr(), 2, None, 0, st))
    b.ref.fork([0, 1], [2, 3])
    n.check(n.lib().eq_kv_compact(b.dev._ref, None, 0, st))
    b.ref.compact()
    b.same_tables()


def test_refusals(cuda):
    c = PagedKVCache(2, 8, 2, 128, 3, 2, page_size=32)
    s = ints([0])
    ok = torch.zeros((1, 2, 128), dtype=torch.bfloat16, device="cuda")
    for k, v in ((ok.float(), ok.float()), (ok, ok.half()), (ok[:, :1], ok[:, :1]), (ok, ok.expand(2, 2, 128)),
                 (ok.cpu(), ok.cpu()), (ok[..., :64], ok[..., :64])):
        with pytest.raises(EreduError):
            c.append(0, k, v, s)
    for bad in (dict(layer=2), dict(seqs=torch.tensor([0], device="cuda")), dict(seqs=torch.tensor([0], dtype=torch.int32)),
                dict(seqs=ints([0, 1])), dict(cu=ints([0])), dict(cu=ints([0, 1]).float()), dict(window=-1),
                dict(window=2, causal=False), dict(scale=math.nan), dict(q=torch.zeros((1, 3, 128), dtype=torch.bfloat16, device="cuda")),
                dict(rope=torch.zeros((63, 128), device="cuda")), dict(rope=torch.zeros((64, 64), device="cuda")),
                dict(out=torch.zeros((1, 2, 128), device="cuda"))):
        a = dict(layer=0, q=ok, seqs=s)
        a.update(bad)
        with pytest.raises(EreduError):
            c.attention(**a)
    with pytest.raises(EreduError):
        c.read(0, s, ints([0, 1]))
    with pytest.raises(EreduError):
        c.read(0, s, 1, dtype=torch.int8)
    with pytest.raises(EreduError):
        c.extend(s, -1)
    with pytest.raises(EreduError):
        c.fork(s, ints([0, 1]))
    assert c.attention(0, ok[:0], ints([])).shape == (0, 2, 128)
    assert int(c.lengths.sum().item()) == 0
