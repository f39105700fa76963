"""Calls over the paged cache that its rules allow and that ordinary use makes
seldom: the same sequence twice, tokens taken back, results over their own
queries, captured prompts, side streams, and softmaxes of very unequal weights."""
import numpy as np
import pytest
import torch

from eredu_amd import PagedKVCache, rope_table
from eredu_amd.decode import llama3_rope_freqs
from tests.test_gpu_paged import Both, ints, offsets, values

pytestmark = pytest.mark.gpu


def filled(held, heads=2, D=128, T=16, seed=1, **kw):
    b = Both(heads=heads, D=D, T=T, seqs=len(held) + 1, width=-(-max(held) // T) + 2,
             pages=sum(-(-x // T) for x in held) + 8, seed=seed, **kw)
    b.extend(list(range(len(held))), held)
    b.append(list(range(len(held))), held)
    b.same_codes()
    return b


@pytest.mark.parametrize("rows", [3, 90])
def test_a_sequence_named_twice_is_attended_twice(cuda, rows):
    print(f"[case] twice rows={rows}", flush=True)
    b = filled([150, 700])
    b.attend([1, 0, 1, 1], [rows, 2, rows, rows - 1], 8)
    b.attend([1, 1], [rows, rows], 8, causal=False)


@pytest.mark.parametrize("rows", [1, 40])
def test_tokens_taken_back(cuda, rows):
    """Drafts that were refused, and what comes in their place."""
    print(f"[case] back rows={rows}", flush=True)
    b = filled([150, 47, 16, 3])
    def back(seqs, counts, tokens):
        b.dev.shrink(ints(seqs), tokens)
        b.ref.shrink(seqs, counts)
        b.same_tables()
    back([0, 1], [7, 7], 7)  # inside a page, and into the one before
    b.attend([0, 1], [rows, rows], 8)
    b.extend([0, 1], [3, 30])
    b.append([0, 1], [3, 30])
    b.same_codes()
    b.attend([0, 1], [rows, rows], 8)
    back([2, 0, 9, 3, 0, -1], [0, 1, 5, 99, 34, 2], ints([0, 1, 5, 99, 34, 2]))  # nothing, all, a later entry's, none there
    b.dev.fork(ints([0]), ints([3]))
    b.ref.fork([0], [3])
    back([3], [33], ints([33]))  # shared pages: the other keeps them
    b.attend([0, 3, 1], [rows] * 3, 8)
    back([1], [0], ints([-5]))  # not fewer than none
    b.dev.free(ints([0, 1, 2, 3]))
    b.ref.free([0, 1, 2, 3])
    b.same_tables()
    assert not b.ref.refs.any()


def test_shrink_in_a_graph(cuda):
    """A captured step of drafts: five tokens come, as many as a device count says go again."""
    b = filled([40, 17], T=16)
    seqs, counts = ints([1, 0]), ints([0, 0])
    saved = [t.clone() for t in (b.dev.tables, b.dev.lengths, b.dev.refs)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.dev.extend(seqs, 5)
        b.dev.shrink(seqs, counts)
    for t, s in zip((b.dev.tables, b.dev.lengths, b.dev.refs), saved):
        assert torch.equal(t, s)
    for no in ([5, 0], [3, 4], [0, 5], [5, 5], [1, 2], [4, 5]):
        counts.copy_(ints(no))
        g.replay()
        b.ref.extend([1, 0], [5, 5])
        b.ref.shrink([1, 0], no)
        b.same_tables()


@pytest.mark.parametrize("lens,rows", [([700], [1]), ([900, 40], [1, 1]), ([700, 1500], [200, 300]), ([64] * 5, [64] * 5)])
def test_out_over_its_queries(cuda, lens, rows):
    print(f"[case] in place {lens} {rows}", flush=True)
    b = filled(lens)
    seqs, cu = ints(range(len(lens))), offsets(rows)
    q = values(b.rng, (sum(rows), 8, 128), torch.bfloat16)
    want = b.dev.attention(0, q, seqs, cu)
    got = b.dev.attention(0, q, seqs, cu, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("lens,rows", [([2100], [300]), ([300, 1200, 17], [300, 1200, 17]), ([2000] * 3, [1] * 3)])
def test_captured_prompts(cuda, lens, rows):
    """Calls of every kernel in a graph, replayed with eager calls of others between."""
    print(f"[case] captured {lens} {rows}", flush=True)
    b = filled(lens, T=64)
    seqs, cu = ints(range(len(lens))), offsets(rows)
    q = values(b.rng, (sum(rows), 8, 128), torch.bfloat16)
    b.dev.attention(0, q, seqs, cu)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = b.dev.attention(0, q, seqs, cu)
        k, v = b.dev.read(0, seqs, cu, total=sum(rows))
    for i in range(4):
        q.copy_(values(b.rng, tuple(q.shape), torch.bfloat16))
        want = b.dev.attention(0, q, seqs, cu)
        b.dev.attention(0, values(b.rng, (7, 8, 128), torch.bfloat16), seqs[:1])
        g.replay()
        rk, rv = b.dev.read(0, seqs, cu, total=sum(rows))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(k, rk) and torch.equal(v, rv), i


def test_parts_of_a_fused_projection_on_a_side_stream(cuda):
    D, heads, kv = 128, 8, 2
    rope = rope_table(llama3_rope_freqs(D, 10000.0), 30 * 16)
    rows = [130, 1, 60]
    x = values(np.random.default_rng(4), (sum(rows), (heads + 2 * kv) * D), torch.bfloat16)
    def run(q, k, v):
        c = PagedKVCache(1, 40, kv, D, 3, 30, page_size=16)
        seqs, cu = ints([2, 0, 1]), offsets(rows)
        c.extend(seqs, cu)
        c.append(0, k, v, seqs, cu, rope=rope)
        return c.attention(0, q, seqs, cu, rope=rope)
    parts = x[:, : heads * D], x[:, heads * D : (heads + kv) * D], x[:, (heads + kv) * D :]
    want = run(*(p.contiguous() for p in parts))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*parts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [1, 80])
@pytest.mark.parametrize("bits", [8, 14, 20, 26])
def test_many_small_weights_beside_a_large_one(cuda, rows, bits):
    """One key whose score is `bits` above the rest's: their weights, 2^-bits each, are f16's
    smallest normal numbers or its subnormal ones, and count all the same."""
    print(f"[case] weights rows={rows} bits={bits}", flush=True)
    n, D = 4000, 64
    b = Both(heads=1, D=D, T=64, seqs=1, width=64, pages=64, seed=bits)
    b.extend([0], [n])
    k = torch.zeros((n, 1, D), dtype=torch.bfloat16, device="cuda")
    k[1234, 0, 0] = 1.0
    v = values(b.rng, (n, 1, D), torch.bfloat16).abs()
    v[1234] = 0  # what is left is theirs alone
    b.append([0], [n], k=k, v=v)
    q = torch.zeros((rows, 1, D), dtype=torch.bfloat16, device="cuda")
    q[:, 0, 0] = 4.0 * bits
    out = b.attend([0], [rows], 1, q=q, scale=0.25 * np.log(2.0), causal=False)
    assert (out.float().abs().sum() > 0).item()
