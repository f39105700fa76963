"""Two host threads, a paged cache each, on one stream: what a call hands from one of
its launches to the next lies in the stream's workspace, and stays its own."""
import threading

import numpy as np
import pytest
import torch

from eredu_amd import PagedKVCache
from tests.test_gpu_paged import ints, offsets, values

pytestmark = pytest.mark.gpu


def filled(seed, held, pages, T=64, kv=2, D=128):
    rng = np.random.default_rng(seed)
    c = PagedKVCache(1, pages, kv, D, 2 * len(held), -(-max(held) // T) + 4, page_size=T)
    seqs, n = ints(range(len(held))), sum(held)
    c.extend(seqs, offsets(held))
    c.append(0, values(rng, (n, kv, D), torch.bfloat16), values(rng, (n, kv, D), torch.bfloat16), seqs, offsets(held))
    return c, seqs, rng


@pytest.mark.parametrize("rows", [[1, 1], [130, 130]])  # waves over runs of tiles, and blocks over splits
def test_attention(cuda, rows):
    print(f"[case] threads attention {rows}", flush=True)
    jobs = []
    for seed, held in ((1, [4100, 2900]), (2, [3500, 5000])):
        c, seqs, rng = filled(seed, held, 200)
        q = [values(rng, (sum(rows), 8, 128), torch.bfloat16) for _ in range(4)]
        jobs.append((c, seqs, q, [c.attention(0, x, seqs) for x in q]))
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def work(c, seqs, q, want):
        go.wait()
        for i in range(40):
            if not torch.equal(c.attention(0, q[i % 4], seqs), want[i % 4]):
                wrong.append(i)
                return

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_extend_copies_its_own_pages(cuda):
    print("[case] threads extend", flush=True)
    jobs = [filled(seed, held, pages) for seed, held, pages in ((3, [100, 77], 900), (4, [70, 90], 40))]
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def work(c, seqs, rng):
        twins = seqs + 2
        kept = c.read(0, seqs, 64)
        go.wait()
        for i in range(40):
            c.fork(seqs, twins)
            c.extend(twins, 1)  # copies the last page, which is shared
            c.shrink(twins, 1)
            got = c.read(0, twins, 64)
            c.free(twins)
            if not all(torch.equal(a, b) for a, b in zip(got, kept)):
                wrong.append(i)
                return
        if not all(torch.equal(a, b) for a, b in zip(c.read(0, seqs, 64), kept)):
            wrong.append(-1)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for c, _, _ in jobs:
        c.check()
