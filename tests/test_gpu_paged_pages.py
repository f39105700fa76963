"""Pages of the 8-bit cache in numbers on both sides of what its planning
holds in shared memory: 256 entries, 65536 pages, 4096 pages taken at once."""
import pytest
import torch

from tests.test_gpu_paged import Both, ints

pytestmark = pytest.mark.gpu


def grow(b, seqs, counts):
    b.extend(seqs, counts)
    b.same_tables()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 300])
def test_entries(cuda, n):
    """Forks of a few prompts, and the same sequence named several times."""
    print(f"[case] entries n={n}", flush=True)
    b = Both(T=16, D=64, heads=1, pages=4 * n + 20, seqs=n + 4, width=5, seed=n)
    grow(b, [n, n + 1, n + 2], [20, 16, 9])
    src, dst = [n + i % 3 for i in range(n)], [int(s) for s in b.rng.permutation(n)]
    b.dev.fork(ints(src), ints(dst))
    b.ref.fork(src, dst)
    b.same_tables()
    grow(b, [int(s) for s in b.rng.permutation(n)], [1] * n)  # the prompts' own sequences still hold their pages
    some = [int(s) for s in b.rng.integers(-2, n + 6, n)]  # repeats, and sequences that there are not
    grow(b, some, [int(c) for c in b.rng.integers(0, 18, n)])
    grow(b, some, [1] * n)
    b.dev.free(ints(some))
    b.ref.free(some)
    b.dev.compact()
    b.ref.compact()
    b.same_tables()


def test_all_holders_of_a_page_write_at_once(cuda):
    """256 sequences that share their last page, all extended: the last entry keeps it."""
    n = 256
    b = Both(T=16, D=64, heads=1, pages=2 * n, seqs=n, width=3, seed=3)
    b.scramble()
    grow(b, [0], [5])
    b.append([0], [5])
    b.dev.fork(ints([0] * (n - 1)), ints(range(1, n)))
    b.ref.fork([0] * (n - 1), list(range(1, n)))
    order = [int(s) for s in b.rng.permutation(n)]
    grow(b, order, [1] * n)
    b.append(order, [1] * n)
    b.same_codes()


@pytest.mark.parametrize("pages", [65536, 65537])
def test_many_pages(cuda, pages):
    print(f"[case] pages={pages}", flush=True)
    b = Both(T=16, D=64, heads=1, pages=pages, seqs=5, width=6000, seed=pages)
    held = torch.from_numpy((b.rng.random(pages) < 0.8).astype("int32"))
    held[-1] = 1
    b.dev.refs.copy_(held)
    b.ref.refs[...] = held.numpy()
    grow(b, [3, 1], [16 * 4000 + 3, 16 * 97])  # over 4096 pages at once
    grow(b, [3, 1, 0], [16, 1, 16 * 500 - 1])
    b.dev.fork(ints([3]), ints([4]))
    b.ref.fork([3], [4])
    grow(b, [4, 3], [1, 1])
    grow(b, [2], [16 * 6000 + 5])  # and over the table
    held = b.ref.refs.copy()
    b.dev.free(ints([3, 4]))
    b.ref.free([3, 4])
    b.dev.compact()
    b.ref.compact()
    b.same_tables()
    assert (held > 0).sum() > (b.ref.refs > 0).sum()


@pytest.mark.parametrize("n,width", [(1, 1), (3, 341), (16, 256), (16, 257), (256, 16), (257, 15), (100, 41)])
def test_forks(cuda, n, width):
    """Permutations, repeats, pairs that name nothing and copies of oneself, on both sides of
    what one workgroup takes (256 pairs, 4096 table entries)."""
    print(f"[case] forks n={n} width={width}", flush=True)
    b = Both(T=16, D=64, heads=1, pages=700, seqs=n + 3, width=width, seed=n + width)
    start = [int(s) for s in b.rng.permutation(n + 3)[:40]]
    grow(b, start, [int(x) for x in b.rng.integers(0, min(16 * width, 200), len(start))])
    for _ in range(4):
        src = [int(s) for s in b.rng.integers(-1, n + 4, n)]
        dst = [int(s) for s in b.rng.permutation(n + 3)[:n]] if _ % 2 else [int(s) for s in b.rng.integers(-1, n + 4, n)]
        b.dev.fork(ints(src), ints(dst))
        b.ref.fork(src, dst)
        b.same_tables()
