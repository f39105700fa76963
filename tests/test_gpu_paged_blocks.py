"""Attention over the paged cache with many rows a sequence: blocks that are
split over their tokens beside blocks that are not, sequences of very different
lengths in one call, more of them than lanes, windows and cross attention at
every head dimension."""
import pytest
import torch

from tests.test_gpu_paged import Both

pytestmark = pytest.mark.gpu

CASES = [  # dim, heads, KV heads, page, tokens held, rows of the call, causal, window
    (64, 16, 16, 16, [300, 700, 1300], [300, 700, 1300], True, 0),
    (64, 6, 2, 128, [1300, 64, 2100], [700, 64, 90], True, 0),
    (64, 20, 20, 32, [1500, 40, 2000], [100, 1, 250], False, 0),
    (128, 8, 2, 64, [1100, 90, 513], [1100, 90, 513], True, 0),
    (128, 5, 1, 16, [2500, 1000], [600, 1000], True, 200),
    (128, 4, 4, 64, [65, 0, 1030, 64], [65, 0, 130, 64], True, 1),
    (128, 4, 2, 32, [40 + i for i in range(70)], [40 + i for i in range(70)], True, 0),
    (128, 4, 2, 32, [40 + i for i in range(64)], [35 + i for i in range(64)], True, 0),
    (256, 8, 4, 64, [1100, 33, 700], [700, 33, 700], True, 0),
    (256, 4, 4, 128, [1500, 200], [140, 150], False, 0),
    (256, 3, 1, 16, [900], [500], True, 77),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4]) + f"-n{len(c[4])}-w{c[7]}")
def test_blocks(cuda, case, dtype):
    D, heads, kv, T, held, rows, causal, window = case
    print(f"[case] {case} {dtype}", flush=True)
    n = len(held)
    b = Both(heads=kv, D=D, T=T, seqs=n, width=-(-max(held) // T), pages=sum(-(-x // T) for x in held), seed=D + n)
    b.extend(list(range(n)), held)
    b.append(list(range(n)), held, dtype=dtype, rope=causal)
    b.same_codes(rotated=causal)
    order = [int(i) for i in b.rng.permutation(n)]
    b.attend(order, [rows[i] for i in order], heads, dtype=dtype, rope=causal, causal=causal, window=window)
    # the same rows one sequence at a time, each in a call of its own
    for i in order[:3]:
        if rows[i]:
            b.attend([i], [rows[i]], heads, dtype=dtype, rope=causal, causal=causal, window=window)


def test_wide_tables(cuda):
    """A table of 8192 tokens a sequence, of which short prompts use little: splits without a tile."""
    b = Both(heads=2, D=128, T=64, seqs=4, width=128, pages=64, seed=9)
    held = [1, 130, 700, 1030]
    b.extend([0, 1, 2, 3], held)
    b.append([0, 1, 2, 3], held, rope=True)
    b.same_codes(rotated=True)
    b.attend([3, 0, 2, 1], [1030, 1, 700, 130], 4, rope=True)
    b.attend([2], [600], 4, rope=True)
    b.attend([1, 0], [40, 1], 4, rope=True)
