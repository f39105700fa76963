"""Offsets out of order over the paged cache: nothing outside the call's rows is read or written."""
import pytest
import torch

from eredu_amd import PagedKVCache
from tests.test_gpu_paged import ints, values

import numpy as np

pytestmark = pytest.mark.gpu


def test_more_tiles_than_an_int_counts(cuda):
    """241 entries that each cover all 68 rows, between entries without a row whose first row
    would be the one behind the last: 241 * 17 units of 2^20 tiles, 2^32 + 2^20 in all."""
    print("[case] offsets out of order", flush=True)
    n, rows, heads, T, D = 482, 68, 4, 128, 64
    c = PagedKVCache(1, 4, 1, D, 2, 2 ** 26 // T, page_size=T)
    c.extend(ints([1]), 300)
    kv = [values(np.random.default_rng(i), (300, 1, D), torch.bfloat16) for i in (1, 2)]
    c.append(0, *kv, ints([1]))
    c.lengths[0] = 2 ** 26  # (of pages that are missing)
    cu = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    cu[0::2] = rows
    q = values(np.random.default_rng(3), (rows, heads, D), torch.bfloat16)
    out = torch.full((rows + 2, heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    c.attention(0, q, torch.zeros(n, dtype=torch.int32, device="cuda"), cu, out=out[1:-1])
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    want = c.attention(0, q, ints([1]))
    torch.cuda.synchronize()
    assert torch.isfinite(want.float()).all() and want.float().abs().sum() > 0
