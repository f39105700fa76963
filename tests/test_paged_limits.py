"""How large a call of the paged cache may be: what the entry points refuse their scratch
queries refuse too, and what those accept is within a grid's 2^32 threads (on the CPU:
every call here is one that is refused before anything is launched)."""
import ctypes

import pytest

from eredu_amd import _native
from tests.test_paged_boundary import L, attend, cache, refused


def scratch(c, heads, n, total, ragged=False):
    return L.eq_kv_attention_scratch(ctypes.byref(c), heads, n, total, ragged)


TOO_MANY = [  # head_dim, heads, KV heads, sequences, rows
    (128, 32, 8, 1, 1 << 24), (64, 4, 4, 4, 1 << 26), (256, 8, 8, 2, 1 << 24), (128, 32, 8, 1 << 16, 1 << 24),
    (128, 127, 127, 4, (1 << 24) - 4),   # 128 rows to a workgroup of 256 threads: 2^23.99 workgroups ..
    (256, 65, 65, 1, (1 << 24) - 128),   # .. and of 512 threads: over 2^23
    (256, 127, 127, 1, (1 << 24) - 128),
]


@pytest.mark.parametrize("D,heads,kv,n,total", TOO_MANY)
def test_the_query_refuses_what_the_call_refuses(D, heads, kv, n, total):
    c = cache(head_dim=D, kv_heads=kv)
    fits = D == 128 and total < 1 << 24
    if fits:
        assert scratch(c, heads, n, total) >= 0
        return
    refused(scratch(c, heads, n, total), "too many rows")
    refused(attend(c, heads=heads, qs=heads * D, n=n, total=total), "too many rows")
    refused(scratch(c, heads, n, total, True), "too many rows")
    refused(attend(c, heads=heads, qs=heads * D, n=n, total=total, cu=4096), "too many rows")


@pytest.mark.parametrize("D,heads,kv,n,total", [(128, 32, 8, 1, (1 << 24) - 1), (256, 63, 63, 1, (1 << 24) - 128), (64, 8, 2, 0, 0),
                                                (128, 4, 1, 1 << 16, 1 << 16)])
def test_sizes_within(D, heads, kv, n, total):
    c = cache(head_dim=D, kv_heads=kv)
    assert scratch(c, heads, n, total) >= 0 and scratch(c, heads, n, total, True) >= 0


@pytest.mark.parametrize("bad,words", [(dict(heads=7), ["multiple"]), (dict(n=(1 << 16) + 1, total=1 << 17), ["n <="]),
                                       (dict(total=1 << 29, n=1), ["2^31"]), (dict(n=-1), ["n <="]), (dict(total=-2), ["total"]),
                                       (dict(n=0, total=3), ["total"]), (dict(total=3), ["divide"])])
def test_other_refusals(bad, words):
    a = dict(heads=8, n=2, total=2)
    a.update(bad)
    refused(attend(**a), *words)
    refused(scratch(cache(), a["heads"], a["n"], a["total"]), *words)


@pytest.mark.parametrize("D,heads,kv,n,each", [(128, 32, 8, 1, 1), (256, 32, 8, 4, 1), (128, 32, 8, 48, 1), (64, 16, 16, 16, 5),
                                               (128, 8, 8, 3, 1), (128, 32, 8, 2, 4), (256, 16, 1, 1, 1), (128, 32, 8, 2, 12)])
def test_a_decode_step_takes_scratch_for_the_rows_it_has(D, heads, kv, n, each):
    """Two slots for each of 2048 waves (of 256 CUs, as where there is no GPU to ask), of the rows that a sequence and
    KV head have, up to 16."""
    c = cache(head_dim=D, kv_heads=kv, width=512)
    rows = min(16, each * heads // kv)
    assert 0 < scratch(c, heads, n, n * each) <= 2 * 2048 * rows * (D + 1) * 4 + 256
    assert scratch(c, heads, n, n * each, True) <= 2 * 2048 * min(16, n * each * heads // kv) * (D + 1) * 4 + 256


def test_scratch_of_calls_of_few_rows():
    """What eager calls of up to 8192 rows and heads keep in their stream's workspace."""
    most = 0
    for D in (64, 128, 256):
        for heads, kv in ((1, 1), (8, 2), (32, 8), (32, 32), (64, 1)):
            for n in (1, 2, 7, 48, 512):
                for each in (1, 2, 5, 13, 33, 64, 128, 300, 8192):
                    if n * each * heads <= 8192:
                        most = max(most, *(scratch(cache(head_dim=D, kv_heads=kv, width=2048), heads, n, n * each, r) for r in (False, True)))
    assert 32 << 20 < most <= 65 << 20
