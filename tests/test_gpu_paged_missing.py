"""Pages that a paged cache had none for are counted whatever their number."""
import pytest
import torch

from eredu_amd import EreduError, PagedKVCache
from tests.test_gpu_paged import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 300])  # an entry a thread, and the kernel of many entries
def test_more_pages_than_an_int_counts(cuda, n):
    print(f"[case] missing n={n}", flush=True)
    c = PagedKVCache(1, 2, 1, 64, n + 1, 2, page_size=16)
    c.extend(ints([n]), 32)  # no page is left
    c.check()
    c.extend(ints(range(64)), 2 ** 30 if n == 64 else 5)  # 64 * 2^26 = 2^32 pages
    if n > 64:
        with pytest.raises(EreduError, match=": 64 could"):
            c.check()
        c.extend(ints(list(range(64)) + [-1] * (n - 64)), 2 ** 30 - 16)  # 2^26 - 1 each: the first is there, as a missing one
        assert int(c.missing.item()) == 2 ** 31 - 1
    with pytest.raises(EreduError, match=": 2147483647 could"):
        c.check()
    c.check()
    c.free(ints([n]))
    c.extend(ints([n]), 40)  # two pages and one that is not to be had
    with pytest.raises(EreduError, match=": 1 could"):
        c.check()
    c.missing.fill_(2 ** 31 - 2)
    c.extend(ints([n]), 48)
    assert int(c.missing.item()) == 2 ** 31 - 1
