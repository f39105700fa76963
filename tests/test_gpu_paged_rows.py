"""Operands of the paged cache at layouts other than whole rows: the results are those of whole rows."""
import numpy as np
import pytest
import torch

from eredu_amd import PagedKVCache, rope_table
from eredu_amd.decode import llama3_rope_freqs
from tests.test_gpu_paged import ints, values

pytestmark = pytest.mark.gpu

HEADS, KV, D = 8, 2, 128


def run(steps, layout):
    """Tokens one by one (q, k, v [1, heads, D] each), handed over by `layout`."""
    rope = rope_table(llama3_rope_freqs(D, 10000.0), 4 * 16)
    c = PagedKVCache(1, 4, KV, D, 1, 4, page_size=16)
    seqs, out = ints([0]), []
    for q, k, v in steps:
        c.extend(seqs, 1)
        c.append(0, layout(k), layout(v), seqs, rope=rope)
        out.append(c.attention(0, layout(q), seqs, rope=rope).clone())
    return torch.cat(out), c.k_codes, c.v_codes


LAYOUTS = {
    "by_head": lambda t: t.transpose(0, 1).clone(memory_format=torch.contiguous_format).transpose(0, 1),
    "expanded": lambda t: t.as_strided(t.shape, (0, D, 1)),
    "odd_stride": lambda t: t.as_strided(t.shape, (3, D, 1)),
    "padded_heads": lambda t: torch.cat((t, t), 2)[..., :D],
    "flat": lambda t: t.reshape(1, -1),
}


@pytest.mark.parametrize("name", LAYOUTS)
def test_one_token_of_one_sequence(cuda, name):
    print(f"[case] one row {name}", flush=True)
    rng = np.random.default_rng(5)
    steps = [[values(rng, (1, h, D), torch.bfloat16) for h in (HEADS, KV, KV)] for _ in range(20)]
    want, got = run(steps, lambda t: t), run(steps, LAYOUTS[name])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
