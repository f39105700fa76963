"""LlamaDecoder over a paged 8-bit cache: its steps are, bit for bit, the public
calls that they stand for (extend; per layer the norms, projections, append and
attention), one captured graph decodes across page borders, and sequences
that share a prefix decode apart."""
import numpy as np
import pytest
import torch

from eredu_amd import EreduError, PagedKVCache, quantized_matmul, rope_table
from eredu_amd import decode as E
from tests.test_gpu_decode import tiny_model

pytestmark = pytest.mark.gpu

KV, LAYERS = 2, 2


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def model(cache, sequence=0, fused=None, seed=6):
    """The tiny model over `cache` (its weights depend on the seed alone)."""
    host, dense, _, _ = tiny_model(seed=seed, layers=LAYERS, n_kv=KV)
    return host, E.LlamaDecoder(dense.layers, dense.embed, dense.final_norm, dense.lm_head, n_heads=4, n_kv_heads=KV,
                                eps=1e-5, freqs=host["freqs"], max_seq=64, kv_cache=cache, sequence=sequence, fused=fused)


def fresh(pages=16, seqs=3, width=6):
    c = PagedKVCache(LAYERS, pages, KV, 128, seqs, width, page_size=16)
    return c


def prefill(c, seq, n, seed=0):
    """A prompt of n tokens, whose keys and values are made up."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.extend(ints(seq), n)
    for layer in range(LAYERS):
        k, v = (torch.randn((n, KV, 128), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        c.append(layer, k, v, ints(seq))


def by_hand(dec, host, c, seq, token):
    """One step by public calls; returns the logits."""
    lin = lambda l, x: quantized_matmul(x, l.w, l.scales, l.biases, transpose=True, group_size=l.group_size, bits=l.bits)
    rope, s = rope_table(host["freqs"], c.max_pages_per_seq * c.page_size), ints(seq)
    c.extend(s, 1)
    x, resid = E.embedding(dec.embed, ints(token)), None
    for li, L in enumerate(dec.layers):
        h = E.rms_norm(x, L.in_norm, 1e-5, resid)
        q, k, v = (lin(p, h).view(1, -1, 128) for p in (L.q, L.k, L.v))
        c.append(li, k, v, s, rope=rope)
        att = c.attention(li, q, s, rope=rope)
        h = E.rms_norm(x, L.post_norm, 1e-5, lin(L.o, att.view(1, -1)))
        resid = lin(L.down, E.silu_mul(lin(L.gate, h), lin(L.up, h)))
    return lin(dec.lm_head, E.rms_norm(x, dec.final_norm, 1e-5, resid)).view(-1)


def test_steps_are_the_calls_they_stand_for(cuda):
    a, b = fresh(), fresh()
    prefill(a, 1, 13), prefill(b, 1, 13)
    host, dec = model(a, 1, fused=False)
    dec.token.fill_(5)
    for i in range(20):  # over the borders at 16 and 32
        token = int(dec.token.item())
        dec.step_device()
        assert torch.equal(dec.logits, by_hand(dec, host, b, 1, token)), i
        assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.tables, b.tables)
        assert int(dec.token.item()) == int(dec.logits.float().argmax().item())
    a.check()


@pytest.mark.parametrize("fused", [False, True])
def test_one_graph_crosses_page_borders(cuda, fused):
    a, b = fresh(), fresh()
    prefill(a, 0, 10), prefill(b, 0, 10)
    _, dec = model(a, fused=fused)
    _, ref = model(b, fused=fused)
    assert dec.fused == fused
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        dec.step_device()  # workspaces and counters of this stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            dec.step_device()
    torch.cuda.synchronize()
    assert int(a.lengths[0].item()) == 11
    ref.step_device()
    for i in range(30):
        with torch.cuda.stream(st):
            g.replay()
        torch.cuda.synchronize()
        ref.step_device()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, ref.logits) and int(dec.token.item()) == int(ref.token.item()), i
    assert int(a.lengths[0].item()) == 41 and torch.equal(a.tables, b.tables)


def test_a_shared_prefix_decodes_apart(cuda):
    """Two continuations of one prompt equal continuations of two copies of it."""
    shared, apart = fresh(), fresh()
    prefill(shared, 0, 21)
    shared.fork(ints(0), ints(2))
    prefill(apart, 0, 21), prefill(apart, 2, 21)
    decs = {(c, s): model(c, s)[1] for c in (shared, apart) for s in (0, 2)}
    for (c, s), d in decs.items():
        d.token.fill_(3 + s)
    for _ in range(14):
        for d in decs.values():
            d.step_device()
        for s in (0, 2):
            assert torch.equal(decs[shared, s].logits, decs[apart, s].logits)
    assert int((shared.refs > 0).sum()) == 1 + 2 * 2  # the first page is still shared


def test_pages_run_out(cuda):
    c = fresh(pages=1)
    _, dec = model(c)
    for _ in range(17):
        dec.step_device()
    with pytest.raises(EreduError, match="ran out"):
        c.check()


def test_refusals(cuda):
    c = fresh()
    _, dec = model(c)
    for f in (lambda: dec.step(0), lambda: dec.set_position(0), lambda: model(c, 3), lambda: model(c, -1),
              lambda: model(PagedKVCache(LAYERS + 1, 4, KV, 128, 1, 2)), lambda: model(PagedKVCache(LAYERS, 4, 1, 128, 1, 2))):
        with pytest.raises(EreduError):
            f()
    assert dec.launches_per_step() == 1 + LAYERS * (7 if dec.fused else 10) + (4 if dec.fused else 5)
    _, dense, _, _ = tiny_model(seed=6, layers=LAYERS, n_kv=KV)
    assert dense.bytes_per_step(40) - dec.bytes_per_step(40) == LAYERS * 42 * 2 * KV * 128
