"""The paged key/value cache's boundary on the CPU: include/eredu_kv.h compiles
as C, its symbols are exported and bound, and bad arguments are refused with a
message before anything is launched (addresses here are never read)."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from eredu_amd import EreduError, PagedKVCache, _native, rope_table
from eredu_amd.build import LIB_PATH

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "eredu_kv.h")
L = _native.lib()


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(eq_[a-z0-9_]+)\s*\(", text)))


def test_every_declared_symbol_is_exported_and_bound():
    out = subprocess.run(["nm", "-D", "--defined-only", LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert set(declared()) <= set(re.findall(r"\bT (eq_[a-z0-9_]+)", out))
    assert set(declared()) == set(_native.KV_SIGNATURES)


def test_header_compiles_as_c_and_the_struct_is_the_bound_one():
    src = (f'#include "{HEADER}"\n_Static_assert(sizeof(eq_kv_cache) == {ctypes.sizeof(_native.KvCache)}, "size");\n'
           "int main(void) { return 0; }\n")
    res = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-x", "c", "-fsyntax-only", "-"], input=src,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def cache(**kw):
    a = dict(k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, tables=4096, lengths=4096, refs=4096, missing=4096,
             layers=2, pages=10, sequences=4, width=3, kv_heads=2, page_tokens=64, head_dim=128)
    a.update(kw)
    return _native.KvCache(**a)


def refused(status, *words):
    msg = L.eq_last_error().decode()
    assert status not in (0,), "accepted"
    for w in words:
        assert w in msg, msg


def append(c=None, layer=0, k=4096, v=4096, ks=256, vs=256, seqs=4096, n=2, cu=None, total=2, rope=None, rn=0, dt=2):
    return L.eq_kv_append(ctypes.byref(c or cache()), layer, k, v, ks, vs, seqs, n, cu, total, rope, rn, dt, None)


def attend(c=None, out=4096, q=4096, qs=1024, heads=8, layer=0, seqs=4096, n=2, cu=None, total=2, scale=0.1, causal=True,
           window=0, rope=None, rn=0, dt=2, ws=None, wb=0):
    return L.eq_kv_attention(out, q, qs, heads, ctypes.byref(c or cache()), layer, seqs, n, cu, total, scale, causal,
                             window, rope, rn, dt, ws, wb, None)


def read(c=None, k=4096, v=4096, layer=0, seqs=4096, n=2, cu=None, total=2, dt=2):
    return L.eq_kv_read(k, v, ctypes.byref(c or cache()), layer, seqs, n, cu, total, dt, None)


BAD_CACHES = [(dict(k_codes=None), "null"), (dict(missing=None), "null"), (dict(page_tokens=48), "page_tokens"),
              (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=256), "page_tokens"), (dict(head_dim=96), "head_dim"),
              (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "positive"), (dict(width=0), "positive"),
              (dict(width=1 << 40), "2^30"), (dict(width=1 << 20, sequences=1 << 11), "2^31"),
              (dict(pages=1 << 40), "positive"), (dict(v_codes=4104), "16-byte")]


@pytest.mark.parametrize("bad,word", BAD_CACHES)
def test_every_entry_point_refuses_a_bad_cache(bad, word):
    c = cache(**bad)
    refused(append(c), word)
    refused(attend(c), word)
    refused(read(c), word)
    r = ctypes.byref(c)
    refused(L.eq_kv_extend(r, 4096, 1, None, 1, None, 0, None), word)
    refused(L.eq_kv_fork(r, 4096, 4096, 1, None, 0, None), word)
    refused(L.eq_kv_shrink(r, 4096, 1, None, 1, None), word)
    refused(L.eq_kv_free(r, 4096, 1, None), word)
    refused(L.eq_kv_compact(r, None, 0, None), word)
    refused(L.eq_kv_pages_scratch(r, 1), word)
    refused(L.eq_kv_attention_scratch(r, 8, 1, 1, False), word)


@pytest.mark.parametrize("call", [append, attend, read])
@pytest.mark.parametrize("bad,word", [(dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(n=-1), "n <="),
                                      (dict(n=(1 << 16) + 1, total=0), "n <="), (dict(seqs=None), "null"),
                                      (dict(total=3), "divide"), (dict(total=-2), "total"), (dict(total=1 << 31), "total"),
                                      (dict(n=0, total=1), "total"), (dict(dt=9), "")])
def test_batches(call, bad, word):
    refused(call(**bad), word)


@pytest.mark.parametrize("bad,word", [(dict(k=None), "null"), (dict(v=None), "null"), (dict(k=4104), "aligned"),
                                      (dict(ks=260), "multiples of 8"), (dict(vs=128), "at least"),
                                      (dict(dt=0), "bfloat16 or float16"), (dict(rope=4096, rn=191), "cover"),
                                      (dict(rope=4100, rn=192), "aligned"), (dict(total=(1 << 30) - 1, n=1), "many")])
def test_append(bad, word):
    refused(append(**bad), word)


@pytest.mark.parametrize("bad,word", [(dict(heads=7), "multiple"), (dict(heads=0), "multiple"), (dict(heads=65536), "65535"),
                                      (dict(out=None), "aligned"), (dict(q=4104), "aligned"), (dict(qs=1028), "q_stride"),
                                      (dict(qs=512), "q_stride"), (dict(window=-1), "window"),
                                      (dict(window=5, causal=False), "window"), (dict(scale=float("nan")), "scale"),
                                      (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
                                      (dict(dt=0), "bfloat16 or float16"), (dict(rope=4096, rn=10), "cover"),
                                      (dict(total=1 << 29, n=1), "2^31")])
def test_attention(bad, word):
    refused(attend(**bad), word)


def test_pages():
    r = ctypes.byref(cache())
    refused(L.eq_kv_extend(r, None, 1, None, 1, None, 0, None), "null")
    refused(L.eq_kv_extend(r, 4096, 1, None, -1, None, 0, None), "count")
    refused(L.eq_kv_extend(r, 4096, -1, None, 1, None, 0, None), "n <=")
    refused(L.eq_kv_extend(r, 4096, 1, None, 1, 4096, 16, None), "scratch")
    refused(L.eq_kv_extend(r, 4096, 1, None, 1, 4100, 1 << 30, None), "scratch")
    refused(L.eq_kv_fork(r, 4096, None, 1, None, 0, None), "null")
    refused(L.eq_kv_fork(r, 4096, 4096, 1 << 21, None, 0, None), "n <=")
    refused(L.eq_kv_fork(r, 4096, 4096, 1, 4096, 4, None), "scratch")
    refused(L.eq_kv_shrink(r, None, 1, None, 1, None), "null")
    refused(L.eq_kv_shrink(r, 4096, 1, None, -1, None), "count")
    refused(L.eq_kv_shrink(r, 4096, 1 << 21, None, 1, None), "n <=")
    refused(L.eq_kv_free(r, None, 1, None), "null")
    refused(L.eq_kv_compact(r, 4096, 4, None), "scratch")
    refused(L.eq_kv_pages_scratch(r, -1), "n <=")


def test_empty_calls_launch_nothing():
    assert append(n=0, total=0, seqs=None, k=None, v=None) == 0
    assert attend(total=0) == 0
    assert read(total=0) == 0
    r = ctypes.byref(cache())
    assert L.eq_kv_extend(r, None, 0, None, 1, None, 0, None) == 0
    assert L.eq_kv_extend(r, 4096, 3, None, 0, None, 0, None) == 0
    assert L.eq_kv_fork(r, None, None, 0, None, 0, None) == 0
    assert L.eq_kv_shrink(r, None, 0, None, 1, None) == 0
    assert L.eq_kv_free(r, None, 0, None) == 0


def test_python_refuses_before_it_allocates_much():
    with pytest.raises(EreduError):
        PagedKVCache(1, 4, 2, 128, 2, 2, page_size=64, device="cpu")
    with pytest.raises(EreduError):
        PagedKVCache(1, 0, 2, 128, 2, 2, device="cpu")
    with pytest.raises(EreduError, match="page size"):
        PagedKVCache(1, 4, 2, 128, 2, 2, page_size=40, device="cpu")
    with pytest.raises(EreduError, match="positions|position"):
        rope_table([1.0], 0, "cpu")
    z = lambda *s, d=torch.int8: torch.zeros(s, dtype=d)
    with pytest.raises(EreduError, match="v_codes"):
        PagedKVCache.over(z(1, 2, 2, 16, 64), z(1, 2, 2, 16, 64), z(1, 2, 2, d=torch.uint8), z(1, 2, 2, d=torch.uint8),
                          z(1, 2, d=torch.int32), z(1, d=torch.int32), z(2, d=torch.int32))


def test_rope_table_is_right_at_far_positions():
    f = np.array([1.0, 10.0, 1e4])
    t = rope_table(f, 131072, "cpu").numpy()
    want = np.concatenate((np.cos(131071 / f), np.sin(131071 / f)))
    assert np.abs(t[131071] - want).max() <= 2.0 ** -24
