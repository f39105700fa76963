"""The boundary of the block-scaled e4m3 linears on the CPU: include/eredu_fp8.h
compiles as C, its symbols are exported and bound, and bad arguments are refused
with a message before anything is launched (addresses here are never read)."""
import os
import re
import subprocess

import pytest
import torch

from eredu_amd import EreduError, _native, fp8
from eredu_amd.build import LIB_PATH

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "eredu_fp8.h")
L = _native.lib()
P = 4096  # an address
F32, F16, BF16, U8, E4M3 = 0, 1, 2, 3, 4


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(eq_[a-z0-9_]+)\s*\(", text)))


def test_every_declared_symbol_is_exported_and_bound():
    out = subprocess.run(["nm", "-D", "--defined-only", LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert set(declared()) <= set(re.findall(r"\bT (eq_[a-z0-9_]+)", out))
    assert set(declared()) == set(_native.FP8_SIGNATURES)


def test_header_compiles_as_c():
    src = f'#include "{HEADER}"\n_Static_assert(EQ_DTYPE_F8E4M3 == {_native.EQ_DTYPE_F8E4M3}, "dtype");\nint main(void) {{ return 0; }}\n'
    res = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-x", "c", "-fsyntax-only", "-"], input=src,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def refused(status, words):
    msg = L.eq_last_error().decode()
    assert status not in (0,), "accepted"
    assert words in msg, msg


def quantize(codes=P, scales=P, ss=4, x=P, xs=128, rows=4, cols=128, dt=BF16):
    return L.eq_fp8_quantize(codes, scales, ss, x, xs, rows, cols, dt, None)


def weight(codes=P, scales=P, w=P, count=1, rows=4, cols=128, dt=BF16):
    return L.eq_fp8_quantize_weight(codes, scales, w, count, rows, cols, dt, None)


def norm(codes=P, scales=P, ss=4, hidden=P, residual=P, w=P, rows=4, dim=128, eps=1e-5, dt=BF16):
    return L.eq_fp8_rms_norm(codes, scales, ss, hidden, residual, w, rows, dim, eps, dt, None)


def silu(codes=P, scales=P, ss=4, gate=P, gs=256, up=P, us=256, rows=4, cols=128, dt=BF16):
    return L.eq_fp8_silu_mul(codes, scales, ss, gate, gs, up, us, rows, cols, dt, None)


def matmul(y=P, x=P, xs=128, sc=P, ss=4, w=P, ws=P, m=4, n=64, k=128, xd=E4M3, yd=BF16, sp=None, sn=0):
    return L.eq_fp8_matmul(y, x, xs, sc, ss, w, ws, m, n, k, xd, yd, sp, sn, None)


def grouped(y=P, x=P, xs=128, sc=P, ss=4, xr=4, w=P, ws=P, e=2, ids=P, rows=P, r=4, n=64, k=128, xd=E4M3, yd=BF16, sp=None,
            sn=0):
    return L.eq_fp8_grouped_matmul(y, x, xs, sc, ss, xr, w, ws, e, ids, rows, r, n, k, xd, yd, sp, sn, None)


@pytest.mark.parametrize("bad,words", [
    (dict(dt=U8), "dtype"), (dict(dt=E4M3), "dtype"), (dict(cols=0), "multiple of 16"), (dict(cols=120), "multiple of 16"),
    (dict(cols=1 << 22), "below 2^22"), (dict(rows=-1), "2^26"), (dict(rows=1 << 26), "2^26"),
    (dict(rows=1 << 25, cols=256, xs=256, ss=1 << 25), "2^26"), (dict(scales=None), "null"), (dict(codes=None), "null"),
    (dict(x=None), "null"), (dict(x=P + 8), "aligned"), (dict(codes=P + 4), "aligned"), (dict(xs=132), "aligned"),
    (dict(xs=112), "row stride"), (dict(xs=1 << 23), "row stride"), (dict(ss=3), "scale_stride")])
def test_quantize_refuses(bad, words):
    refused(quantize(**bad), words)


@pytest.mark.parametrize("bad,words", [
    (dict(dt=9), "dtype"), (dict(cols=8), "multiple of 16"), (dict(rows=-1), "rows"), (dict(count=-1), "count"),
    (dict(count=1 << 22), "2^22"), (dict(rows=1 << 30), "2^22"), (dict(scales=None), "null"), (dict(w=None), "null"),
    (dict(w=P + 2), "aligned")])
def test_quantize_weight_refuses(bad, words):
    refused(weight(**bad), words)


@pytest.mark.parametrize("bad,words", [
    (dict(dt=E4M3), "dtype"), (dict(dim=100), "multiple of 16"), (dict(rows=1 << 26), "2^26"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(hidden=None), "null"), (dict(w=None), "null"), (dict(codes=None), "null"),
    (dict(scales=None), "null"), (dict(residual=P + 2), "aligned"), (dict(hidden=P + 8), "aligned"), (dict(ss=1), "scale_stride")])
def test_rms_norm_refuses(bad, words):
    refused(norm(**bad), words)


@pytest.mark.parametrize("bad,words", [
    (dict(dt=E4M3), "dtype"), (dict(cols=24), "multiple of 16"), (dict(up=None), "null"), (dict(gate=None), "null"),
    (dict(us=100), "aligned"), (dict(us=120), "row stride"), (dict(gate=P + 4), "aligned"), (dict(ss=0), "scale_stride")])
def test_silu_mul_refuses(bad, words):
    refused(silu(**bad), words)


SHARED = [
    (dict(k=0), "multiple of 16"), (dict(k=136, xs=144), "multiple of 16"), (dict(k=1 << 22), "2^22"), (dict(n=-1), "2^30"),
    (dict(n=1 << 30), "2^30"), (dict(xd=U8), "codes"), (dict(xd=7), "codes"), (dict(yd=E4M3), "y must be"), (dict(y=None), "null"),
    (dict(x=None), "null"), (dict(sc=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(x=P + 8), "aligned"),
    (dict(w=P + 8), "aligned"), (dict(y=P + 1), "aligned"), (dict(ws=P + 2), "aligned"), (dict(xs=136), "aligned"),
    (dict(xs=64), "row stride"), (dict(ss=3), "scale_stride"), (dict(xd=BF16), "belong to codes")]


@pytest.mark.parametrize("bad,words", SHARED + [(dict(m=-1), "2^30"), (dict(m=1 << 30), "2^30"), (dict(m=1 << 26), "2^26"),
                                                (dict(m=1 << 25, n=1 << 20), "tiles"), (dict(m=2, n=1 << 27), "tiles"),
                                                (dict(m=1 << 21, n=1 << 20, ss=1 << 21), "tiles")])
def test_matmul_refuses(bad, words):
    refused(matmul(**bad), words)
    sizes = dict(m=4, n=64, k=128, xd=E4M3, yd=BF16)
    if set(bad) <= set(sizes) and words != "belong to codes":
        sizes.update(bad)
        refused(L.eq_fp8_matmul_scratch(*sizes.values()), words)


@pytest.mark.parametrize("bad,words", SHARED + [
    (dict(e=0), "experts"), (dict(e=4096), "experts"), (dict(ids=None), "ids"), (dict(ids=P + 2), "ids"), (dict(rows=P + 1), "ids"),
    (dict(xr=0), "x must have"), (dict(rows=None, r=5), "without `rows`"), (dict(r=-1), "2^30"), (dict(xr=-1), "2^30"),
    (dict(xr=1 << 26), "2^26"), (dict(r=1 << 26), "2^26"), (dict(xr=1 << 20, ss=1 << 20, xs=4096), "3 * 2^30"),
    (dict(sp=P + 16, sn=1 << 30, r=1000), "scratch"), (dict(sp=P, sn=16, r=1000), "scratch")])
def test_grouped_matmul_refuses(bad, words):
    refused(grouped(**bad), words)


def test_scratch_of_float_rows_must_be_enough():
    need = L.eq_fp8_matmul_scratch(1000, 64, 128, BF16, BF16)
    assert need >= 1000 * 132
    refused(matmul(m=1000, xd=BF16, sc=None, sp=P, sn=need - 1), "scratch")
    refused(matmul(m=1000, xd=BF16, sc=None, sp=P + 128, sn=need), "scratch")


def test_scratch_is_for_what_a_call_hands_on():
    """None for rows in codes where K is not split (nor for few rows of values), else codes and scales of the values, and at most
    16 parts of the result's tiles in f32 (whole tiles, of 256 x 256 or fewer), never more than a pass of them."""
    def q(m, n, k, xd=E4M3, yd=BF16):
        return L.eq_fp8_matmul_scratch(m, n, k, xd, yd)

    assert q(1, 4096, 4096) == q(16, 128256, 4096) == q(4096, 14336, 4096) == q(1, 4096, 14336, BF16) == q(4, 4096, 4096, F32) == 0
    assert q(16, 14336, 4096, BF16) == 16 * 4096 + 16 * 32 * 4
    assert 0 < q(77, 4097, 14320) <= 16 * 128 * 4224 * 4
    for m in (17, 33, 64, 100, 300, 1000, 5000):
        for n in (1, 64, 1000, 4096, 20000):
            for k in (16, 2048, 14336, 60000):
                # (256 workgroups with a tile of 256 x 256 each: 64 MiB)
                assert 0 <= q(m, n, k) <= min(16 * -(-m // 256) * -(-n // 256) * 256 * 256 * 4, 64 << 20)
                assert q(m, n, k, F16) >= m * k
    assert q(1 << 10, 1 << 18, (1 << 22) - 16) == 0  # (parts of a large result would be larger than it is worth)
    g = L.eq_fp8_grouped_matmul_scratch
    assert g(1, 128, 8, 768, 2048, BF16, BF16) == 0 and g(64, 128, 64, 768, 2048, E4M3, BF16) == 0
    assert 4096 * 8 <= g(512, 128, 4096, 768, 2048, E4M3, BF16) <= 4096 * 8 + (128 + 4096 // 32 + 2) * 16 + 512


def test_nothing_to_do_is_no_error():
    assert quantize(rows=0, codes=None, x=None, scales=None, ss=0) == 0
    assert weight(rows=0) == 0 and weight(count=0) == 0 and norm(rows=0) == 0 and silu(rows=0) == 0
    assert matmul(m=0) == 0 and matmul(n=0, w=None) == 0 and grouped(r=0, ids=None) == 0 and grouped(n=0) == 0
    assert L.eq_fp8_matmul_scratch(0, 5, 16, E4M3, F32) == 0


def cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape).to(dtype)


@pytest.mark.parametrize("call,words", [
    (lambda: fp8.quantize(cpu(2, 128).int()), "float32"),
    (lambda: fp8.quantize_weight(cpu(128)), "[..., N, K]"),
    (lambda: fp8.rms_norm(cpu(2, 64)[0, 0], cpu(64), 1e-5), "one dimension"), (lambda: fp8._rows(cpu(2)[0], "x"), "one dimension"),
    (lambda: fp8.rms_norm(cpu(2, 64), cpu(65), 1e-5), "weight"),
    (lambda: fp8.rms_norm(cpu(2, 64), cpu(64, dtype=torch.float32), 1e-5), "weight"),
    (lambda: fp8.rms_norm(cpu(64, 2).t(), cpu(64), 1e-5), "contiguous"),
    (lambda: fp8.rms_norm(cpu(2, 64), cpu(64), 1e-5, cpu(1, 64)), "residual"),
    (lambda: fp8.silu_mul(cpu(2, 64), cpu(2, 80)), "match"),
    (lambda: fp8.matmul(cpu(2, 64), cpu(8, 64), cpu(1, 1)), "float8"),
    (lambda: fp8.matmul(cpu(2, 64), cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 2, dtype=torch.float32)), "w_scales"),
    (lambda: fp8.matmul(cpu(2, 80), cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 1, dtype=torch.float32)), "80"),
    (lambda: fp8.matmul(cpu(2, 64, dtype=fp8.CODE_DTYPE), cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 1, dtype=torch.float32)), "Fp8Rows"),
    (lambda: fp8.matmul(fp8.Fp8Rows(cpu(2, 64, dtype=fp8.CODE_DTYPE), cpu(2, 2, dtype=torch.float32)),
                        cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 1, dtype=torch.float32)), "scales has shape"),
    (lambda: fp8.matmul(fp8.Fp8Rows(cpu(2, 64, dtype=fp8.CODE_DTYPE), cpu(2, 1, dtype=torch.float32)),
                        cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 1, dtype=torch.float32)), "dtype"),
    (lambda: fp8.matmul(cpu(2, 64), cpu(8, 64, dtype=fp8.CODE_DTYPE), cpu(1, 1, dtype=torch.float32), torch.int8), "dtype"),
    (lambda: fp8.grouped_matmul(cpu(1, 2, 64), cpu(3, 8, 64, dtype=fp8.CODE_DTYPE), cpu(3, 1, 1, dtype=torch.float32),
                                cpu(2, dtype=torch.int32)), "[rows, 64]"),
])
def test_python_refusals(call, words):
    """Shapes and types are looked at before the device is."""
    with pytest.raises(EreduError) as e:
        call()
    assert words in str(e.value)


def test_layouts_that_are_taken_and_copied():
    x = torch.zeros(4, 96, dtype=torch.bfloat16)
    assert fp8._rows(x[:, :64], "x").data_ptr() == x.data_ptr() and fp8._rows(x[:, :64], "x").stride(0) == 96
    assert fp8._rows(x[:, 1:65], "x").stride(0) == 64  # not 16-byte aligned
    assert fp8._rows(x.t(), "x").is_contiguous()
    assert fp8._rows(x[1:2].as_strided((1, 64), (3, 1)), "x").stride(0) == 64  # one row, any stride
    assert fp8._rows(x.expand(3, 4, 96), "x").shape == (12, 96)
    assert fp8._rows(x[:0], "x").shape == (0, 96) and fp8._rows(x[0], "x").shape == (1, 96)
