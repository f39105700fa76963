"""Linears in 8-bit floating point with block scales, on the HIP kernels
(``include/eredu_fp8.h``: eq_fp8_*).

Stands beside the affine and MXFP4 matmuls of :mod:`eredu_amd.quantization`, in
the place of the reference's block-FP8 projections
(eredu/src/backend/mlx/nn/fp8.rs).  A value is an e4m3 code times a float32
scale: weights [N, K] have a scale for each block of 128 x 128, activations one
for each 128 columns of a row, so both operands of a product go to the matrix
cores as they are.  An MLP over rows of 16-bit activations:

    h = fp8.rms_norm(hidden, norm, eps, residual)        # Fp8Rows
    both = fp8.matmul(h, gate_up, gate_up_scales, torch.bfloat16)
    a = fp8.silu_mul(both[:, :F], both[:, F:])           # Fp8Rows
    out = fp8.matmul(a, down, down_scales, torch.bfloat16)

A group of 128 values v gets the scale max|v| / 448 (at least 2^-126) and codes
448 v / max|v|, rounded to the nearest, ties to even (once of 16-bit values; of float32 ones the
quotient is off by up to 3 * 2^-24 of itself before); a group that holds a value that is not finite gets the scale NaN and
codes 0.  Row lengths are multiples of 16; sizes have limits, which the header names.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _native
from ._native import EreduError, check
from .quantization import _DTYPE_CODE, _get_device, _raw_stream, _stream

BLOCK = 128  # columns of a scale, and rows of a weight's
CODE_DTYPE = torch.float8_e4m3fn

# Whether the current stream is being captured (a method of torch.cuda without its wrapper).
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


class Fp8Rows(NamedTuple):
    """Rows in codes: ``codes`` [..., K] float8_e4m3fn and ``scales`` [...,
    ceil(K / 128)] float32, value = code * scale of its 128 columns.  The scales
    of a block lie side by side for all rows (the last axis has the larger stride)."""

    codes: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        wide = self.scales.repeat_interleave(BLOCK, -1)[..., :self.codes.shape[-1]]
        return (self.codes.float() * wide).to(dtype)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _here(*tensors: Optional[torch.Tensor]) -> int:
    """The current stream, once every tensor lives on the current device."""
    index = _get_device() if _get_device is not None else torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise EreduError(f"all arrays must live on the current device, cuda:{index}: got one on {t.device}")
    return _raw_stream(index) if _raw_stream is not None else _stream()


def _float_code(t: torch.Tensor, what: str) -> int:
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise EreduError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """t [..., K] as rows [M, K] whose values are contiguous, at any stride of a
    multiple of 16 bytes, as slices of a fused projection are.  Any other layout is copied."""
    d = t.dim()
    if d == 2:
        stride, one = t.stride()
        if one == 1 and t.shape[1] <= stride < 1 << 23 and stride * t.itemsize % 16 == 0 and t.data_ptr() % 16 == 0:
            return t
    elif d == 0:
        raise EreduError(f"{what} must have at least one dimension")
    K = t.shape[-1]
    if d != 2:
        t = t.reshape(-1, K) if K else t.reshape(t.numel(), 0)
    if t.is_contiguous():
        # (a single row is contiguous at any stride)
        t = t if t.stride(0) == K or t.shape[0] != 1 else t.as_strided(t.shape, (K, 1))
    elif t.stride(1) != 1 or t.stride(0) < K or t.stride(0) >= 1 << 23 or t.stride(0) * t.element_size() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _codes_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, dtype=CODE_DTYPE, memory_format=torch.contiguous_format)


def _scales_like(t: torch.Tensor, rows: int, K: int) -> torch.Tensor:
    """Scales [rows, blocks] whose rows of a block lie side by side."""
    return t.new_empty_strided((rows, -(-K // BLOCK)), (1, rows or 1), dtype=torch.float32)


def _out(codes: torch.Tensor, scales: torch.Tensor) -> Fp8Rows:
    d = codes.dim()
    return Fp8Rows(codes, scales if d == 2 else scales.unflatten(0, codes.shape[:-1]) if d > 2 else scales[0])


def quantize(x: torch.Tensor) -> Fp8Rows:
    """Codes and scales of x [..., K] (C ABI: eq_fp8_quantize)."""
    code = _float_code(x, "x")
    st = _here(x)
    x2 = _rows(x, "x")
    K = x2.shape[1]
    rows = x2.shape[0]
    codes, scales = _codes_like(x), _scales_like(x, rows, K)
    check(_native.lib().eq_fp8_quantize(codes.data_ptr(), scales.data_ptr(), rows, x2.data_ptr(), x2.stride(0), rows, K,
                                        code, st))
    return _out(codes, scales)


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes float8_e4m3fn, scales float32) of weights w [..., N, K]: a scale
    for each block of 128 x 128 (C ABI: eq_fp8_quantize_weight)."""
    code = _float_code(w, "w")
    if w.dim() < 2:
        raise EreduError("w must be [..., N, K]")
    st = _here(w)
    w = w.contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    N, K = w.shape[-2:]
    count = 1
    for d in w.shape[:-2]:
        count *= d
    codes = torch.empty(w.shape, dtype=CODE_DTYPE, device=w.device)
    scales = torch.empty((*w.shape[:-2], _blocks(N), _blocks(K)), dtype=torch.float32, device=w.device)
    check(_native.lib().eq_fp8_quantize_weight(codes.data_ptr(), scales.data_ptr(), w.data_ptr(), count, N, K, code, st))
    return codes, scales


def rms_norm(hidden: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None) -> Fp8Rows:
    """``hidden += residual`` (in place, when given), then RMSNorm(hidden) *
    weight in codes (C ABI: eq_fp8_rms_norm): ``decode.rms_norm`` for what a
    projection in codes reads next, of any of the three float types."""
    code, dtype, shape = _float_code(hidden, "hidden"), hidden.dtype, hidden.shape
    if not shape:
        raise EreduError("hidden must have at least one dimension")
    K = shape[-1]
    if weight.dtype is not dtype or weight.shape != shape[-1:] or not weight.is_contiguous():
        raise EreduError(f"weight must be a contiguous {dtype} tensor [{K}]")
    if not hidden.is_contiguous():
        raise EreduError("hidden must be contiguous")
    rp = None
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            raise EreduError("residual must match hidden in shape and dtype")
        residual = residual.contiguous()
        rp = residual.data_ptr()
    st = _here(hidden, weight, residual)
    rows = shape[0] if len(shape) == 2 else hidden.numel() // K if K else 0
    codes, scales = _codes_like(hidden), _scales_like(hidden, rows, K)
    check(_native.lib().eq_fp8_rms_norm(codes.data_ptr(), scales.data_ptr(), rows, hidden.data_ptr(), rp, weight.data_ptr(),
                                        rows, K, eps, code, st))
    return _out(codes, scales)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> Fp8Rows:
    """silu(gate) * up in codes, gate and up [..., F] (slices of one projection
    will do); nothing is rounded before the codes (C ABI: eq_fp8_silu_mul)."""
    code = _float_code(gate, "gate")
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise EreduError("gate and up must match in shape and dtype")
    st = _here(gate, up)
    g, u = _rows(gate, "gate"), _rows(up, "up")
    rows, K = g.shape
    codes, scales = _codes_like(gate), _scales_like(gate, rows, K)
    check(_native.lib().eq_fp8_silu_mul(codes.data_ptr(), scales.data_ptr(), rows, g.data_ptr(), g.stride(0),
                                        u.data_ptr(), u.stride(0), rows, K, code, st))
    return _out(codes, scales)


def _x_of(x: Union[Fp8Rows, torch.Tensor], K: int):
    """(rows, scales or None, scale stride, dtype code) of a product's left operand."""
    if isinstance(x, torch.Tensor):
        code = _DTYPE_CODE.get(x.dtype)
        if code is None:
            if x.dtype is CODE_DTYPE:
                raise EreduError("rows in codes come with their scales: pass Fp8Rows(codes, scales)")
            raise EreduError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
        rows, scales, stride = _rows(x, "x"), None, 0
    else:
        codes, scales = x
        if codes.dtype is not CODE_DTYPE or scales.dtype is not torch.float32:
            raise EreduError(f"codes must be float8_e4m3fn and scales float32, got {codes.dtype} and {scales.dtype}")
        code, rows = _native.EQ_DTYPE_F8E4M3, _rows(codes, "x")
        M, blocks = rows.shape[0], -(-rows.shape[1] // BLOCK)
        expect = (*codes.shape[:-1], blocks)
        if scales.shape != expect:
            raise EreduError(f"scales has shape {tuple(scales.shape)}, expected {expect}")
        if len(expect) != 2:
            scales = scales.reshape(-1, blocks)
        if (M > 1 and scales.stride(0) != 1) or (blocks > 1 and scales.stride(1) < M):
            scales = scales.t().contiguous().t()
        stride = scales.stride(1) if blocks > 1 else M
    if rows.shape[1] != K:
        raise EreduError(f"x has rows of {rows.shape[1]} values, the weight of {K}")
    return rows, scales, stride, code


def _weight(w: torch.Tensor, w_scales: torch.Tensor, dims: int):
    """w's shape, once it and its scales are what the products take."""
    shape, blocks = w.shape, w_scales.shape
    if len(shape) != dims or w.dtype is not CODE_DTYPE or not w.is_contiguous():
        raise EreduError(f"w must be a contiguous float8_e4m3fn tensor {'[N, K]' if dims == 2 else '[experts, N, K]'}")
    if (w_scales.dtype is not torch.float32 or len(blocks) != dims or blocks[-1] != -(-shape[-1] // BLOCK) or
            blocks[-2] != -(-shape[-2] // BLOCK) or blocks[0] != (shape[0] if dims == 3 else blocks[0]) or
            not w_scales.is_contiguous()):
        expect = (*shape[:-2], -(-shape[-2] // BLOCK), -(-shape[-1] // BLOCK))
        raise EreduError(f"w_scales must be a contiguous float32 tensor {expect}, got {w_scales.dtype} {tuple(blocks)}")
    return shape


def _out_dtype(x, dtype: Optional[torch.dtype]) -> torch.dtype:
    if dtype is None:
        if not isinstance(x, torch.Tensor):
            raise EreduError("rows in codes have no dtype of their own: say which the result has")
        return x.dtype
    if dtype not in _DTYPE_CODE:
        raise EreduError(f"the result's dtype must be float32, float16 or bfloat16, got {dtype}")
    return dtype


def _scratch(need: int, device) -> Tuple[Optional[int], int, Optional[torch.Tensor]]:
    """Scratch of a call from torch: a graph's own, so that graphs share nothing.
    (Eager calls take the library's workspace of their stream.)"""
    if need < 0:
        check(1)
    if need == 0:
        return None, 0, None
    t = torch.empty((need,), dtype=torch.uint8, device=device)
    return t.data_ptr(), need, t


def matmul(x: Union[Fp8Rows, torch.Tensor], w: torch.Tensor, w_scales: torch.Tensor,
           dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x . w^T of x [..., K] and w [N, K] in codes with w_scales [ceil(N / 128),
    ceil(K / 128)]: [..., N] in ``dtype`` (x's own where it is None).  x is
    ``Fp8Rows``, or float rows that the call quantizes first, as ``quantize``
    does (C ABI: eq_fp8_matmul).  16-bit results take the matrix cores' e4m3 products,
    which keep 13 bits below the largest of 8 (cut off, so off by up to 7 * 2^-13 of it where all 8 are of its size); float32
    results exact ones at half the rate."""
    N, K = _weight(w, w_scales, 2)
    rows, scales, stride, code = _x_of(x, K)
    dtype = _out_dtype(x, dtype)
    st = _here(rows, scales, w, w_scales)
    M, lib, out = rows.shape[0], _native.lib(), _DTYPE_CODE[dtype]
    y = rows.new_empty((M, N), dtype=dtype)
    sp, sn, hold = _scratch(lib.eq_fp8_matmul_scratch(M, N, K, code, out), rows.device) if _capturing() else (None, 0, None)
    check(lib.eq_fp8_matmul(y.data_ptr(), rows.data_ptr(), rows.stride(0), None if scales is None else scales.data_ptr(),
                            stride, w.data_ptr(), w_scales.data_ptr(), M, N, K, code, out, sp, sn, st))
    lead = (x if scales is None else x[0]).shape[:-1]
    return y if len(lead) == 1 else y.view(*lead, N)


def grouped_matmul(x: Union[Fp8Rows, torch.Tensor], w: torch.Tensor, w_scales: torch.Tensor, ids: torch.Tensor,
                   rows: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Routed experts: y [routes, N], y[r] = x[rows[r]] . w[ids[r]]^T, with
    x [T, K] as in ``matmul``, a bank w [experts, N, K], w_scales [experts,
    ceil(N / 128), ceil(K / 128)], and ids and rows int32 [routes] on the device, in
    any order (rows None: x has a row for each route).  A route whose expert or
    row is out of range, as padded ones may have, gives zeros (C ABI:
    eq_fp8_grouped_matmul)."""
    E, N, K = _weight(w, w_scales, 3)
    if (x if isinstance(x, torch.Tensor) else x[0]).dim() != 2:
        raise EreduError(f"x must be [rows, {K}]")
    xr, scales, stride, code = _x_of(x, K)
    dtype = _out_dtype(x, dtype)
    st = _here(xr, scales, w, w_scales, ids, rows)
    if ids.dtype is not torch.int32 or ids.dim() != 1:
        raise EreduError("ids must be a one-dimensional int32 tensor")
    if rows is not None:
        if rows.dtype is not torch.int32 or rows.shape != ids.shape:
            raise EreduError("rows must be an int32 tensor as long as ids")
        rows = rows.contiguous()
    ids = ids.contiguous()
    R, T = ids.shape[0], xr.shape[0]
    lib, out = _native.lib(), _DTYPE_CODE[dtype]
    y = xr.new_empty((R, N), dtype=dtype)
    sp, sn, hold = (_scratch(lib.eq_fp8_grouped_matmul_scratch(T, E, R, N, K, code, out), xr.device) if _capturing()
                    else (None, 0, None))
    check(lib.eq_fp8_grouped_matmul(y.data_ptr(), xr.data_ptr(), xr.stride(0),
                                    None if scales is None else scales.data_ptr(), stride, T, w.data_ptr(),
                                    w_scales.data_ptr(), E, ids.data_ptr(), None if rows is None else rows.data_ptr(), R, N,
                                    K, code, out, sp, sn, st))
    return y
