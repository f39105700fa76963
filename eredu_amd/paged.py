"""Paged 8-bit key/value cache: many sequences, shared prefixes, any number of
tokens a call, on the HIP kernels (``include/eredu_kv.h``: eq_kv_*).

Stands beside the dense one-sequence cache of :mod:`eredu_amd.decode`
(``rope_attention_decode``), in the place of the reference's caches and
``fast::scaled_dot_product_attention`` (``Attention::attend``,
eredu-architectures/src/llama.rs:296-330).  One step of a model over a batch:

    cache.extend(seqs, 1)                                # pages for the new tokens
    for layer in range(cache.n_layers):
        cache.append(layer, k, v, seqs, rope=rope)       # rotate, quantize, write
        out = cache.attention(layer, q, seqs, rope=rope)

Sequences are rows of a page table, named by int32 device tensors.  A call with
rows of several tokens a sequence takes their offsets ``cu`` ([n + 1] int32 on
the device; None: the rows divide evenly); the rows are always the last ones of
their sequences.  Tables, lengths and reference counts live on the device and
are read when the kernels run: nothing here waits for the GPU but ``check`` and
``free_pages``, and a captured graph decodes across page borders.

Calls that write a cache (extend, append, fork, shrink, free, compact) have to be
ordered with every other call on it, as with any tensor that is written in
place.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import numpy as np
import torch

from . import _native
from ._native import EreduError, check
from .quantization import _DTYPE_CODE, _get_device, _stream

_HALVES = (torch.bfloat16, torch.float16)


def rope_table(freqs, positions: int, device=None) -> torch.Tensor:
    """The rotation table that ``append`` and ``attention`` take: [positions,
    2 * len(freqs)] float32, row p the cosines of the angles p / freqs[i], then the
    sines (angles in 64 bits; freqs as ``decode.llama3_rope_freqs`` gives)."""
    f = np.asarray(freqs, dtype=np.float64).reshape(-1)
    if positions <= 0 or f.size == 0:
        raise EreduError("rope_table needs at least one position and one frequency")
    a = np.arange(positions, dtype=np.float64)[:, None] / f[None, :]
    t = torch.from_numpy(np.concatenate((np.cos(a), np.sin(a)), axis=1).astype(np.float32))
    return t.to(torch.device("cuda") if device is None else device)


def _ids(t: torch.Tensor, what: str, index: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.get_device() != index or t.dim() != 1:
        raise EreduError(f"{what} must be a one-dimensional int32 tensor on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


# Whether the current stream is being captured (a method of torch.cuda without its wrapper).
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)

class PagedKVCache:
    """``n_pages`` pages of ``page_size`` tokens (16, 32, 64 or 128) for
    ``n_layers`` layers of ``n_kv_heads`` heads of ``head_dim`` (64, 128 or 256),
    and ``max_seqs`` sequences of at most ``max_pages_per_seq`` pages.

    Keys and values are int8 codes with a power-of-two scale for each page and
    head (E8M0 bytes): half the bytes of a bf16 cache, a value off by less than one
    step, at most max|x| / 63.5 over its page and head.  A page takes
    2 * n_layers * n_kv_heads * (page_size * head_dim + 1) bytes.  Long contexts
    are read about 15 % slower from pages of 128 than from smaller ones."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: int, page_size: int = 64, device=None):
        dev = torch.device("cuda") if device is None else torch.device(device)
        for v, n in ((n_layers, "n_layers"), (n_pages, "n_pages"), (n_kv_heads, "n_kv_heads"), (max_seqs, "max_seqs"),
                     (max_pages_per_seq, "max_pages_per_seq")):
            if v <= 0:
                raise EreduError(f"{n} must be positive")
        codes = lambda *s: torch.zeros((n_layers, n_pages, n_kv_heads, *s), dtype=torch.int8, device=dev)
        scales = lambda: torch.ones((n_layers, n_pages, n_kv_heads), dtype=torch.uint8, device=dev)
        ints = lambda *s, fill=0: torch.full(s, fill, dtype=torch.int32, device=dev)
        self._adopt(codes(page_size, head_dim), codes(head_dim, page_size), scales(), scales(),
                    ints(max_seqs, max_pages_per_seq, fill=-1), ints(max_seqs), ints(n_pages))

    @classmethod
    def over(cls, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
             tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor) -> "PagedKVCache":
        """A cache in tensors that the caller holds: int8 k_codes [layers, pages,
        heads, page, dim] and v_codes [layers, pages, heads, dim, page], uint8 scales
        [layers, pages, heads], int32 tables [sequences, pages each] (-1: none),
        lengths [sequences] and refs [pages] (how many table entries name a page)."""
        self = cls.__new__(cls)
        self._adopt(k_codes, v_codes, k_scales, v_scales, tables, lengths, refs)
        return self

    def _adopt(self, k_codes, v_codes, k_scales, v_scales, tables, lengths, refs) -> None:
        if k_codes.dim() != 5 or tables.dim() != 2:
            raise EreduError("k_codes must be [layers, pages, heads, page, dim], tables [sequences, pages]")
        L, P, H, T, D = k_codes.shape
        S, W = tables.shape
        for t, n, dt, shape in ((k_codes, "k_codes", torch.int8, (L, P, H, T, D)),
                                (v_codes, "v_codes", torch.int8, (L, P, H, D, T)),
                                (k_scales, "k_scales", torch.uint8, (L, P, H)),
                                (v_scales, "v_scales", torch.uint8, (L, P, H)),
                                (tables, "tables", torch.int32, (S, W)), (lengths, "lengths", torch.int32, (S,)),
                                (refs, "refs", torch.int32, (P,))):
            if t.dtype != dt or tuple(t.shape) != shape or not t.is_contiguous() or t.device != k_codes.device:
                raise EreduError(f"{n} must be a contiguous {dt} tensor of shape {shape} on {k_codes.device}")
        if T not in (16, 32, 64, 128) or D not in (64, 128, 256):
            raise EreduError(f"page size must be 16, 32, 64 or 128 and head_dim 64, 128 or 256, got {T} and {D}")
        if not k_codes.is_cuda:
            raise EreduError("all arrays must live on the GPU (the library has no host path)")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.tables, self.lengths, self.refs = tables, lengths, refs
        self.missing = torch.zeros((1,), dtype=torch.int32, device=k_codes.device)
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = L, P, H, T, D
        self.max_seqs, self.max_pages_per_seq = S, W
        self._scale = D ** -0.5
        self.device = k_codes.device
        c = _native.KvCache(*(t.data_ptr() for t in (k_codes, v_codes, k_scales, v_scales, tables, lengths, refs,
                                                     self.missing)), L, P, S, W, H, T, D)
        self._c, self._ref, self._index = c, ctypes.byref(c), k_codes.get_device()

    # ------------------------------------------------------------ operands

    def _here(self) -> int:
        """The current stream, once the current device is the cache's."""
        if (_get_device() if _get_device is not None else torch.cuda.current_device()) != self._index:
            raise EreduError(f"the cache lives on {self.device}: make that the current device")
        return _stream()

    def _rows(self, t: torch.Tensor, what: str) -> torch.Tensor:
        """[rows, heads, dim] or [rows, heads * dim] as the kernels read it: heads and
        dimensions contiguous, rows at any stride of a multiple of 8, as parts of a
        fused projection are.  Any other layout is copied."""
        if t.get_device() != self._index:
            raise EreduError(f"{what} must live on {self.device}")
        if t.dtype not in _HALVES:
            raise EreduError(f"{what} must be bfloat16 or float16, got {t.dtype}")
        D = self.head_dim
        if t.dim() == 2 and t.shape[1] % D == 0:
            t = t.unflatten(1, (t.shape[1] // D, D))
        if t.dim() != 3 or t.shape[2] != D:
            raise EreduError(f"{what} must be [rows, heads, {D}], got {tuple(t.shape)}")
        if t.is_contiguous() and t.data_ptr() % 16 == 0:
            # (a single row is contiguous at any stride: heads that were turned to the front of one token)
            row = t.shape[1] * D
            return t if t.stride(0) == row or t.shape[0] != 1 else t.as_strided(t.shape, (row, D, 1))
        if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != D) or t.stride(0) % 8 or \
                t.stride(0) < t.shape[1] * D or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def _batch(self, seqs: torch.Tensor, cu: Optional[torch.Tensor], total: int) -> Tuple[torch.Tensor, int, Optional[torch.Tensor]]:
        seqs = _ids(seqs, "seqs", self._index)
        n = seqs.shape[0]
        if cu is not None:
            cu = _ids(cu, "cu", self._index)
            if cu.shape[0] != n + 1:
                raise EreduError(f"cu must hold {n + 1} offsets for {n} sequences, got {cu.shape[0]}")
        elif total % n if n else total:
            raise EreduError(f"{total} rows do not divide evenly among {n} sequences: pass cu")
        return seqs, n, cu

    def _rope(self, rope: Optional[torch.Tensor]) -> Tuple[Optional[int], int]:
        if rope is None:
            return None, 0
        if rope.dtype is not torch.float32 or rope.dim() != 2 or rope.shape[1] != self.head_dim or \
                not rope.is_contiguous() or rope.get_device() != self._index:
            raise EreduError(f"rope must be a contiguous float32 tensor [positions, {self.head_dim}] on {self.device}")
        return rope.data_ptr(), rope.shape[0]

    def _scratch(self, need: int) -> Tuple[Optional[int], int, Optional[torch.Tensor]]:
        """Scratch of a call from torch: in stream order, and under capture a graph's
        own, so that graphs share nothing.  (Other eager calls take the library's
        workspace of their stream, which saves them the allocation, and which keeps the
        most that such a call needed as long as the process runs.)"""
        if need < 0:
            check(1)
        if need == 0:
            return None, 0, None
        t = torch.empty((need,), dtype=torch.uint8, device=self.device)
        return t.data_ptr(), need, t

    # ------------------------------------------------------------ tokens

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor,
               cu: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None) -> None:
        """Writes k and v [rows, n_kv_heads, head_dim] (bf16 or f16) as the last
        tokens of their sequences, k turned by ``rope`` (``rope_table``) at their
        positions first (C ABI: eq_kv_append)."""
        k, v = self._rows(k, "k"), self._rows(v, "v")
        if k.shape != v.shape or k.dtype != v.dtype or k.shape[1] != self.n_kv_heads:
            raise EreduError(f"k and v must both be [rows, {self.n_kv_heads}, {self.head_dim}] of one dtype")
        seqs, n, cu = self._batch(seqs, cu, k.shape[0])
        rp, rn = self._rope(rope)
        check(_native.lib().eq_kv_append(self._ref, layer, k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0),
                                         seqs.data_ptr(), n, None if cu is None else cu.data_ptr(), k.shape[0], rp,
                                         rn, _DTYPE_CODE[k.dtype], self._here()))

    def attention(self, layer: int, q: torch.Tensor, seqs: torch.Tensor, cu: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None, causal: bool = True, window: int = 0,
                  rope: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale * q . K^T) . V for q [rows, n_heads, head_dim] (bf16 or
        f16; n_heads any multiple of n_kv_heads), the rows the last tokens of their
        sequences: causal with an optional sliding ``window``, or, not causal, over all
        tokens of the sequence (cross attention).  scale: 1 / sqrt(head_dim) if None.
        Rows that see no token give zeros; rows that no entry of cu covers are left as
        they are in ``out``.  The work is laid out by the entries' rows on average: long
        prompts and single tokens after long contexts are faster in calls of their own
        (C ABI: eq_kv_attention)."""
        q = self._rows(q, "q")
        rows, heads, D = q.shape
        seqs, n, cu = self._batch(seqs, cu, rows)
        rp, rn = self._rope(rope)
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty((rows, heads, D), dtype=q.dtype, device=self.device)
        elif out.dtype != q.dtype or out.numel() != q.numel() or not out.is_contiguous() or out.get_device() != self._index:
            raise EreduError(f"out must be a contiguous {q.dtype} tensor of {q.numel()} values on {self.device}")
        L, st = _native.lib(), self._here()
        wp, wn, ws = None, 0, None
        if rows * heads > 8192 or _capturing():  # (fewer rows need at most 64 MiB, decode steps of 4 heads a group 8)
            wp, wn, ws = self._scratch(L.eq_kv_attention_scratch(self._ref, heads, n, rows, cu is not None))
        check(L.eq_kv_attention(out.data_ptr(), q.data_ptr(), q.stride(0), heads, self._ref, layer, seqs.data_ptr(), n,
                                None if cu is None else cu.data_ptr(), rows, self._scale if scale is None else scale,
                                causal, window, rp, rn, _DTYPE_CODE[q.dtype], wp, wn, st))
        return out

    def read(self, layer: int, seqs: torch.Tensor, tokens: Union[int, torch.Tensor], total: Optional[int] = None,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The last tokens' keys and values back, each [rows, n_kv_heads, head_dim]:
        ``tokens`` of every sequence, or by offsets cu with their ``total`` (bf16 holds
        the stored values exactly; C ABI: eq_kv_read)."""
        cu = tokens if isinstance(tokens, torch.Tensor) else None
        if cu is not None and total is None:
            raise EreduError("read by offsets needs total, the number of rows")
        rows = int(total) if cu is not None else int(tokens) * seqs.numel()
        if rows < 0 or dtype not in _DTYPE_CODE:
            raise EreduError("read needs a number of tokens that is not negative, and float32, float16 or bfloat16")
        seqs, n, cu = self._batch(seqs, cu, rows)
        k, v = (torch.empty((rows, self.n_kv_heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2))
        check(_native.lib().eq_kv_read(k.data_ptr(), v.data_ptr(), self._ref, layer, seqs.data_ptr(), n,
                                       None if cu is None else cu.data_ptr(), rows, _DTYPE_CODE[dtype],
                                       self._here()))
        return k, v

    # ------------------------------------------------------------ pages

    def extend(self, seqs: torch.Tensor, tokens: Union[int, torch.Tensor]) -> None:
        """Grows the sequences by ``tokens`` each, or by the differences of offsets
        cu: lengths, pages (the lowest free ones), and a page of its own for a sequence
        whose last page is partly filled and shared (C ABI: eq_kv_extend).  Pages that
        are not to be had are counted; see ``check``."""
        cu = tokens if isinstance(tokens, torch.Tensor) else None
        seqs, n, cu = self._batch(seqs, cu, 0)
        L, st = _native.lib(), self._here()
        wp, wn, ws = self._scratch(L.eq_kv_pages_scratch(self._ref, n) if _capturing() else 0)
        check(L.eq_kv_extend(self._ref, seqs.data_ptr(), n, None if cu is None else cu.data_ptr(),
                             0 if cu is not None else tokens, wp, wn, st))

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Sequence dst[i] becomes a copy of src[i], sharing its pages; all pairs from
        the state before the call, so beams can be permuted (C ABI: eq_kv_fork)."""
        src, dst = _ids(src, "src", self._index), _ids(dst, "dst", self._index)
        if src.numel() != dst.numel():
            raise EreduError(f"src and dst must be of one length, got {src.numel()} and {dst.numel()}")
        L, st = _native.lib(), self._here()
        wp, wn, ws = self._scratch(L.eq_kv_pages_scratch(self._ref, src.numel()) if _capturing() else 0)
        check(L.eq_kv_fork(self._ref, src.data_ptr(), dst.data_ptr(), src.numel(), wp, wn, st))

    def shrink(self, seqs: torch.Tensor, tokens: Union[int, torch.Tensor]) -> None:
        """Takes the sequences' last ``tokens`` back (of all the same number, or int32
        [n] on the device, at most what each has) with the pages behind the rest: the
        drafts of a step that were refused (C ABI: eq_kv_shrink)."""
        seqs = _ids(seqs, "seqs", self._index)
        counts = _ids(tokens, "tokens", self._index) if isinstance(tokens, torch.Tensor) else None
        if counts is not None and counts.numel() != seqs.numel():
            raise EreduError(f"tokens must hold {seqs.numel()} numbers for as many sequences, got {counts.numel()}")
        check(_native.lib().eq_kv_shrink(self._ref, seqs.data_ptr(), seqs.numel(),
                                         None if counts is None else counts.data_ptr(),
                                         0 if counts is not None else tokens, self._here()))

    def free(self, seqs: torch.Tensor) -> None:
        """Empties the sequences and gives up their pages (C ABI: eq_kv_free)."""
        seqs = _ids(seqs, "seqs", self._index)
        check(_native.lib().eq_kv_free(self._ref, seqs.data_ptr(), seqs.numel(), self._here()))

    def compact(self) -> None:
        """Moves the pages in use to the lowest indices (C ABI: eq_kv_compact)."""
        L, st = _native.lib(), self._here()
        wp, wn, ws = self._scratch(L.eq_kv_pages_scratch(self._ref, 0) if _capturing() else 0)
        check(L.eq_kv_compact(self._ref, wp, wn, st))

    def free_pages(self) -> int:
        """Pages that no sequence holds (waits for the GPU)."""
        return int((self.refs <= 0).sum().item())

    def check(self) -> None:
        """Raises if ``extend`` had no page for some tokens since the last check (waits for the GPU)."""
        lost = int(self.missing.item())
        if lost:
            self.missing.zero_()
            raise EreduError(f"the cache ran out of pages: {lost} could not be given")
