"""The paged 8-bit key/value cache, as cases that can be timed and checked.

A cache holds tokens in pages of ``page`` tokens: int8 codes and one E8M0 scale
byte for each page and KV head, keys [page, heads, token, dim] and values
[page, heads, dim, token], value = code * 2^(byte - 127), byte 255 = NaN.
Sequences name their pages in a table, pages count the sequences that hold
them.  Four kinds of case: attention over the cache (one token, a few, prompts, cross
attention), new tokens appended and read back, sequences forked and extended,
and sequences that finish, are compacted away and replaced.

``listed()`` names representative points, ``draw()`` picks others of the same
ranges.  The plain form of every operator is written in elementary torch
operations here; ``exact()`` restates them in 64 bits, one sequence at a time.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_BASE = 500000.0


def listed():
    return [
        # One conversation, one token after 1024 cached ones: the smallest call, latency.
        dict(name="decode-1024", kind="attend", n=1, q=1, lo=1025, hi=1025, heads=32, kv=8, dim=128, page=64,
             dtype="bf16", rope=True, causal=True, window=0, fresh=False, mix=0),
        # A serving batch of 48 conversations of very different lengths.
        dict(name="decode-48-ragged", kind="attend", n=48, q=1, lo=17, hi=8191, heads=32, kv=8, dim=128, page=64,
             dtype="bf16", rope=True, causal=True, window=0, fresh=False, mix=1),
        # One token after a book: work has to be split over the one long axis.
        dict(name="decode-131071", kind="attend", n=1, q=1, lo=131071, hi=131071, heads=32, kv=8, dim=128, page=128,
             dtype="bf16", rope=True, causal=True, window=0, fresh=False, mix=2),
        # Five drafted tokens for each of 16 sequences checked at once, every head with keys of its own, small pages.
        dict(name="verify-16x5", kind="attend", n=16, q=5, lo=300, hi=4099, heads=16, kv=16, dim=64, page=16,
             dtype="f16", rope=True, causal=True, window=0, fresh=False, mix=3),
        # Seven new prompts of different lengths prefilled in one batch.
        dict(name="prompts-7-ragged", kind="attend", n=7, q=2500, lo=0, hi=0, heads=32, kv=8, dim=128, page=64,
             dtype="bf16", rope=True, causal=True, window=0, fresh=True, mix=4),
        # The last chunk of a long prompt: 2048 queries over 32768 tokens, the largest product.
        dict(name="chunk-2048-of-32768", kind="attend", n=1, q=2048, lo=32768, hi=32768, heads=32, kv=8, dim=128, page=64,
             dtype="bf16", rope=True, causal=True, window=0, fresh=False, mix=5),
        # Decoder tokens of 8 requests over the 1500 states of an encoder (no mask, no rotation).
        dict(name="cross-8x1500", kind="attend", n=8, q=100, lo=1500, hi=1500, heads=20, kv=20, dim=64, page=32,
             dtype="f16", rope=False, causal=False, window=0, fresh=False, mix=6),
        # One new token for each of 64 sequences into half-filled pages, and the last 64 tokens read back.
        dict(name="append-64x1", kind="append", n=64, q=1, lo=70, hi=4096, kv=8, dim=128, page=64, dtype="bf16", rope=True,
             back=64, mix=7),
        # Prompts of about 10000 tokens in all written behind cached prefixes, and read back.
        dict(name="append-5-prompts", kind="append", n=5, q=4000, lo=0, hi=0, kv=8, dim=128, page=64, dtype="bf16", rope=True,
             back=0, mix=8),
        # One prompt sampled 15 times: the children share its pages and get the page they write to for themselves.
        dict(name="fork-15-extend", kind="fork", n=15, tokens=1957, layers=32, kv=8, dim=128, page=64, mix=9),
        # Half of the sequences end, the pages close ranks, new sequences come; then the other half.
        dict(name="compact-16", kind="compact", n=16, lo=40, hi=700, layers=32, kv=8, dim=128, page=64, mix=10),
        # The same for a small cache of one layer: latency.
        dict(name="compact-4-small", kind="compact", n=4, lo=16, hi=250, layers=1, kv=4, dim=64, page=16, mix=11),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "append", "append", "fork", "compact"))
    heads, kv, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 16, 64), (4, 1, 128), (24, 3, 64), (8, 4, 256), (40, 8, 128)))
    page, dtype, mix = rng.choice((16, 32, 64, 64, 128)), rng.choice(("bf16", "bf16", "f16")), rng.randrange(1 << 20)
    if kind == "attend":
        form = rng.choice(("decode", "decode", "verify", "prompts", "chunk", "cross"))
        c = dict(kind=kind, n=1, q=1, lo=1, hi=1, heads=heads, kv=kv, dim=dim, page=page, dtype=dtype,
                 rope=form != "cross" and rng.random() < 0.8, causal=form != "cross",
                 window=rng.choice((0, 0, _log(rng, 100, 5000))) if form != "cross" else 0, fresh=form == "prompts", mix=mix)
        if form == "decode":
            c["n"] = _log(rng, 1, 64)
            c["hi"] = _log(rng, 64, min(131072, 400000 // c["n"]))
            c["lo"] = _log(rng, max(1, c["hi"] // 50), c["hi"])
        elif form == "verify":
            c["n"], c["q"] = _log(rng, 1, 24), rng.randint(2, 12)
            c["hi"] = _log(rng, 64, 8000)
            c["lo"] = max(c["q"], c["hi"] // 9)
        elif form == "prompts":
            c["n"], c["q"] = _log(rng, 1, 10), _log(rng, 20, 3500)
        elif form == "chunk":
            c["n"], c["q"] = 1, _log(rng, 64, 2048)
            c["lo"] = c["hi"] = max(c["q"], _log(rng, 512, 24000))
        else:
            c["n"], c["q"] = _log(rng, 1, 12), _log(rng, 1, 250)
            c["lo"], c["hi"] = 100, _log(rng, 128, 3000)
        return c
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, n=_log(rng, 1, 128), q=1, lo=1, hi=_log(rng, 2, 4000), kv=kv, dim=dim, page=page, dtype=dtype,
                        rope=rng.random() < 0.8, back=page, mix=mix)
        return dict(kind=kind, n=_log(rng, 1, 8), q=_log(rng, 10, 5000), lo=0, hi=0, kv=kv, dim=dim, page=page, dtype=dtype,
                    rope=rng.random() < 0.8, back=0, mix=mix)
    if kind == "fork":
        return dict(kind=kind, n=_log(rng, 1, 24), tokens=_log(rng, 10, 3000), layers=rng.choice((1, 4, 16, 32)), kv=kv,
                    dim=min(dim, 128), page=page, mix=mix)
    return dict(kind=kind, n=_log(rng, 2, 24), lo=8, hi=_log(rng, 32, 800), layers=rng.choice((1, 4, 16)), kv=min(kv, 8),
                dim=min(dim, 128), page=page, mix=mix)


# ------------------------------------------------------------ what a case's sequences are like

def _shape(c):
    """(tokens of each sequence, how many of them are this call's), from the case alone."""
    r = random.Random(c["mix"])
    n, q = c["n"], c.get("q", 1)
    if c["kind"] == "fork":
        return [c["tokens"]], [0]
    if c["kind"] == "compact":
        return [r.randint(c["lo"], c["hi"]) for _ in range(n)], [0] * n
    if c["kind"] == "append" and q > 1:  # prompts behind a cached prefix of any length
        new = [max(1, round(q * r.uniform(0.05, 1.0))) for _ in range(n)]
        return [x + r.randint(0, 3 * c["page"]) for x in new], new
    if c.get("fresh"):
        new = [max(1, round(q * r.uniform(0.02, 1.0))) for _ in range(n)]
        return list(new), new
    lens = [max(q, _log(r, c["lo"], c["hi"])) for _ in range(n)]
    if c["kind"] == "attend" and not c["causal"]:
        return [max(1, x) for x in lens], [r.randint(max(1, q // 2), q) for _ in range(n)]
    return lens, [q] * n


def _cdiv(a, b):
    return -(-a // b)


def _cu(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEVICE)


def _pages(lens, page):
    return [_cdiv(x, page) for x in lens]


def work(c):
    lens, new = _shape(c)
    kv, D, T = c["kv"], c["dim"], c["page"]
    if c["kind"] == "attend":
        H, pairs, seen = c["heads"], 0, 0
        for L, q in zip(lens, new):
            if not c["causal"]:
                pairs, seen = pairs + L * q, seen + L
                continue
            w = c["window"] or L
            pairs += sum(min(p + 1, w) for p in range(L - q, L))
            seen += L - max(0, L - q + 1 - w)
        moved = 2 * seen * kv * D + 2 * kv * _cdiv(seen, T) + 4 * sum(new) * H * D
        return {"bytes": moved, "flops": 4 * pairs * H * D}
    if c["kind"] == "append":
        values = 2 * sum(new) * kv * D
        back = 2 * sum(min(x, c["back"] or x) for x in (lens if c["back"] else new)) * kv * D
        return {"bytes": 3 * values + 3 * back, "flops": 0}
    one = 2 * c["layers"] * kv * (T * D + 1)
    if c["kind"] == "fork":
        copies = c["n"] if c["tokens"] % T else 0
        return {"bytes": one * (copies + (1 if copies else 0)) + 4 * c["n"] * _cdiv(c["tokens"] + 1, T), "flops": 0}
    held = _pages(lens, T)
    a, b = sum(held[0::2]), sum(held[1::2])
    return {"bytes": 2 * one * min(a, b) * 2 + 16 * sum(held), "flops": 0}


# ------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _codes(g, *shape):
    """Codes of normally distributed values whose largest is most of the range."""
    out = torch.empty(shape, dtype=torch.int8, device=DEVICE)
    for part in out.view(-1).split(1 << 26):
        part.copy_((torch.randn(part.shape, generator=g, device=DEVICE) * 28).round_().clamp_(-127, 127))
    return out


def _rope(positions, D):
    """The rotation of every position, [positions, D] f32: cosines, then sines (angles in 64 bits)."""
    inv = ROPE_BASE ** (-torch.arange(D // 2, dtype=torch.float64, device=DEVICE) * 2 / D)
    a = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).float()


def prepare(c, seed):
    g = _gen(seed)
    lens, new = _shape(c)
    kv, D, T = c["kv"], c["dim"], c["page"]
    held = _pages(lens, T)
    layers = c.get("layers", 1)
    if c["kind"] == "fork":
        rows, width, P = 1 + c["n"], _cdiv(c["tokens"] + 1, T), held[0] + 2 * c["n"] + 3
    else:
        rows, width, P = c["n"] + 3, max(held) + 2, sum(held) + 7 + sum(held) // 8
    s = dict(case=c, lens=lens, new=new, layers=layers)
    s["k_codes"], s["v_codes"] = _codes(g, layers, P, kv, T, D), _codes(g, layers, P, kv, D, T)
    s["k_scales"] = torch.randint(121, 124, (layers, P, kv), generator=g, device=DEVICE, dtype=torch.uint8)
    s["v_scales"] = torch.randint(121, 124, (layers, P, kv), generator=g, device=DEVICE, dtype=torch.uint8)
    order = torch.randperm(P, generator=g, device=DEVICE).int()  # pages lie anywhere
    seqs = torch.randperm(rows, generator=g, device=DEVICE).int()[: len(lens)]  # and so do sequences
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for i, (row, h) in enumerate(zip(seqs.tolist(), held)):
        tables[row, :h] = order[at:at + h].cpu()
        at += h
    s["tables"] = tables.to(DEVICE)
    s["lengths"] = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    s["lengths"][seqs.long()] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    s["refs"] = torch.zeros(P, dtype=torch.int32, device=DEVICE)
    s["refs"][order[:at].long()] = 1
    s["seqs"] = seqs
    total = sum(new)
    dt = DTYPES[c.get("dtype", "bf16")]
    s["cu"] = None if all(x == new[0] for x in new) else _cu(new)
    s["rope"] = _rope(width * T, D) if c.get("rope") else None
    if c["kind"] == "attend":
        s["q"] = (torch.randn(total, c["heads"], D, generator=g, device=DEVICE) * 1.5).to(dt)
    elif c["kind"] == "append":
        s["k"] = (torch.randn(total, kv, D, generator=g, device=DEVICE) * torch.linspace(0.3, 2.5, D, device=DEVICE)).to(dt)
        s["v"] = (torch.randn(total, kv, D, generator=g, device=DEVICE) * 1.2).to(dt)
        back = [min(x, c["back"]) if c["back"] else y for x, y in zip(lens, new)]
        s["back"], s["back_cu"] = back, _cu(back)
    elif c["kind"] == "fork":
        others = [i for i in range(rows) if i != seqs.item()]
        s["src"] = seqs.expand(c["n"]).contiguous()
        s["dst"] = torch.tensor(others, dtype=torch.int32, device=DEVICE)
    else:
        s["halves"] = [(seqs[k::2].contiguous(), _cu(lens[k::2])) for k in (0, 1)]
    if own:
        from eredu_amd import PagedKVCache

        s["cache"] = PagedKVCache.over(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], s["tables"], s["lengths"],
                                       s["refs"])
    return s


# ------------------------------------------------------------ one pass

def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "attend":
        if own:
            return s["cache"].attention(0, s["q"], s["seqs"], s["cu"], causal=c["causal"], window=c["window"], rope=s["rope"])
        return _attention(s, c)
    if kind == "append":
        if own:
            s["cache"].append(0, s["k"], s["v"], s["seqs"], s["cu"], rope=s["rope"])
            return s["cache"].read(0, s["seqs"], s["back_cu"], total=sum(s["back"]))
        _append(s, c)
        return _read(s, c)
    if kind == "fork":
        if own:
            s["cache"].free(s["dst"])
            s["cache"].fork(s["src"], s["dst"])
            s["cache"].extend(s["dst"], 1)
        else:
            _free(s, s["dst"])
            _fork(s, s["src"], s["dst"])
            _extend(s, s["dst"], torch.ones_like(s["dst"]))
    else:
        for seqs, cu in s["halves"]:
            if own:
                s["cache"].free(seqs)
                s["cache"].compact()
                s["cache"].extend(seqs, cu)
            else:
                _free(s, seqs)
                _compact(s)
                _extend(s, seqs, cu[1:] - cu[:-1])
    return {n: s[n] for n in ("tables", "lengths", "refs", "k_codes", "v_codes", "k_scales", "v_scales")}


# ------------------------------------------------------------ the plain forms

def _pow2(e):
    """2^e in f32, from its bits; 0 below the normal values."""
    return torch.where(e < -126, 0, e.int().clamp_min(-126) + 127 << 23).view(torch.float32)


def _scale_of(b):
    """2^(byte - 127) in f32, NaN for 255."""
    return torch.where(b == 255, float("nan"), _pow2(b.int() - 127))


def _rotate(x, rot):
    """x [rows, heads, D] f32 turned by the rows' angles, pairs (d, d + D/2)."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cs, sn = rot[:, None, :half], rot[:, None, half:]
    return torch.cat((a * cs - b * sn, b * cs + a * sn), -1)


def _spread(s, counts):
    """For the tokens of a call that covers the last counts[i] tokens of each sequence: which one, and its position."""
    which = torch.repeat_interleave(torch.arange(len(counts), device=DEVICE), torch.tensor(counts, device=DEVICE))
    first = _cu(counts)[:-1].long()
    lens = s["lengths"][s["seqs"].long()].long()
    pos = torch.arange(which.numel(), device=DEVICE) - first[which] + (lens - torch.tensor(counts, device=DEVICE))[which]
    return which, pos


def _dense(s, c):
    """Every sequence's keys and values in f32, [n, kv, tokens padded to whole pages, D], and their number of tokens."""
    pages = _cdiv(max(s["lens"]), c["page"])
    tab = s["tables"][s["seqs"].long(), :pages].clamp_min(0).long()
    k, v = s["k_codes"][0][tab].float(), s["v_codes"][0][tab].float()
    k = k * _scale_of(s["k_scales"][0][tab])[..., None, None]
    v = v * _scale_of(s["v_scales"][0][tab])[..., None, None]
    n, _, kv, T, D = k.shape
    return (k.permute(0, 2, 1, 3, 4).reshape(n, kv, pages * T, D), v.permute(0, 2, 1, 4, 3).reshape(n, kv, pages * T, D))


def _attention(s, c):
    q, new, lens = s["q"].float(), s["new"], s["lengths"][s["seqs"].long()].long()
    which, pos = _spread(s, new)
    if s["rope"] is not None:
        q = _rotate(q, s["rope"][pos])
    n, most, D, H, kv = c["n"], max(new), c["dim"], c["heads"], c["kv"]
    slot = torch.arange(which.numel(), device=DEVICE) - _cu(new)[:-1].long()[which]
    qp = torch.zeros(n, most, H, D, device=DEVICE)
    qp[which, slot] = q
    at = torch.full((n, most), -1, dtype=torch.int64, device=DEVICE)
    at[which, slot] = pos if c["causal"] else 1 << 40
    k, v = _dense(s, c)
    j = torch.arange(k.shape[2], device=DEVICE)
    seen = (j[None, None] <= at[..., None]) & (j < lens[:, None])[:, None]
    if c["window"]:
        seen &= j[None, None] > at[..., None] - c["window"]
    qg = qp.view(n, most, kv, H // kv, D).permute(0, 2, 3, 1, 4).reshape(n, kv, H // kv * most, D)
    p = (qg @ k.transpose(-1, -2)).mul_(D ** -0.5).view(n, kv, H // kv, most, -1)
    p.masked_fill_(~seen[:, None, None], float("-inf"))
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == float("-inf"), 0, m)).exp_()
    z = p.sum(-1, keepdim=True)
    p.div_(torch.where(z == 0, 1, z))
    o = (p.view(n, kv, H // kv * most, -1) @ v).view(n, H, most, D)
    return o[which, :, slot].to(s["q"].dtype)


def _byte(most):
    """The scale byte of values whose largest magnitude is `most`."""
    m, e = torch.frexp(most)
    b = torch.where(m <= 127 / 128, e + 120, e + 121).clamp(1, 254)
    return torch.where(torch.isfinite(most), torch.where(most == 0, 1, b), 255).to(torch.uint8)


def _append(s, c):
    T = c["page"]
    which, pos = _spread(s, s["new"])
    page = s["tables"][s["seqs"].long()[which], pos // T].long()
    off = pos % T
    lens = s["lengths"][s["seqs"].long()].long()
    start = lens - torch.tensor(s["new"], device=DEVICE)  # of each sequence's new tokens
    width = s["tables"].shape[1]
    first = s["tables"][s["seqs"].long(), (start // T).clamp_max(width - 1)].long()
    kept = torch.arange(T, device=DEVICE) < (start % T)[:, None]  # tokens that the first page already has
    old = (start % T) > 0
    k = s["k"].float()
    if s["rope"] is not None:
        k = _rotate(k, s["rope"][pos])
    for x, name, turned in ((k, "k", False), (s["v"].float(), "v", True)):
        codes, scales = s[name + "_codes"][0], s[name + "_scales"][0]
        most = torch.zeros(scales.shape, device=DEVICE).index_reduce_(0, page, x.abs().amax(-1), "amax")
        was = torch.zeros_like(scales)
        was[first[old]] = scales[first[old]]
        now = torch.maximum(_byte(most), was)
        # the codes that the first pages hold, in the new scale
        sel = first[old]
        held = codes[sel].float()
        held = held.transpose(-1, -2) if turned else held
        moved = torch.round(held * _pow2(was[sel].int() - now[sel].int())[..., None, None])
        held = torch.where(kept[old][:, None, :, None] & (now[sel] != 255)[..., None, None], moved, held).to(torch.int8)
        codes[sel] = held.transpose(-1, -2) if turned else held
        new = torch.round(x * _pow2(127 - now[page].int())[..., None])
        new = torch.where((now[page] == 255)[..., None], 0, new).to(torch.int8)
        if turned:
            codes[page, :, :, off] = new
        else:
            codes[page, :, off] = new
        scales[page] = now[page]


def _read(s, c):
    T = c["page"]
    which, pos = _spread(s, s["back"])
    page, off = s["tables"][s["seqs"].long()[which], pos // T].long(), pos % T
    k = s["k_codes"][0][page, :, off].float() * _scale_of(s["k_scales"][0][page])[..., None]
    v = s["v_codes"][0][page, :, :, off].float() * _scale_of(s["v_scales"][0][page])[..., None]
    return k.bfloat16(), v.bfloat16()


def _free(s, seqs):
    rows = s["tables"][seqs.long()]
    s["refs"].index_add_(0, rows.clamp_min(0).view(-1).long(), -(rows >= 0).view(-1).int())
    s["tables"][seqs.long()] = -1
    s["lengths"][seqs.long()] = 0


def _fork(s, src, dst):
    rows = s["tables"][src.long()]
    s["refs"].index_add_(0, rows.clamp_min(0).view(-1).long(), (rows >= 0).view(-1).int())
    s["tables"][dst.long()] = rows
    s["lengths"][dst.long()] = s["lengths"][src.long()]


def _extend(s, seqs, counts):
    """Lowest free pages first, sequence by sequence; a shared last page is copied, unless all who hold it extend it
    now: then the last of them keeps it."""
    T, P, n = s["case"]["page"], s["refs"].numel(), seqs.numel()
    rows = seqs.long()
    lens, grow = s["lengths"][rows].long(), counts.long()
    have, need = (lens + T - 1) // T, (lens + grow + T - 1) // T
    writes = (lens % T > 0) & (grow > 0)
    last = torch.where(writes, s["tables"][rows, (lens // T).clamp_max(s["tables"].shape[1] - 1)].long(), 0)
    i = torch.arange(n, device=DEVICE)
    writers = torch.zeros(P, dtype=torch.int64, device=DEVICE).index_add_(0, last, writes.long())
    keeper = torch.full((P,), -1, dtype=torch.int64, device=DEVICE).index_reduce_(0, last, torch.where(writes, i, -1), "amax")
    refs = s["refs"].long()
    copy = writes & ((refs[last] > writers[last]) | (keeper[last] != i))
    take = need - have + copy.long()
    at = torch.cumsum(take, 0) - take
    free = (refs == 0).nonzero().view(-1)
    src, dst = last[copy], free[at[copy]]
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        s[name][:, dst] = s[name][:, src]
    s["refs"].index_add_(0, src, -torch.ones_like(src, dtype=torch.int32))
    s["tables"][rows[copy], lens[copy] // T] = dst.int()
    fresh = torch.repeat_interleave(i, need - have)
    nth = torch.arange(fresh.numel(), device=DEVICE) - (torch.cumsum(need - have, 0) - (need - have))[fresh]
    s["tables"][rows[fresh], have[fresh] + nth] = free[at[fresh] + copy.long()[fresh] + nth].int()
    s["refs"][free[: int(take.sum())]] = 1
    s["lengths"][rows] = (lens + grow).int()


def _compact(s):
    """The live pages behind the first `live` ones move, in order, into the holes before it."""
    held = s["refs"] > 0
    live = int(held.sum())
    p = torch.arange(held.numel(), device=DEVICE)
    src, dst = p[held & (p >= live)], p[~held & (p < live)]
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        s[name][:, dst] = s[name][:, src]
    to = p.clone()
    to[src] = dst
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["tables"].copy_(torch.where(s["tables"] >= 0, to[s["tables"].clamp_min(0).long()].int(), s["tables"]))


# ------------------------------------------------------------ in 64 bits

def _exp64(e):
    """2^e of whole e (a device's pow() may be off by a bit, and a tie then goes the other way)."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _tokens64(s, i, name, count):
    """The first `count` tokens of sequence i's keys or values, [tokens, kv, D] f64."""
    T = s["case"]["page"]
    pages = s["tables"][int(s["seqs"][i]), : _cdiv(count, T)].long()
    x, b = s[name + "_codes"][0][pages].double(), s[name + "_scales"][0][pages].double()
    if name == "v":
        x = x.transpose(2, 3)
    x = x * _exp64(b - 127)[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:count]


def _turn64(x, table, pos):
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h], x[..., h:]) * torch.complex(table[pos, :h].double(), table[pos, h:].double())[:, None]
    return torch.cat((z.real, z.imag), -1)


def exact(c, seed):
    if c["kind"] in ("fork", "compact"):
        return None  # whole numbers alone
    s = prepare(c, seed)
    lens, new, D, kv = s["lens"], s["new"], c["dim"], c["kv"]
    if c["kind"] == "attend":
        out, at, G = [], 0, c["heads"] // kv
        for i, (L, n) in enumerate(zip(lens, new)):
            pos = torch.arange(L - n, L, device=DEVICE)
            q = s["q"][at:at + n].double()
            at += n
            if s["rope"] is not None:
                q = _turn64(q, s["rope"], pos)
            k, v = _tokens64(s, i, "k", L), _tokens64(s, i, "v", L)
            j = torch.arange(L, device=DEVICE)
            o = torch.empty_like(q)
            for h in range(c["heads"]):
                x = (q[:, h] @ k[:, h // G].T) / math.sqrt(D)
                if c["causal"]:
                    x = torch.where(j > pos[:, None], -math.inf, x)
                    if c["window"]:
                        x = torch.where(j <= pos[:, None] - c["window"], -math.inf, x)
                o[:, h] = torch.softmax(x, -1) @ v[:, h // G]
            out.append(o)
        return torch.cat(out)
    got, at, T = {"k": [], "v": []}, 0, c["page"]
    for i, (L, n, back) in enumerate(zip(lens, new, s["back"])):
        pos = torch.arange(L - n, L, device=DEVICE)
        for name in ("k", "v"):
            x = s[name][at:at + n].double()
            if name == "k" and s["rope"] is not None:
                x = _turn64(x, s["rope"], pos)
            before = _tokens64(s, i, name, L - n)
            both = torch.cat((before, x))
            whole = both.new_zeros(_cdiv(L, T) * T, kv, D)
            whole[:L] = both
            part = torch.arange(whole.shape[0], device=DEVICE)
            fresh = torch.where(((part >= L - n) & (part < L))[:, None, None], whole, 0).view(-1, T, kv, D)
            part, up = torch.frexp(fresh.abs().amax((1, 3)) / 127)  # [pages, kv]: the power of two that is not below
            e = torch.where(part == 0, -126, up - (part == 0.5).int()).clamp(-126, 127).double()
            pages = s["tables"][int(s["seqs"][i]), : e.shape[0]].long()
            was = s[name + "_scales"][0][pages].double() - 127
            begun = (torch.arange(e.shape[0], device=DEVICE) * T < L - n)[:, None]
            e = torch.where(begun, torch.maximum(e, was), e)
            step = _exp64(e)[:, None, :, None]
            y = (torch.round(whole.view(-1, T, kv, D) / step) * step).view(-1, kv, D)
            got[name].append(y[L - back:L])
        at += n
    return torch.cat(got["k"]), torch.cat(got["v"])
