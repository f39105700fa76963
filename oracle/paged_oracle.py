"""Plain restatement of the paged 8-bit key/value cache (include/eredu_kv.h), in
numpy and 64 bits, one token, page and sequence at a time."""
import math

import numpy as np


class Paged:
    """codes k [layers, pages, heads, T, D], v [layers, pages, heads, D, T] (int64 here),
    scale bytes, tables, lengths, refs: the state of eq_kv_cache."""

    def __init__(self, layers, pages, heads, D, seqs, width, T):
        self.T, self.D, self.heads, self.layers, self.width = T, D, heads, layers, width
        self.k = np.zeros((layers, pages, heads, T, D), np.int64)
        self.v = np.zeros((layers, pages, heads, D, T), np.int64)
        self.ks = np.ones((layers, pages, heads), np.int64)
        self.vs = np.ones((layers, pages, heads), np.int64)
        self.tables = np.full((seqs, width), -1, np.int64)
        self.lengths = np.zeros(seqs, np.int64)
        self.refs = np.zeros(pages, np.int64)
        self.missing = 0

    def page(self, seq, index):
        if not 0 <= index < self.width:
            return -1
        p = self.tables[seq, index]
        return int(p) if 0 <= p < len(self.refs) else -1

    # ------------------------------------------------------------ pages

    def _take(self):
        free = np.nonzero(self.refs <= 0)[0]
        free = [p for p in free if p not in self._taken]
        if not free:
            self.missing += 1
            return -1
        self._taken.add(free[0])
        return int(free[0])

    def extend(self, seqs, counts):
        T = self.T
        last = {s: i for i, s in enumerate(seqs)}
        todo = [(i, s, n) for i, (s, n) in enumerate(zip(seqs, counts)) if last[s] == i and 0 <= s < len(self.lengths) and n > 0]
        opened = {}
        for i, s, _ in todo:
            if self.lengths[s] % T:
                p = self.page(s, self.lengths[s] // T)
                if p >= 0:
                    opened.setdefault(p, []).append(i)
        before, self._taken = self.refs.copy(), set()
        copies = []
        for i, s, n in todo:
            L = int(self.lengths[s])
            p = self.page(s, L // T) if L % T else -1
            if p >= 0 and (before[p] > len(opened[p]) or opened[p][-1] != i):
                q = self._take()
                if q >= 0:
                    copies.append((p, q))
                    self.refs[q] = 1
                self.refs[p] -= 1
                self.tables[s, L // T] = q
            for w in range(-(-L // T), -(-(L + n) // T)):
                if w >= self.width:
                    self.missing += 1
                    continue
                q = self._take()
                if q >= 0:
                    self.refs[q] = 1
                self.tables[s, w] = q
            self.lengths[s] = L + n
        self._copy(copies)

    def _copy(self, pairs):
        for a, b in pairs:
            for x in (self.k, self.v, self.ks, self.vs):
                x[:, b] = x[:, a]

    def fork(self, src, dst):
        last = {d: i for i, d in enumerate(dst)}
        ok = range(len(self.lengths))
        rows = [(d, self.tables[s].copy(), self.lengths[s]) for i, (s, d) in enumerate(zip(src, dst))
                if last[d] == i and s in ok and d in ok]
        for _, row, _ in rows:
            for p in row[row >= 0]:
                self.refs[p] += 1
        for d, row, n in rows:
            for p in self.tables[d][self.tables[d] >= 0]:
                self.refs[p] -= 1
            self.tables[d], self.lengths[d] = row, n

    def shrink(self, seqs, counts):
        last = {s: i for i, s in enumerate(seqs)}
        for i, (s, n) in enumerate(zip(seqs, counts)):
            if last[s] != i or not 0 <= s < len(self.lengths):
                continue
            self.lengths[s] -= min(max(n, 0), self.lengths[s])
            behind = self.tables[s, -(-self.lengths[s] // self.T):]
            for p in behind[behind >= 0]:
                self.refs[p] -= 1
            behind[...] = -1

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lengths):
                for p in self.tables[s][self.tables[s] >= 0]:
                    self.refs[p] -= 1
                self.tables[s], self.lengths[s] = -1, 0

    def compact(self):
        live = int((self.refs > 0).sum())
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(live) if self.refs[p] <= 0]
        to = dict(zip(movers, holes))
        self._copy(to.items())
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        for x in np.nditer(self.tables, op_flags=["readwrite"]):
            x[...] = to.get(int(x), int(x))

    # ------------------------------------------------------------ tokens

    @staticmethod
    def turn(x, rot):
        h = x.shape[-1] // 2
        a, b, c, s = x[..., :h], x[..., h:], rot[:h], rot[h:]
        return np.concatenate((a * c - b * s, b * c + a * s), -1)

    @staticmethod
    def byte(most):
        if not np.isfinite(most):
            return 255
        b = 1
        while b < 254 and most > 127 * 2.0 ** (b - 127):
            b += 1
        return b

    @staticmethod
    def value(codes, byte):
        return codes * (math.nan if byte == 255 else 2.0 ** (int(byte) - 127))

    def append(self, layer, k, v, seqs, counts, rope=None):
        """k, v [rows, heads, D] f64; rope [positions, D] or None."""
        T, row = self.T, 0
        last = {s: i for i, s in enumerate(seqs)}
        for i, (s, n) in enumerate(zip(seqs, counts)):
            rows = range(row, row + n)
            row += n
            if last[s] != i or not 0 <= s < len(self.lengths):
                continue
            L = int(self.lengths[s])
            pages = {}
            for j, r in enumerate(rows):
                pos = L - n + j
                p = self.page(s, pos // T) if pos >= 0 else -1
                if p >= 0:
                    pages.setdefault(p, []).append((pos % T, r, pos))
            for p, tokens in pages.items():
                for h in range(self.heads):
                    for codes, bytes_, x, turned in ((self.k, self.ks, k, True), (self.v, self.vs, v, False)):
                        new = [self.turn(x[r, h], rope[pos]) if turned and rope is not None else x[r, h]
                               for _, r, pos in tokens]
                        at = tokens[0][0]
                        was = int(bytes_[layer, p, h]) if at else 0
                        now = max(max(self.byte(np.abs(y).max()) if np.isfinite(y).all() else 255 for y in new), was)
                        bytes_[layer, p, h] = now
                        page = codes[layer, p, h] if turned else codes[layer, p, h].T
                        if now == 255:
                            for off, _, _ in tokens:
                                page[off] = 0
                            continue
                        if at and was < now:
                            page[:at] = np.rint(page[:at] * 2.0 ** (was - now))
                        for (off, _, _), y in zip(tokens, new):
                            page[off] = np.rint(y * 2.0 ** (127 - now))

    def token(self, layer, s, pos, h):
        p = self.page(s, pos // self.T) if pos >= 0 else -1
        if p < 0:
            return None
        o = pos % self.T
        return (self.value(self.k[layer, p, h, o], self.ks[layer, p, h]),
                self.value(self.v[layer, p, h, :, o], self.vs[layer, p, h]))

    def read(self, layer, seqs, counts):
        rows = []
        for s, n in zip(seqs, counts):
            L = int(self.lengths[s]) if 0 <= s < len(self.lengths) else 0
            for j in range(n):
                t = [self.token(layer, s, L - n + j, h) if L else None for h in range(self.heads)]
                rows.append([(np.zeros(self.D), np.zeros(self.D)) if x is None else x for x in t])
        a = np.array(rows)
        return (a[:, :, 0], a[:, :, 1]) if rows else (np.zeros((0, self.heads, self.D)),) * 2

    def attention(self, layer, q, seqs, counts, scale, causal=True, window=0, rope=None):
        """q [rows, n_heads, D] f64 -> (out, what its errors are relative to): sums of w |v|, the
        largest score error of a unit error in q, the largest |score|, the number of tokens."""
        rows, H, D = q.shape
        out, mag, unit, top = np.zeros((rows, H, D)), np.zeros((rows, H, D)), np.zeros((rows, H, 1)), np.zeros((rows, H, 1))
        row = 0
        for s, n in zip(seqs, counts):
            L = int(self.lengths[s]) if 0 <= s < len(self.lengths) else 0
            toks = {}
            for h in range(self.heads):
                have = [(j, self.token(layer, s, j, h)) for j in range(min(L, self.width * self.T))]
                have = [(j, t) for j, t in have if t is not None]
                toks[h] = (np.array([j for j, _ in have]), np.array([t[0] for _, t in have]), np.array([t[1] for _, t in have]))
            for i in range(n):
                pos = L - n + i
                for h in range(H):
                    j, k, v = toks[h // (H // self.heads)]
                    x = q[row + i, h]
                    if rope is not None and pos >= 0:
                        x = self.turn(x, rope[pos])
                    if len(j):
                        see = (j <= pos if causal else np.ones(len(j), bool)) & (j > pos - window if window else True)
                        j, k, v = j[see], k[see], v[see]
                    if not len(j):
                        continue
                    bad = np.isnan(k).any(1) | np.isnan(v).any(1)
                    if bad.any() or not np.isfinite(x).all():
                        out[row + i, h] = math.nan
                        continue
                    sc = k @ x * scale
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    out[row + i, h], mag[row + i, h] = w @ v, w @ np.abs(v)
                    unit[row + i, h] = scale * np.abs(k).sum(1).max() * np.abs(x).max()
                    top[row + i, h] = np.abs(sc).max()
            row += n
        return out, mag, unit, top
