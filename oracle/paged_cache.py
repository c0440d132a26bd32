"""64-bit restatement of the 8-bit paged KV cache (TEST INFRASTRUCTURE ONLY).

Codes are kept as the numbers they stand for (float64), one loop per token or
page: slow and plain.  Rules are the ones the product documents: power-of-two
scales that only grow while a page fills, finite codes, lowest free pages first.
"""

from __future__ import annotations

import numpy as np

MIN_EXP = -100
# the largest exponent, and the largest code there: code * scale stays below 2^128
MAX_EXP = {"e4m3": 120, "int8": 121}
TOP_CODE = {"e4m3": 240.0, "int8": 127.0}
EXHAUSTED, ROW_FULL, BAD_INDEX = 1, 2, 4


def to_grid(x: np.ndarray, fmt: str, exp: int = 0) -> np.ndarray:
    """Nearest code (ties to even), saturating (under the scale 2^exp); NaN becomes 0."""
    x = np.where(np.isnan(x), 0.0, x)
    if fmt == "int8":
        return np.clip(np.rint(np.clip(x, -1e6, 1e6)), -127, 127)
    top = TOP_CODE[fmt] if exp == MAX_EXP[fmt] else 448.0
    x = np.clip(x, -top, top)
    _, e = np.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(x / step) * step


def block_exponent(x: np.ndarray, fmt: str) -> int:
    """Least e with max|x| <= top * 2^e over the finite values."""
    top = 127.0 if fmt == "int8" else 448.0
    finite = np.abs(x[np.isfinite(x)])
    largest = finite.max() if finite.size else 0.0
    e = MIN_EXP
    while e < MAX_EXP[fmt] and largest > top * 2.0 ** e:
        e += 1
    return e


class PagedCache:
    def __init__(self, fmt, layers, pages, heads, page, d, slots, per_slot):
        self.fmt, self.page = fmt, page
        shape = (layers, pages, heads, page, d)
        self.k, self.v = np.zeros(shape), np.zeros(shape)
        self.k_scale, self.v_scale = np.ones(shape[:3]), np.ones(shape[:3])
        self.tables = np.full((slots, per_slot), -1, dtype=np.int64)
        self.lengths = np.zeros(slots, dtype=np.int64)
        self.refcounts = np.zeros(pages, dtype=np.int64)
        self.status = 0

    # -- rows ---------------------------------------------------------------------
    def _row(self, slot, start, end, tokens, max_end=1 << 40):
        if end <= start:
            return 0  # asks for nothing
        if (0 <= slot < len(self.lengths) and 0 <= start and end <= max_end
                and (end - 1) // self.page < self.tables.shape[1]):
            return min(end - start, tokens)
        self.status |= BAD_INDEX
        return 0

    def _page(self, slot, pos):
        p = self.tables[slot, pos // self.page]
        return p if 0 <= p < len(self.refcounts) else -1

    # -- storage --------------------------------------------------------------------
    def append(self, layer, k, v, slots, starts, ends):
        for b, slot in enumerate(slots):
            n = self._row(slot, starts[b], ends[b], k.shape[1])
            if not n:
                continue
            if any(slots[j] == slot and ends[j] > starts[j] for j in range(b)):
                self.status |= BAD_INDEX
                continue
            for first in range(starts[b] // self.page * self.page, starts[b] + n, self.page):
                a, z = max(first, starts[b]), min(first + self.page, starts[b] + n)
                page = self._page(slot, first)
                if page < 0:
                    self.status |= BAD_INDEX
                    continue
                for codes, scales, new in ((self.k, self.k_scale, k), (self.v, self.v_scale, v)):
                    for h in range(codes.shape[2]):
                        x = new[b, a - starts[b]:z - starts[b], h]
                        e = block_exponent(x, self.fmt)
                        if a > first:
                            old = scales[layer, page, h]
                            m, oe = np.frexp(old)
                            e = max(e, min(max(int(oe) - (m == 0.5), MIN_EXP),
                                           MAX_EXP[self.fmt]))
                            held = codes[layer, page, h, :a - first]
                            if old != 2.0 ** e:
                                codes[layer, page, h, :a - first] = to_grid(
                                    held * old / 2.0 ** e, self.fmt, e)
                        codes[layer, page, h, a - first:z - first] = to_grid(
                            x / 2.0 ** e, self.fmt, e)
                        scales[layer, page, h] = 2.0 ** e

    def read(self, layer, slots, starts, ends, max_tokens):
        shape = (len(slots), max_tokens, self.k.shape[2], self.k.shape[4])
        k, v = np.zeros(shape), np.zeros(shape)
        for b, slot in enumerate(slots):
            for i in range(self._row(slot, starts[b], ends[b], max_tokens)):
                pos = starts[b] + i
                page = self._page(slot, pos)
                if page >= 0:
                    at = (layer, page, slice(None), pos % self.page)
                    k[b, i] = self.k[at] * self.k_scale[layer, page][:, None]
                    v[b, i] = self.v[at] * self.v_scale[layer, page][:, None]
        return k, v

    def attention(self, layer, q, slots, starts, ends, window=0, max_seqlen_k=1 << 40):
        """(out, lse, spread, grain, size), the last three to state error bounds in:
        spread = sum p |v|, grain = max(p s_v) sum |v8| (s_v, v8: a value's scale and
        code), size = max over visible keys of sum |q k|."""
        rows, tokens, hq, d = q.shape
        group = hq // self.k.shape[2]
        out, spread, grain = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
        lse, size = np.full((rows, hq, tokens), -np.inf), np.zeros((rows, hq, tokens))
        for b, slot in enumerate(slots):
            n = self._row(slot, starts[b], ends[b], tokens, max_seqlen_k)
            for i in range(n):
                pos = starts[b] + i
                lo = max(0, pos - window + 1) if window else 0
                keys = np.arange(lo, pos + 1)
                pages = np.array([self._page(slot, int(x)) for x in keys])
                keys, pages = keys[pages >= 0], pages[pages >= 0]
                if not len(keys):
                    continue
                for h in range(self.k.shape[2]):
                    at = (layer, pages, h, keys % self.page)
                    k = self.k[at] * self.k_scale[layer, pages, h][:, None]
                    v = self.v[at] * self.v_scale[layer, pages, h][:, None]
                    for j in range(h * group, (h + 1) * group):
                        s = k @ q[b, i, j]
                        top = s.max()
                        p = np.exp(s - top)
                        total = p.sum()
                        out[b, i, j] = p @ v / total
                        spread[b, i, j] = p @ np.abs(v) / total
                        grain[b, i, j] = ((p * self.v_scale[layer, pages, h]).max() / total
                                          * np.abs(self.v[at]).sum(0))
                        lse[b, j, i] = top + np.log(total)
                        size[b, j, i] = (np.abs(k) @ np.abs(q[b, i, j])).max()
        return out, lse, spread, grain, size

    # -- pages ------------------------------------------------------------------------
    def _slot(self, s):
        return 0 <= s < len(self.lengths)

    def _refs(self, s, i):
        """Tables that list slot s's i-th page; 0 where it has none."""
        p = self.tables[s, i]
        return self.refcounts[p] if 0 <= p < len(self.refcounts) else 0

    def extend(self, slots, counts):
        starts, ends = np.zeros(len(slots), int), np.zeros(len(slots), int)
        free = [p for p in range(len(self.refcounts)) if self.refcounts[p] == 0]
        for b, (s, n) in enumerate(zip(slots, counts)):
            if self._slot(s):
                starts[b] = ends[b] = self.lengths[s]
                if b and s in slots[:b]:  # the device reads every length before it writes
                    first = list(slots).index(s)
                    starts[b] = ends[b] = starts[first]
            if not self._slot(s) or s in list(slots[:b]) or n < 0:
                self.status |= BAD_INDEX
                continue
            new = self.lengths[s] + n
            if new > self.tables.shape[1] * self.page:
                self.status |= ROW_FULL
                continue
            # pages behind a length that was lowered are used again
            have, want = -(-self.lengths[s] // self.page), -(-new // self.page)
            if self.lengths[s] % self.page and n and self._refs(s, have - 1) > 1:
                self.status |= BAD_INDEX
                continue
            while have < want and self._refs(s, have) == 1:
                have += 1
            if have < want and self._refs(s, have) > 1:
                self.status |= BAD_INDEX
                continue
            if want - have > len(free):
                self.status |= EXHAUSTED
                continue
            for j in range(want - have):
                page = free.pop(0)
                self.tables[s, have + j] = page
                self.refcounts[page] = 1
            self.lengths[s] = ends[b] = new
        return starts, ends

    def _move(self, src, dst):
        for x in (self.k, self.v, self.k_scale, self.v_scale):
            x[:, dst] = x[:, src]

    def fork(self, parents, children):
        before = self.lengths.copy()
        free = [p for p in range(len(self.refcounts)) if self.refcounts[p] == 0]
        wanted = 0
        for b, (s, c) in enumerate(zip(parents, children)):
            if (not self._slot(s) or not self._slot(c) or c in list(children[:b])
                    or before[c] != 0 or self.tables[c, 0] >= 0):
                self.status |= BAD_INDEX
                continue
            whole, part = divmod(int(before[s]), self.page)
            if part and self._page(s, int(before[s])) < 0:  # trimmed, then lowered
                self.status |= BAD_INDEX
                continue
            if part:
                wanted += 1
                if wanted > len(free):
                    self.status |= EXHAUSTED
                    continue
                new = free[wanted - 1]
                self._move(self.tables[s, whole], new)
                self.tables[c, whole] = new
                self.refcounts[new] = 1
            for j in range(whole):
                self.tables[c, j] = self.tables[s, j]
                if self.tables[s, j] >= 0:
                    self.refcounts[self.tables[s, j]] += 1
            self.lengths[c] = before[s]

    def free(self, slots, window=0):
        for s in slots:
            if not self._slot(s):
                self.status |= BAD_INDEX
                continue
            upto = self.tables.shape[1]
            if window:
                upto = min(-(-self.lengths[s] // self.page),
                           max(0, self.lengths[s] - window + 1) // self.page)
            for j in range(upto):
                if self.tables[s, j] >= 0:
                    self.refcounts[self.tables[s, j]] -= 1
                    self.tables[s, j] = -1
            if not window:
                self.lengths[s] = 0

    def compact(self):
        live = int((self.refcounts > 0).sum())
        holes = [p for p in range(live) if self.refcounts[p] == 0]
        movers = [p for p in range(live, len(self.refcounts)) if self.refcounts[p] > 0]
        for src, dst in zip(movers, holes):
            self._move(src, dst)
            self.tables[self.tables == src] = dst
            self.refcounts[dst], self.refcounts[src] = self.refcounts[src], 0

    def copy_pages(self, src, dst):
        ok = lambda p: 0 <= p < len(self.refcounts)
        for i, (s, d) in enumerate(zip(src, dst)):
            if not ok(s) or not ok(d) or d in list(dst[:i]) or d in list(src):
                self.status |= BAD_INDEX
                continue
            self._move(s, d)
