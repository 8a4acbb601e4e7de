"""What the FP8 KV cache's operators are to do, in plain Python and float64, one page and one row after the other."""

from __future__ import annotations

import math
import random

import torch

E4M3 = torch.float8_e4m3fn


def grid(v):
    """float64 -> the nearest e4m3 value, ties to even; past 464, and for what is not finite, NaN (448's neighbour is NaN's code)."""
    exponent = torch.frexp(v).exponent.long()
    step = (((exponent - 4).clamp_min(-9) + 1023) << 52).view(torch.float64)
    r = torch.round(v / step) * step
    return torch.where(v.isfinite() & (v.abs() <= 464.0), r.clamp(-448.0, 448.0), torch.full_like(v, math.nan))


def scale_of(amax: float) -> float:
    """The least power of two in 2^-48 .. 2^48 that takes amax to 448 at most."""
    if amax == 0.0:
        return 2.0 ** -48
    f, e = math.frexp(amax / 448.0)
    return math.ldexp(1.0, max(-48, min(48, e - (f == 0.5))))


def pages_of(n, page):
    return -(-n // page)


class Cache:
    """A cache's state on the CPU: codes as float64 values, tokens first in both K and V."""

    def __init__(self, c):
        self.page = c.page
        self.k = c.k.cpu().double()
        self.v = c.v.cpu().double().transpose(3, 4).contiguous()
        self.ks, self.vs = c.k_scales.cpu().double(), c.v_scales.cpu().double()
        self.refs = c.refs.tolist()

    def same(self, c):
        def eq(a, b):
            return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())

        assert eq(self.ks, c.k_scales.cpu().double()) and eq(self.vs, c.v_scales.cpu().double())
        assert eq(self.k, c.k.cpu().double()) and eq(self.v, c.v.cpu().double().transpose(3, 4).contiguous())
        assert self.refs == c.refs.tolist()

    def append(self, layer, k, v, table, lengths, offsets):
        width = len(table[0]) if table else 0
        for x, codes, scales in ((k.cpu().double(), self.k, self.ks), (v.cpu().double(), self.v, self.vs)):
            for b, row in enumerate(table):
                first, n = (b, 1) if offsets is None else (offsets[b], offsets[b + 1] - offsets[b])
                length = max(0, min(lengths[b], width * self.page))
                at = length - n  # place of the first; those before the start have none
                while at < length:
                    if at < 0:
                        at += 1
                        continue
                    p, slot = row[at // self.page], at % self.page
                    take = min(self.page - slot, length - at)
                    if 0 <= p < codes.shape[1]:
                        src = first + n - (length - at)
                        part = x[src: src + take]
                        for h in range(codes.shape[2]):
                            w = part[:, h]
                            fin = w[w.isfinite()]
                            s = scale_of(float(fin.abs().max()) if fin.numel() else 0.0)
                            if slot:
                                old = float(scales[layer, p, h])
                                s = max(s, old)
                                if s != old:
                                    codes[layer, p, h, :slot] = grid(codes[layer, p, h, :slot] * (old / s))
                            codes[layer, p, h, slot: slot + take] = grid(w / s)
                            scales[layer, p, h] = s
                    at += take

    def rows_of(self, table, lengths):
        return [row[: pages_of(max(0, min(n, len(row) * self.page)), self.page)] for row, n in zip(table, lengths)]

    def count(self, p, by):
        if 0 <= p < len(self.refs):
            self.refs[p] += by

    def copy(self, a, b):
        for x in (self.k, self.v, self.ks, self.vs):
            x[:, b] = x[:, a]

    def fork(self, table, lengths, parents):
        width = len(table[0]) if table else 0
        rows = self.rows_of(table, lengths)
        lens = [max(0, min(n, width * self.page)) for n in lengths]
        parents = [p if 0 <= p < len(rows) else r for r, p in enumerate(parents)]
        for r, p in enumerate(parents):
            if p != r:
                for x in rows[r]:
                    self.count(x, -1)
                for x in rows[p]:
                    self.count(x, 1)
        return [rows[p] + [-1] * (width - len(rows[p])) for p in parents], [lens[p] for p in parents]

    def resize(self, table, lengths, wanted):
        width = len(table[0]) if table else 0
        rows = [list(r) for r in self.rows_of(table, lengths)]
        lens = [max(0, min(n, width * self.page)) for n in lengths]
        wanted = [n if w > width * self.page else max(0, w) for n, w in zip(lens, wanted)]
        for r, w in enumerate(wanted):
            while len(rows[r]) > pages_of(w, self.page):
                self.count(rows[r].pop(), -1)
        free = [p for p, c in enumerate(self.refs) if c <= 0]
        shared = [bool(row) and 0 <= row[-1] < len(self.refs) and self.refs[row[-1]] > 1 for row in rows]
        need = 0
        for r, w in enumerate(wanted):
            if w <= lens[r]:
                lens[r] = w
                continue
            copy = lens[r] % self.page > 0 and shared[r]
            mine = pages_of(w, self.page) - len(rows[r]) + copy
            need += mine
            if mine and need > len(free):
                continue
            take = free[need - mine: need]
            if copy:
                self.copy(rows[r][-1], take[0])
                self.refs[rows[r][-1]] -= 1
                rows[r][-1] = take[0]
                self.refs[take.pop(0)] = 1
            for p in take:
                self.refs[p] = 1
            rows[r] += take
            lens[r] = w
        return [row + [-1] * (width - len(row)) for row in rows], lens, max(0, need - len(free))

    def compact(self, table):
        live = [p for p, c in enumerate(self.refs) if c > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        to = dict(zip([p for p in live if p >= n], holes))
        for a, b in to.items():
            self.copy(a, b)
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.refs = [max(0, c) for c in self.refs]
        return [[to.get(p, p) for p in row] for row in table], n


def attend(cache, layer, q, table, lengths, offsets, scale, window):
    """(out, bound, lse) in float64 on the cache's device: the definition, and how far a right kernel may be from it.

    The bound: scores are float32 sums of dim exact products (dim 2^-24 of the sum of their sizes, twice over for p and its sum), 2^e and
    its argument have 2^-21 together, p is rounded to fp16 (2^-11; 2^-35 of the largest where that is subnormal), sums of n terms have
    n 2^-24 and their joining 2^-20; the result is rounded to its type."""
    tokens, heads, dim = q.shape
    dev = q.device
    group = heads // cache.kv_heads
    half = torch.finfo(q.dtype).eps / 2
    out, bound = (torch.zeros(tokens, heads, dim, dtype=torch.float64, device=dev) for _ in range(2))
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device=dev)
    kd = cache.k[layer].double() * cache.k_scales[layer].double()[..., None, None]
    vd = cache.v[layer].double() * cache.v_scales[layer].double()[..., None, None]
    width = len(table[0]) if table else 0
    for b, row in enumerate(table):
        first, n = (b, 1) if offsets is None else (offsets[b], offsets[b + 1] - offsets[b])
        length = max(0, min(lengths[b], width * cache.page))
        used = pages_of(length, cache.page)
        ok = torch.tensor([0 <= p < cache.pages for p in row[:used]], dtype=torch.bool, device=dev).repeat_interleave(cache.page)[:length]
        idx = torch.tensor([p if 0 <= p < cache.pages else 0 for p in row[:used]], dtype=torch.long, device=dev)
        for i in range(n):
            pos = length - n + i
            lo = max(0, pos + 1 - window) if window else 0
            see = torch.arange(lo, max(lo, pos + 1), device=dev)
            see = see[ok[see]]
            if see.numel() == 0:
                continue
            for h in range(cache.kv_heads):
                k = kd[idx, h].reshape(-1, dim)[see]
                v = vd[idx, h].transpose(1, 2).reshape(-1, dim)[see]
                qq = q[first + i, h * group: (h + 1) * group].double()
                s = qq @ k.T * scale
                p = torch.softmax(s, -1)
                o = p @ v
                err = 2 * dim * 2.0 ** -24 * (qq.abs() @ k.abs().T).amax(-1, keepdim=True) * abs(scale) + 2.0 ** -21 * (1 + s.abs().amax(-1, keepdim=True))
                rel = 2.0 ** -11 + 2 * err + see.numel() * 2.0 ** -23 + 2.0 ** -19
                r = slice(h * group, (h + 1) * group)
                out[first + i, r] = o
                bound[first + i, r] = half * o.abs() + rel * (p @ v.abs()) + 2.0 ** -35 * see.numel() * v.abs().amax() + 2.0 ** -24 * half
                lse[first + i, r] = torch.logsumexp(s, -1)
    return out, bound, lse


def spread_table(lengths, page, width, pool, seed):
    """Rows of distinct pages, scattered; -1 behind them."""
    places = list(range(pool))
    random.Random(seed).shuffle(places)
    table = []
    for n in lengths:
        k = pages_of(n, page)
        table.append(places[:k] + [-1] * (width - k))
        del places[:k]
    return table
