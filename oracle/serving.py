"""Token generation in 64 bits: attention over a paged cache, the cache's bookkeeping, and linears with 4-bit
weights and floating-point activations. Plain loops over sequences, heads and pages in numpy."""
from __future__ import annotations

import math

import numpy as np

from . import hadamard


def attention(q, k, v, table, lens, cu=None, scale=None, window=None, sinks=0):
    """q [T, Hq, D]; k, v [pages, H, page_size, D]; table [B, width] (entries that are no page hold nothing); lens [B];
    cu [B + 1] or None. Returns (out, weight, reach): out [T, Hq, D]; weight[t, hq, d] = sum_j p_j |v_j,d|, what an
    error relative to the probabilities moves the output by; reach[t, hq] = max_j sum_d |q_d k_j,d| * scale."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    t_all, hq, d = q.shape
    pages, h, ps, _ = k.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((t_all, hq))
    for b in range(len(lens)):
        first, last = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        place = [(j, int(table[b][j // ps])) for j in range(min(int(lens[b]), len(table[b]) * ps))]
        place = [(j, p) for j, p in place if 0 <= p < pages]
        js = np.array([j for j, _ in place], dtype=np.int64)
        ps_, slots = np.array([p for _, p in place], dtype=np.int64), js % ps
        for t in range(first, last):
            pos = int(lens[b]) - last + t
            see = js <= pos
            if window is not None:
                see &= (js > pos - window) | (js < sinks)
            if not see.any():
                continue
            for g in range(hq):
                kk, vv = k[ps_[see], g // (hq // h), slots[see]], v[ps_[see], g // (hq // h), slots[see]]
                with np.errstate(all="ignore"):
                    s = kk @ q[t, g] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[t, g], weight[t, g] = p @ vv, p @ np.abs(vv)
                    reach[t, g] = (np.abs(kk) @ np.abs(q[t, g])).max() * abs(scale)
    return out, weight, reach


class Pages:
    """The bookkeeping of a paged cache: table, lens, refs as lists, `moves` the page copies of the last call."""

    def __init__(self, table, lens, refs, page_size):
        self.table = [list(map(int, r)) for r in table]
        self.lens, self.refs, self.ps = list(map(int, lens)), list(map(int, refs)), page_size
        self.moves = []

    def _count(self, n):
        return -(-n // self.ps)

    def _free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def fork(self, src, dst):
        """The status of kv_fork; unless it is 0, nothing has changed."""
        self.moves, rows, width, pages = [], len(self.table), len(self.table[0]), len(self.refs)
        if any(not 0 <= r < rows for r in [*src, *dst]) or len(set(dst)) != len(dst) or set(src) & set(dst):
            return -1
        if any(self.lens[d] for d in dst) or any(self._count(self.lens[s]) > width for s in src):
            return -1
        if any(not 0 <= p < pages for s in src for p in self.table[s][: self._count(self.lens[s])]):
            return -1
        free = self._free()
        need = sum(self.lens[s] % self.ps > 0 for s in src)
        if need > len(free):
            return need - len(free)
        for s, d in zip(src, dst):
            full, part = divmod(self.lens[s], self.ps)
            self.table[d] = self.table[s][:full] + [-1] * (width - full)
            for p in self.table[s][:full]:
                self.refs[p] += 1
            if part:
                p = free.pop(0)
                self.table[d][full], self.refs[p] = p, 1
                self.moves.append((self.table[s][full], p))
            self.lens[d] = self.lens[s]
        return 0

    def grow(self, rows, counts):
        width = len(self.table[0])
        if any(not 0 <= r < len(self.table) for r in rows) or len(set(rows)) != len(rows) or min(counts, default=0) < 0:
            return -1
        if any(self.lens[r] + c > width * self.ps for r, c in zip(rows, counts)):
            return -1
        free = self._free()
        need = sum(self._count(self.lens[r] + c) - self._count(self.lens[r]) for r, c in zip(rows, counts))
        if need > len(free):
            return need - len(free)
        for r, c in zip(rows, counts):
            for j in range(self._count(self.lens[r]), self._count(self.lens[r] + c)):
                self.table[r][j] = free.pop(0)
                self.refs[self.table[r][j]] = 1
            self.lens[r] += c
        return 0

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.table):
                for p in self.table[r]:
                    if 0 <= p < len(self.refs):
                        self.refs[p] -= 1
                self.table[r], self.lens[r] = [-1] * len(self.table[r]), 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        self.moves = list(zip([p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]))
        to = dict(self.moves)
        for s, d in self.moves:
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return n


def w4_weight(qweight, scales, zeros, group):
    """The weight [N, K] that packed 4-bit codes stand for: zeros None (signed codes), packed uint4 or floating."""
    qweight = np.asarray(qweight, dtype=np.uint8)
    code = np.empty((qweight.shape[0], 2 * qweight.shape[1]))
    code[:, 0::2], code[:, 1::2] = qweight & 15, qweight >> 4
    s = np.repeat(np.asarray(scales, dtype=np.float64), group, axis=1)
    if zeros is None:
        return np.where(code > 7, code - 16, code) * s
    zeros = np.asarray(zeros)
    if zeros.dtype == np.uint8:
        z = np.empty((zeros.shape[0], 2 * zeros.shape[1]))
        z[:, 0::2], z[:, 1::2] = zeros & 15, zeros >> 4
        return (code - np.repeat(z, group, axis=1)[:, : code.shape[1]]) * s
    return code * s + np.repeat(zeros.astype(np.float64), group, axis=1)


def w4a16_linear(x, qweight, scales, zeros=None, bias=None, group=64, block=0):
    """(y, spread): spread[m, n] = sum_k |x'_k w_nk|, what a relative error of the products moves y by; with zeros,
    of the parts that are summed apart (codes, zero-points)."""
    x = np.asarray(x, dtype=np.float64)
    if block:
        x = (x.reshape(-1, block) @ hadamard.hadamard(block)).reshape(x.shape)
    w = w4_weight(qweight, scales, zeros, group)
    y = x @ w.T
    big = np.abs(w) + np.repeat(np.abs(np.asarray(scales, dtype=np.float64)), group, axis=1) * 24
    if bias is not None:
        y = y + np.asarray(bias, dtype=np.float64)
    return y, np.abs(x) @ big.T
