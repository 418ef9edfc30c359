"""What a step of token generation does between its linears and behind them, in 64 bits: norms, positions turned into
heads, groups of sequences that share pages, and the choice of the next token. Plain numpy, rows by loops."""
from __future__ import annotations

import math

import numpy as np

from . import hadamard


def rms_norm(h, weight=None, eps=1e-6):
    """h [M, K] (what the residual stream holds) -> y."""
    h = np.asarray(h, dtype=np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * np.asarray(weight, dtype=np.float64)


def quantize(y, block=0):
    """(z, scale): the rotated rows and max |z| / 127 (at least 1e-10); codes are rne(z / scale)."""
    z = np.asarray(y, dtype=np.float64)
    if block:
        z = hadamard.rotate_matmul64(z, block)
    return z, np.maximum(np.abs(z).max(-1) / 127, 1e-10)


def frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=4096, fast=32.0, slow=1.0):
    """(radians a position of pair i, size)."""
    i = np.arange(dim // 2, dtype=np.float64)
    f = base ** (-2 * i / dim)
    if scaling is None:
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    turns = np.array([fast, slow])
    at = dim / 2 * np.log(original / (2 * np.pi * turns)) / np.log(base)
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
    part = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
    return f * (part / factor + 1 - part), 0.1 * math.log(max(factor, 1)) + 1


def turn(x, pos, f, size=1.0, interleaved=False):
    """x [..., D] at positions pos (of x's first dimension), its first 2 len(f) values as pairs turned by pos f."""
    x, n = np.array(x, dtype=np.float64), len(f)
    a, b = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    angle = np.asarray(pos, dtype=np.float64).reshape(-1, *[1] * (x.ndim - 1)) * f
    c, s = size * np.cos(angle), size * np.sin(angle)
    x[..., a], x[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return x


def shared(table, lens, page):
    """(groups, start): groups [(tokens, members)] of sequences with the same first pages, in the order of their first
    sequences; start[b]: what sequence b shares."""
    by_first = {}
    for b, n in enumerate(lens):
        if n > 0 and len(table[b]) and table[b][0] >= 0:
            by_first.setdefault(int(table[b][0]), []).append(b)
    groups, start = [], [0] * len(lens)
    for members in by_first.values():
        if len(members) < 2:
            continue
        lead, tokens = members[0], 1 << 62
        for b in members:
            most = min(lens[b], lens[lead])
            same = 0
            while same < min(-(-most // page), len(table[b])) and table[b][same] >= 0 and table[b][same] == table[lead][same]:
                same += 1
            tokens = min(tokens, same * page, most)
        if tokens > 0:
            groups.append((tokens, members))
            for b in members:
                start[b] = tokens
    return groups, start


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of one row of logits."""
    x = np.asarray(row, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temperature) if np.isfinite(x.max()) else 0.0)
    kept = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        sums = np.cumsum(w[kept])
        kept = kept[:1 + int(np.searchsorted(sums, top_p * sums[-1], side="left"))]
    kept = np.sort(kept[(w[kept] >= min_p) | (x[kept] == x.max())])
    sums = np.cumsum(w[kept])
    at = int(np.searchsorted(sums, max(0.0, u if u == u else 0.0) * sums[-1], side="right"))
    return int(kept[min(at, np.flatnonzero(w[kept])[-1])])
