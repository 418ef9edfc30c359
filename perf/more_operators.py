"""Performance cases of what a step of token generation does around its linears: norms with the residual's addition,
new tokens turned by their positions into the paged cache, attention of sequences that share a long beginning, and the
choice of the next token.

Four operators, as a program that generates tokens with quantized weights calls them:

  norm     h = x + residual and its root-mean-square norm, in x's type or, rotated by Hadamard blocks where the
           linear's weights ask for it, as int8 codes with a scale per token
  append   queries and keys of new tokens turned by their positions (pairs as halves or side by side, all of the
           head or its first part, frequencies scaled for long contexts), keys and values into their sequences' pages
  shared   attention of one new token per sequence, in every layer, where groups of sequences hold the same pages
           up to some length: alternatives of one prompt, questions about one document
  sample   the next token of every row of logits for a given random number: temperature, the k likeliest, the
           likeliest of a share of the mass, those of a share of the best one's probability

Sequence lengths belong to the case (`lens_seed`); values and the pages' places come from the seed. Codes of 8 bits are
returned as the values that they stand for, in bf16.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
_ck = None
_rotary: dict = {}      # the handles of position rotations that a program makes once for its model


def _framework():
    global _ck
    if _ck is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfy-quant-bench_amd"))
        import kitchen_amd

        _ck = kitchen_amd
    return _ck


# ------------------------------------------------------------------------------------------------ cases

def _named(case, name):
    return dict(case, name=name) if name else case


def _norm(name, m, k, dtype, residual=True, weight=True, bits=16, h=0):
    return _named({"op": "norm", "m": m, "k": k, "dtype": dtype, "residual": residual, "weight": weight, "bits": bits, "h": h}, name)


def _append(name, seqs, heads, kv_heads, dim, page, dtype, kv, lo, hi, q_lo, q_hi, lens_seed=1, turn=0, interleaved=False,
            base=10000.0, scaling="none", factor=1.0, original=4096, empty=0):
    """`seqs` sequences of q_lo .. q_hi new tokens behind lo .. hi earlier ones; `empty` of them hold nothing. turn: how
    much of the head is turned (0: all of it)."""
    return _named({"op": "append", "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
                   "kv": kv, "lo": lo, "hi": hi, "q_lo": q_lo, "q_hi": q_hi, "lens_seed": lens_seed, "turn": turn or dim,
                   "interleaved": interleaved, "base": base, "scaling": scaling, "factor": factor, "original": original,
                   "empty": empty}, name)


def _shared(name, groups, members, heads, kv_heads, dim, page, dtype, kv, p_lo, p_hi, lo, hi, layers, lens_seed=1, empty=0):
    """`groups` beginnings of p_lo .. p_hi tokens, each with `members` sequences that go on for lo .. hi tokens of their
    own (sequence i belongs to beginning i % groups); `empty` of them have ended."""
    return _named({"op": "shared", "groups": groups, "members": members, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                   "page": page, "dtype": dtype, "kv": kv, "p_lo": p_lo, "p_hi": p_hi, "lo": lo, "hi": hi, "layers": layers,
                   "lens_seed": lens_seed, "empty": empty}, name)


def _sample(name, rows, vocab, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, spread=2.5, mixed=False):
    """mixed: every row has settings of its own, drawn around these."""
    return _named({"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "top_k": top_k,
                   "top_p": top_p, "min_p": min_p, "spread": spread, "mixed": mixed}, name)


def listed():
    return [
        # one user's token between two linears of the small decoder: latency
        _norm("norm_b1", 1, 2048, "bf16"),
        # prompts of a batch in front of a linear with floating activations
        _norm("norm_prompts", 8192, 4096, "bf16"),
        # prompts of a batch in front of an int8 linear whose weights are rotated by 256
        _norm("norm_prompts_rot_i8", 8192, 5120, "fp16", bits=8, h=256),
        # a step's new tokens of a full batch, some slots idle
        _append("append_b64", 64, 32, 8, 128, 16, "bf16", "same", 40, 2000, 1, 1, lens_seed=3, empty=3),
        # chunks of several users' long prompts, neighbours as pairs, frequencies scaled for a longer context
        _append("append_prompts_far", 5, 32, 8, 128, 64, "bf16", "same", 1000, 60000, 500, 6000, lens_seed=5, interleaved=True,
                base=500000.0, scaling="yarn", factor=8.0, original=8192),
        # fresh prompts into a cache of 8 bits, half of each head turned
        _append("append_prompts_i8", 6, 16, 4, 128, 16, "fp16", "int8", 0, 0, 300, 4000, lens_seed=6, turn=64),
        # four alternatives of one prompt on the small decoder: latency
        _shared("shared_1x4", 1, 4, 16, 4, 128, 16, "bf16", "same", 2000, 2000, 20, 100, 4),
        # a batch's questions about one long document
        _shared("shared_1x32_long", 1, 32, 32, 8, 128, 64, "bf16", "same", 32000, 32000, 10, 1500, 2, lens_seed=4),
        # several prompts' alternatives, some ended, the cache held in 8 bits
        _shared("shared_8x8_i8", 8, 8, 32, 8, 128, 16, "fp16", "int8", 500, 9000, 30, 700, 2, lens_seed=9, empty=5),
        # one user's next token on the small decoder: latency
        _sample("sample_b1", 1, 4096, "bf16", 0.75, top_k=50),
        # a serving batch whose requests have settings of their own, a vocabulary of odd size
        _sample("sample_b64_mixed", 64, 100003, "bf16", 0.8, 40, 0.9, 0.05, mixed=True),
        # a large batch that samples from most of the mass of full-precision logits
        _sample("sample_b256_p", 256, 131072, "fp32", 1.0, top_p=0.9375),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_NORM = 8192 * 5120                # values of a drawn norm at most
MOST_APPEND = 15000 * 48 * 128         # values of drawn new tokens at most
MOST_SHARED = 32 * 33000 * 8 * 128 * 2     # key elements over all sequences and layers, as if nothing were shared, at most
MOST_HELD = 50000 * 8 * 128 * 2            # and those that are held
MOST_LOGITS = 256 * 131072


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "append", "shared", "shared", "sample", "sample", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    kv = rng.choice(["same", "same", "int8"])
    seed = rng.randrange(1 << 30)
    if op == "norm":
        bits = rng.choice([16, 8])
        h = rng.choice([0, 16, 64, 256, 256]) if bits == 8 else 0
        k = _log(rng, 64, 16384)
        k = max(h, k // h * h) if h else k // 8 * 8 if rng.random() < 0.6 else k
        m = _log(rng, 1, max(1, min(40000, MOST_NORM // k)))
        return _norm("", m, k, rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"]), rng.random() < 0.8, rng.random() < 0.8, bits, h)
    if op == "append":
        seqs = _log(rng, 1, 128)
        q_hi = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, MOST_APPEND // (seqs * (heads + 2 * kv_heads) * dim)))
        hi = 0 if kv == "int8" else rng.choice([0, _log(rng, 1, 4000), _log(rng, 1, 120000 // seqs + 1)])
        scaling = rng.choice(["none", "none", "linear", "yarn"])
        return _append("", seqs, heads, kv_heads, dim, page, dtype, kv, hi // 3, hi, max(1, q_hi // 5), q_hi, seed,
                       rng.choice([dim, dim, dim // 2, 32, 16, 24]), rng.random() < 0.5, rng.choice([10000.0, 500000.0, 1e6]),
                       scaling, 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 40.0]), rng.choice([2048, 4096, 8192]),
                       empty=seqs // 7 if hi else 0)
    if op == "shared":
        groups, members = _log(rng, 1, 12), _log(rng, 1, 64)
        layers = rng.choice([1, 2, 4])
        most = max(2, MOST_SHARED // (groups * members * kv_heads * dim * layers))
        held = MOST_HELD // (groups * kv_heads * dim * layers)             # tokens of a beginning with its sequences' own
        p_hi = _log(rng, 1, max(1, min(32000, most - 1, held // 2)))
        hi = _log(rng, 1, max(1, min(2000, most - p_hi, held // (2 * members))))
        return _shared("", groups, members, heads, kv_heads, dim, page, dtype, kv, max(1, p_hi // rng.choice([1, 2, 9])), p_hi,
                       max(1, hi // rng.choice([1, 4, 20])), hi, layers, seed, empty=groups * members // rng.choice([3, 8, 1000]))
    rows = _log(rng, 1, 512)
    vocab = _log(rng, 64, max(64, min(262144, MOST_LOGITS // rows)))
    return _sample("", rows, vocab, rng.choice(["bf16", "fp16", "fp32"]), rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]),
                   rng.choice([0, 0, 1, 20, _log(rng, 2, 2000)]), rng.choice([1.0, 1.0, 0.5, 0.8, 0.95]),
                   rng.choice([0.0, 0.0, 0.02, 0.1]), rng.choice([0.5, 2.5, 2.5, 6.0]), rng.random() < 0.4)


def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """(tokens in the cache with the new ones, new tokens) of every sequence of an append."""
    rng = random.Random(case["lens_seed"])
    q = [_log(rng, case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    lens = [n + (_log(rng, max(1, case["lo"]), case["hi"]) if case["hi"] else 0) for n in q]
    for i in rng.sample(range(case["seqs"]), case["empty"]):
        lens[i] = 0
    return lens, q


def _shared_lens(case):
    """(tokens of every beginning, tokens in the cache of every sequence)."""
    rng = random.Random(case["lens_seed"])
    first = [_log(rng, case["p_lo"], case["p_hi"]) for _ in range(case["groups"])]
    lens = [first[i % case["groups"]] + _log(rng, case["lo"], case["hi"]) for i in range(case["groups"] * case["members"])]
    for i in rng.sample(range(len(lens)), case["empty"]):
        lens[i] = 0
    return first, lens


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    return _PREPARE[case["op"]](case, dict(case), gen, dev)


def _prepare_norm(case, s, gen, dev):
    m, k, dt = case["m"], case["k"], DTYPES[case["dtype"]]
    x = torch.randn((m, k), generator=gen, device=dev)
    x[:, torch.randperm(k, generator=gen, device=dev)[: max(1, k // 100)]] *= 20       # a few strong channels
    s["res"] = (x * 0.7).to(dt) if case["residual"] else None
    s["x"] = torch.randn((m, k), generator=gen, device=dev).to(dt) if case["residual"] else x.to(dt)
    s["w"] = (1 + 0.2 * torch.randn(k, generator=gen, device=dev)).to(dt) if case["weight"] else None
    s["values"] = torch.empty((m, k), dtype=torch.bfloat16, device=dev) if case["bits"] == 8 else None
    return s


def _prepare_append(case, s, gen, dev):
    dt, h, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    lens, new = _lens(case)
    counts = [_ceil(n, page) for n in lens]
    pages = sum(counts) + 1
    place = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = place[at:at + c]
        at += c
    s["page_table"], s["kv_lens"] = table, torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor([0] + new).cumsum(0).to(dtype=torch.int32, device=dev)
    s["cu_q"] = cu if case["q_hi"] > 1 else None
    # the projection's output holds queries, keys and values of a token side by side
    qkv = torch.randn((sum(new), case["heads"] + 2 * h, d), generator=gen, device=dev, dtype=dt)
    s["q"], s["k"], s["v"] = qkv.split([case["heads"], h, h], 1)
    shape = (pages, h, page, d)
    s["k_scale"] = s["v_scale"] = None
    if case["kv"] == "int8":
        s["k_cache"], s["v_cache"] = (torch.zeros(shape, device=dev, dtype=torch.int8) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.ones(shape[:3], device=dev) for _ in range(2))
        s["values"] = [torch.empty(shape, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    else:
        s["k_cache"], s["v_cache"] = (torch.randn(shape, generator=gen, device=dev, dtype=dt) for _ in range(2))
    return s


def _cache(shape, dtype, kind, gen, dev):
    """Keys with a few strong channels or values, (cache, scales or None); an int8 cache is quantized per token
    and head as a program's would be."""
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16 if kind == "same" else torch.float32)
    x[..., :: 37] *= 3
    if kind == "same":
        return x.to(dtype), None
    s = (x.abs().amax(-1) / 127).clamp_min(1e-10)
    return torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8), s


def _prepare_shared(case, s, gen, dev):
    dt, h, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    first, lens = _shared_lens(case)
    g = case["groups"]
    full = [n // page for n in first]                                  # pages that a beginning's sequences hold together
    counts = [_ceil(n, page) for n in lens]
    pages = sum(full) + sum(max(0, c - full[b % g]) for b, c in enumerate(counts)) + 1
    place = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32, device=dev)
    at = sum(full)
    for b, c in enumerate(counts):
        if c:
            n, from_ = full[b % g], sum(full[: b % g])
            table[b, :n] = place[from_: from_ + n]
            table[b, n:c] = place[at: at + c - n]
            at += c - n
    s["page_table"], s["kv_lens"] = table, torch.tensor(lens, dtype=torch.int32, device=dev)
    shape = (pages, h, page, d)
    s["layer"] = []
    for _ in range(case["layers"]):
        q = torch.randn((len(lens), case["heads"], d), generator=gen, device=dev, dtype=dt)
        k, ks = _cache(shape, dt, case["kv"], gen, dev)
        v, vs = _cache(shape, dt, case["kv"], gen, dev)
        s["layer"].append((q, k, v, ks, vs))
    return s


def _prepare_sample(case, s, gen, dev):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn((rows, vocab), generator=gen, device=dev) * case["spread"]
    at = torch.randint(vocab, (rows, max(1, vocab // 4000)), generator=gen, device=dev)
    x.scatter_add_(1, at, 2 * case["spread"] * torch.ones(at.shape, device=dev))                # a few likely tokens
    banned = torch.randint(vocab, (rows, max(1, vocab // 100)), generator=gen, device=dev)      # and some that may not come
    x.scatter_(1, banned, -math.inf)
    s["logits"] = x.to(DTYPES[case["dtype"]])
    s["u"] = torch.rand(rows, generator=gen, device=dev)
    s["set"] = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    if case["mixed"]:
        r = torch.rand((4, rows), generator=gen, device=dev)
        off = torch.randint(4, (4, rows), generator=gen, device=dev) == 0                       # every fourth goes without
        s["set"] = {"temperature": torch.where(off[0], 0.0, case["temperature"] * (0.5 + r[0])),
                    "top_k": torch.where(off[1], 0, (case["top_k"] * 2 * r[1]).long()).to(torch.int32),
                    "top_p": torch.where(off[2], 1.0, case["top_p"] * (0.5 + r[2] / 2)),
                    "min_p": torch.where(off[3], 0.0, case["min_p"] * r[3])}
    return s


_PREPARE = {"norm": _prepare_norm, "append": _prepare_append, "shared": _prepare_shared, "sample": _prepare_sample}


# ------------------------------------------------------------------------------------------------ a pass

def run(state):
    op = state["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_norm(s):
    ck = _framework()
    if s["bits"] == 8:
        q, scale, *h = ck.rms_norm_quantize(s["x"], s["w"], s["res"], eps=EPS, convrot_groupsize=s["h"] or None)
        return [torch.mul(q, scale[:, None], out=s["values"]), scale, *h]
    y = ck.rms_norm(s["x"], s["w"], s["res"], eps=EPS)
    return list(y) if s["residual"] else [y]


def _own_append(s):
    ck = _framework()
    key = (s["turn"], s["base"], s["interleaved"], s["scaling"], s["factor"], s["original"])
    if key not in _rotary:
        _rotary[key] = ck.Rotary(s["turn"], base=s["base"], interleaved=s["interleaved"],
                                 scaling=None if s["scaling"] == "none" else s["scaling"], factor=s["factor"],
                                 original=s["original"])
    q = ck.kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"], rotary=_rotary[key],
                     cu_q=s["cu_q"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return [q, *_held(s)]


def _held(s):
    if s["kv"] != "int8":
        return [s["k_cache"], s["v_cache"]]
    return [torch.mul(s[c + "_cache"], s[c + "_scale"][..., None], out=to) for c, to in zip("kv", s["values"])] + \
        [s["k_scale"], s["v_scale"]]


def _own_shared(s):
    ck = _framework()
    plan = ck.kv_shared(s["page_table"], s["kv_lens"], s["page"])       # once a step, for all layers
    return [ck.paged_attention(q, k, v, s["page_table"], s["kv_lens"], k_scale=ks, v_scale=vs, shared=plan)
            for q, k, v, ks, vs in s["layer"]]


def _own_sample(s):
    return _framework().sample(s["logits"], s["u"], **s["set"])


def _hadamard(h, dtype, dev):
    """H_h = (H4 / 2)^(x log4 h): each radix-4 stage is y_i = (x0 + x1 + x2 + x3) / 2 - x_(3-i)."""
    one = torch.full((4, 4), 0.5, dtype=dtype, device=dev) - torch.eye(4, dtype=dtype, device=dev).flip(0)
    mat = torch.kron(one, one)
    if h >= 64:
        mat = torch.kron(mat, one)
    return torch.kron(mat, one) if h == 256 else mat


def _plain_norm(s):
    h = s["x"]
    if s["res"] is not None:
        h = (h.float() + s["res"].float()).to(h.dtype)
    y = h.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    if s["w"] is not None:
        y = y * s["w"].float()
    more = [] if s["res"] is None else [h]
    if s["bits"] == 16:
        return [y.to(h.dtype), *more]
    if s["h"]:
        y = torch.matmul(y.view(-1, s["h"]), _hadamard(s["h"], torch.float32, y.device)).view(y.shape)
    scale = (y.abs().amax(-1) / 127).clamp_min(1e-10)
    return [(torch.round(y / scale[:, None]) * scale[:, None]).to(torch.bfloat16), scale, *more]


def _frequencies(s):
    """(radians a position of every pair, what cosines and sines are multiplied by)."""
    n, base, factor = s["turn"] // 2, s["base"], s["factor"]
    f = [base ** (-i / n) for i in range(n)]
    if s["scaling"] == "none":
        return f, 1.0
    if s["scaling"] == "linear":
        return [x / factor for x in f], 1.0

    def pair(turns):        # the pair that turns so often over the context that the model was trained on
        return n * math.log(s["original"] / (turns * 2 * math.pi)) / math.log(base)

    lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), 2 * n - 1)
    ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(n)]
    return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0


def _positions(s, tokens, dev):
    """(sequence, position) of every new token."""
    tok, lens = torch.arange(tokens, device=dev), s["kv_lens"].long()
    if s["cu_q"] is None:
        return tok, lens - 1
    cu = s["cu_q"].long()
    seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    return seq, lens[seq] - cu[seq + 1] + tok


def _turned(x, c, sn, s):
    """fp32 [tokens, heads, dim] with its first `turn` values as pairs turned."""
    n, x = s["turn"], x.float()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if s["interleaved"] else (x[..., : n // 2], x[..., n // 2: n])
    y = (a * c - b * sn, a * sn + b * c)
    y = torch.stack(y, -1).flatten(-2) if s["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., n:]], -1)


def _plain_append(s):
    q, k, v, page = s["q"], s["k"], s["v"], s["page"]
    seq, pos = _positions(s, q.shape[0], q.device)
    f, size = _frequencies(s)
    a = pos.clamp_min(0).double()[:, None] * torch.tensor(f, dtype=torch.float64, device=q.device)
    c, sn = (a.cos() * size).float()[:, None], (a.sin() * size).float()[:, None]
    turned = pos >= 0                                                  # a token without a position stays as it is
    q = torch.where(turned[:, None, None], _turned(q, c, sn, s), q.float()).to(q.dtype)
    k = _turned(k, c, sn, s)
    seq, pos = seq[turned], pos[turned]
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    for n, x in (("k", k[turned]), ("v", v[turned].float())):
        if s["kv"] == "int8":
            scale = (x.abs().amax(-1) / 127).clamp_min(1e-10)
            s[n + "_scale"][at, :, slot] = scale
            x = torch.round(x / scale[..., None])
        s[n + "_cache"][at, :, slot] = x.to(s[n + "_cache"].dtype)
    return [q, *_held(s)]


def _gather(cache, scale, table):
    """Pages of every sequence side by side: fp32 [seqs, kv_heads, tokens, dim]."""
    at = table.clamp_min(0).long()
    x = cache[at].float()                                     # [seqs, pages, kv_heads, page, dim]
    if scale is not None:
        x = x * scale[at][..., None]
    b, w, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, w * p, d)


def _plain_shared(s):
    return [_plain_attention(s, *layer) for layer in s["layer"]]


def _plain_attention(s, q, k, v, ks, vs):
    (b, heads, d), h, lens = q.shape, s["kv_heads"], s["kv_lens"].long()
    key, value = _gather(k, ks, s["page_table"]), _gather(v, vs, s["page_table"])
    held = (torch.arange(key.shape[2], device=q.device) < lens[:, None])[:, None, None]      # [seqs, 1, 1, tokens]
    value = torch.where(held.transpose(2, 3), value, torch.zeros((), device=q.device))
    rows = q.float().view(b, h, heads // h, d)
    score = torch.matmul(rows, key.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d)).masked_fill_(~held, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    out = torch.matmul(p, value) / p.sum(-1, keepdim=True)
    return torch.where((lens > 0)[:, None, None, None], out, torch.zeros((), device=q.device)).view(q.shape).to(q.dtype)


def _setting(x, dev):
    return (x if isinstance(x, torch.Tensor) else torch.tensor([x], device=dev)).double()[:, None]


def _plain_sample(s):
    x, dev = s["logits"].float(), s["logits"].device
    vocab = x.shape[1]
    t, k, p, least = (_setting(s["set"][n], dev) for n in ("temperature", "top_k", "top_p", "min_p"))
    value, at = torch.sort(x, dim=-1, descending=True, stable=True)
    value = value.double()
    w = torch.exp((value - value[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    rank = torch.arange(vocab, device=dev)
    keep = (k <= 0) | (rank < k)
    mass = w * keep
    before = mass.cumsum(-1) - mass
    keep = keep & ((p >= 1) | (before < p * mass.sum(-1, keepdim=True))) & (w >= least) | (rank == 0)
    keep = keep & ((t > 0) | (rank == 0))                     # temperature 0: the best one
    mass = torch.zeros_like(w).scatter_(1, at, w * keep)
    sums = mass.cumsum(-1)
    token = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(-1)
    last = torch.where(mass > 0, rank, -1).amax(-1)
    return torch.minimum(token, last)


_OWN = {"norm": _own_norm, "append": _own_append, "shared": _own_shared, "sample": _own_sample}
_PLAIN = {"norm": _plain_norm, "append": _plain_append, "shared": _plain_shared, "sample": _plain_sample}


# ------------------------------------------------------------------------------------------------ work

def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "fp32" else 2
    if op == "norm":
        m, k = case["m"], case["k"]
        out = m * k * e if case["bits"] == 16 else m * (k + 4)
        stages = {0: 0, 16: 2, 64: 3, 256: 4}[case["h"]]
        return {"bytes": m * k * e * (3 if case["residual"] else 1) + out + k * e * case["weight"], "flops": m * k * (4 + 2 * stages)}
    if op == "append":
        n, d, h = sum(_lens(case)[1]), case["dim"], case["kv_heads"]
        one = 2 * h * (d + 4 if case["kv"] == "int8" else 2 * d)           # a token's keys and values as they are held
        return {"bytes": n * (2 * (case["heads"] + 2 * h) * d + 2 * case["heads"] * d + one),
                "flops": n * (case["heads"] + h) * case["turn"] * 3}
    if op == "shared":
        first, lens = _shared_lens(case)
        h, d, g, page = case["kv_heads"], case["dim"], case["groups"], case["page"]
        one = h * (2 * d + 8 if case["kv"] == "int8" else 4 * d)           # K and V of a token
        tokens = 0
        for b in range(g):
            own_lens = [n for n in lens[b::g] if n]
            once = first[b] // page * page
            tokens += sum(own_lens) - max(0, len(own_lens) - 1) * once
        io = 4 * sum(1 for n in lens if n) * case["heads"] * d
        return {"bytes": case["layers"] * (one * tokens + io), "flops": case["layers"] * 4 * case["heads"] * d * sum(lens)}
    return {"bytes": case["rows"] * (case["vocab"] * e + 12), "flops": 0 if case["temperature"] == 0 else 2 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "shared": _exact_shared, "sample": _exact_sample}[case["op"]](case, s)


def _exact_norm(case, s):
    h = s["x"].double()
    if case["residual"]:
        h = (h + s["res"].double()).to(s["x"].dtype).double()              # what the residual stream holds
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["k"] + EPS)
    if case["weight"]:
        y *= s["w"].double()
    more = [h] if case["residual"] else []
    if case["bits"] == 16:
        return [y] + more
    if case["h"]:
        y = (y.reshape(case["m"], -1, case["h"]) @ _hadamard(case["h"], torch.float64, y.device)).reshape(case["m"], -1)
    step = torch.maximum(y.abs().max(1).values / 127, torch.tensor(1e-10, dtype=torch.float64, device=y.device))
    return [torch.round(y / step.unsqueeze(1)) * step.unsqueeze(1), step] + more


def _exact_append(case, s):
    lens, new = _lens(case)
    f, size = _frequencies(s)
    dev, n = s["q"].device, case["turn"] // 2
    f = torch.tensor(f, dtype=torch.float64, device=dev)
    first = [2 * i if case["interleaved"] else i for i in range(n)]
    second = [2 * i + 1 if case["interleaved"] else i + n for i in range(n)]

    def turn(x, pos):
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(pos * f, size), pos * f).unsqueeze(1)
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = [s["q"].double(), s["k_cache"].double(), s["v_cache"].double()]
    scales = [s["k_scale"].double(), s["v_scale"].double()] if case["kv"] == "int8" else []
    for c, sc in zip(out[1:], scales):
        c *= sc.unsqueeze(-1)
    begin = 0
    for b, (length, count) in enumerate(zip(lens, new)):
        rows = slice(begin, begin + count)
        begin += count
        if not length:
            continue
        where = torch.arange(length - count, length, device=dev)
        pos = where.double().unsqueeze(1)
        out[0][rows] = turn(out[0][rows].clone(), pos)
        page, slot = s["page_table"][b].long()[torch.div(where, case["page"], rounding_mode="floor")], where % case["page"]
        for i, x in enumerate((turn(s["k"][rows].double(), pos), s["v"][rows].double())):
            if scales:
                step = torch.clamp(x.abs().max(-1).values / 127, min=1e-10)
                scales[i][page, :, slot] = step
                x = torch.round(x / step.unsqueeze(-1)) * step.unsqueeze(-1)
            out[1 + i][page, :, slot] = x
    return out + scales


def _exact_shared(case, s):
    _, lens = _shared_lens(case)
    d, page, group = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    outs = []
    for q, k, v, ks, vs in s["layer"]:
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for b, length in enumerate(lens):
            if not length:
                continue
            at = s["page_table"][b, : _ceil(length, page)].long()
            kk, vv = k[at].double(), v[at].double()
            if ks is not None:
                kk, vv = kk * ks[at].double().unsqueeze(-1), vv * vs[at].double().unsqueeze(-1)
            for h in range(case["kv_heads"]):
                keys, values = (x[:, h].reshape(-1, d)[:length] for x in (kk, vv))
                rows = slice(h * group, (h + 1) * group)
                out[b, rows] = torch.softmax(q[b, rows].double() @ keys.t() / math.sqrt(d), -1) @ values
        outs.append(out)
    return outs


def _exact_sample(case, s):
    x, u = s["logits"].float().cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    rows, vocab = x.shape
    sets = {n: np.broadcast_to(v.cpu().numpy().astype(np.float64) if isinstance(v, torch.Tensor) else np.float64(v), (rows,))
            for n, v in s["set"].items()}
    tokens = np.zeros(rows, dtype=np.int64)
    for r in range(rows):
        order = np.lexsort((np.arange(vocab), -x[r]))                      # the best first, ties by their number
        best = x[r, order[0]]
        if sets["temperature"][r] <= 0:
            tokens[r] = order[0]
            continue
        if sets["top_k"][r] > 0:
            order = order[: int(sets["top_k"][r])]
        w = np.exp((x[r, order] - best) / sets["temperature"][r])
        if sets["top_p"][r] < 1:
            sums = np.cumsum(w)
            n = 1 + int(np.searchsorted(sums, sets["top_p"][r] * sums[-1], side="left"))
            order, w = order[:n], w[:n]
        fine = w >= sets["min_p"][r]
        fine[0] = True
        order, w = order[fine], w[fine]
        by = np.argsort(order)
        order, w = order[by], w[by]
        sums = np.cumsum(w)
        n = int(np.searchsorted(sums, u[r] * sums[-1], side="right"))
        tokens[r] = order[min(n, np.flatnonzero(w)[-1])]
    return torch.from_numpy(tokens)
