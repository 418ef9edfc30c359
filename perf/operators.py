"""Performance cases of single-token serving: attention over a paged key-value cache, the cache's upkeep, and
products of a few rows with 4-bit weights whose activations stay in floating point.

Five operators, as a program that generates tokens with quantized weights calls them:

  decode   attention of one new token per sequence over the pages of a cache (grouped heads, 16-bit or int8
           cache, sliding window with a few first tokens that stay visible)
  prompt   attention of a ragged batch of prompt chunks over the same pages (causal, window, first tokens)
  write    the new tokens' keys and values into their sequences' pages
  pages    forking sequences (full pages shared, the last one copied) and growing them; freeing
           sequences and compacting the pages that are left
  w4a16    y = x W^T + bias with 4-bit weights, a scale per group and integer or floating zero-points, the
           activations optionally rotated by Hadamard blocks as the converted checkpoints ask for

Sequence lengths belong to the case (`lens_seed`); values and the pages' places come from the seed.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ck = None


def _framework():
    global _ck
    if _ck is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfy-quant-bench_amd"))
        import kitchen_amd

        _ck = kitchen_amd
    return _ck


# ------------------------------------------------------------------------------------------------ cases

def _attn(op, name, seqs, heads, kv_heads, dim, page, dtype, kv, lo, hi, lens_seed=1, window=0, sinks=0, empty=0,
          q_lo=1, q_hi=1):
    """`seqs` sequences of lo .. hi cached tokens (`empty` of them idle: length 0); prompt: chunks of q_lo .. q_hi
    new tokens behind lo .. hi earlier ones."""
    case = {"op": op, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "kv": kv, "lo": lo, "hi": hi, "lens_seed": lens_seed, "window": window, "sinks": sinks, "empty": empty,
            "q_lo": q_lo, "q_hi": q_hi}
    return dict(case, name=name) if name else case


def _write(name, seqs, kv_heads, dim, page, dtype, lo, hi, q_lo, q_hi, lens_seed=1):
    case = {"op": "write", "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "lo": lo,
            "hi": hi, "lens_seed": lens_seed, "empty": 0, "q_lo": q_lo, "q_hi": q_hi}
    return dict(case, name=name) if name else case


def _pages(name, what, layers, pages, kv_heads, dim, page, dtype, seqs, lo, hi, n, lens_seed=1):
    """fork: n children of `seqs` sequences; compact: n of `seqs` sequences end."""
    case = {"op": "pages", "what": what, "layers": layers, "pages": pages, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "n": n, "lens_seed": lens_seed}
    return dict(case, name=name) if name else case


def _w4(name, m, n, k, group, zeros, dtype, h=0, bias=True):
    case = {"op": "w4a16", "m": m, "n": n, "k": k, "group": group, "zeros": zeros, "dtype": dtype, "h": h, "bias": bias}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one user's chat a few hundred tokens in, a small model with a sliding window: latency
        _attn("decode", "decode_b1_window", 1, 16, 16, 64, 32, "fp16", "same", 517, 517, window=256, sinks=4),
        # one user over a long document: the whole cache is read for one token
        _attn("decode", "decode_b1_131071", 1, 32, 8, 128, 64, "bf16", "same", 131071, 131071),
        # a full serving batch of ragged lengths, some slots idle, the cache held in 8 bits
        _attn("decode", "decode_b64_ragged_i8", 64, 32, 8, 128, 16, "bf16", "int8", 40, 8000, lens_seed=3, empty=3),
        # a short text prompt at the start of a chat
        _attn("prompt", "prompt_77", 1, 24, 24, 128, 16, "bf16", "same", 0, 0, q_lo=77, q_hi=77),
        # chunks of several users' prompts behind what they said before, sliding window
        _attn("prompt", "prompt_ragged_window", 5, 32, 8, 128, 16, "fp16", "same", 0, 3000, lens_seed=5, window=1024,
              sinks=4, q_lo=100, q_hi=3000),
        # a whole long prompt at once, full causal attention
        _attn("prompt", "prompt_8192", 1, 32, 8, 128, 64, "bf16", "same", 0, 0, q_lo=8192, q_hi=8192),
        # a step's new tokens of a batch into their pages
        _write("write_b64", 64, 8, 128, 16, "bf16", 40, 8000, 1, 1, lens_seed=3),
        # prompt chunks into their pages
        _write("write_prompts", 6, 8, 128, 16, "fp16", 0, 3000, 1000, 6000, lens_seed=6),
        # 16 sequences fork three alternatives each, and every alternative gets room for its next token
        _pages("fork_16x3", "fork", 16, 2048, 8, 128, 16, "bf16", 16, 200, 1500, 48, lens_seed=7),
        # half the sequences of a batch have ended: their pages are freed and the others' moved together
        _pages("compact_half", "compact", 16, 2048, 8, 128, 16, "bf16", 32, 100, 1800, 16, lens_seed=8),
        # a one-token linear of a converted checkpoint (uint4 weights rotated by 256, zero-points)
        _w4("w4a16_m1_rot", 1, 18432, 3072, 64, "u4", "bf16", h=256),
        # a batch's projection with floating zero-points
        _w4("w4a16_m16", 16, 12288, 4096, 128, "float", "fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_CACHE = 131071 * 8 * 128          # key elements that a drawn decode reads at most
MOST_PAIRS = 8192 * 8192 // 2 * 32     # query-key pairs over all heads of a drawn prompt at most


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "write", "pages", "w4a16", "w4a16"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    window, sinks = rng.choice([(0, 0), (_log(rng, 8, 4096), rng.choice([0, 1, 4, 17]))])
    seed = rng.randrange(1 << 30)
    if op == "decode":
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, max(1, min(131071, MOST_CACHE // (seqs * kv_heads * dim))))
        lo = rng.choice([hi, 1 + hi // 4, 1])
        kv = rng.choice(["same", "int8"])
        return _attn(op, "", seqs, kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv_heads, dim, page, dtype, kv, lo, hi,
                     seed, window, sinks, empty=seqs // 5)
    if op == "prompt":
        seqs, group = _log(rng, 1, 12), rng.choice([1, 2, 3, 4, 7])
        q_hi = _log(rng, 1, 4096)
        hi = rng.choice([0, _log(rng, 1, 4096)])
        while seqs * kv_heads * group * q_hi * (q_hi + hi) > MOST_PAIRS // 2 and q_hi > 1:
            q_hi, hi, seqs = q_hi // 2, hi // 2, max(1, seqs - 1)
        return _attn(op, "", seqs, kv_heads * group, kv_heads, dim, page, dtype, rng.choice(["same", "same", "int8"]),
                     hi // 3, hi, seed, window, sinks, q_lo=max(1, q_hi // 7), q_hi=q_hi)
    if op == "write":
        seqs = _log(rng, 1, 128)
        q_hi = _log(rng, 1, max(1, 20000 // seqs))
        hi = rng.choice([0, _log(rng, 1, 4000)])
        return _write("", seqs, kv_heads, dim, page, dtype, hi // 3, hi, max(1, q_hi // 5), q_hi, seed)
    if op == "pages":
        what = rng.choice(["fork", "compact"])
        layers = rng.choice([1, 4, 16, 28])
        seqs = _log(rng, 2, 48)
        hi = _log(rng, 1, 1500)
        n = rng.choice([1, seqs, 2 * seqs]) if what == "fork" else max(1, seqs // rng.choice([2, 3, 8]))
        used = seqs * (-(-hi // page)) + 2 * n + 3
        while used * page * kv_heads * dim * layers > 12 * 2048 * 8 * 16 * 128 and layers > 1:
            layers = layers // 2
        return _pages("", what, layers, used + rng.choice([0, 5, used // 2]), kv_heads, dim, page, dtype, seqs,
                      max(1, hi // 6), hi, n, seed)
    group = rng.choice([32, 64, 64, 128])
    k = group * max(1, _log(rng, 256, 16384) // group)
    n = _log(rng, 16, 32768)
    while n * k > 1 << 26:
        n //= 2
    h = rng.choice([0, 0, 16, 64, 256])
    return _w4("", _log(rng, 1, 64), n, k, group, rng.choice(["none", "u4", "float"]), rng.choice(["bf16", "fp16", "fp32"]),
               h if h and k % h == 0 else 0, rng.random() < 0.5)


def _lens(case):
    """(tokens in the cache with the new ones, new tokens) of every sequence."""
    rng = random.Random(case["lens_seed"])
    q = [_log(rng, case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    if case["op"] == "decode":
        lens = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    else:
        lens = [n + (_log(rng, max(1, case["lo"]), case["hi"]) if case["hi"] else 0) for n in q]
    for i in rng.sample(range(case["seqs"]), case["empty"]):
        lens[i] = 0
    return lens, q


def _row_lens(case):
    rng = random.Random(case["lens_seed"])
    return [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------------------ inputs

def _table(lens, page, gen, dev, pages=None, width=None, rows=None):
    """int32 table of pages in random places (-1 behind a sequence's end)."""
    counts = [_ceil(n, page) for n in lens]
    pages = sum(counts) + 1 if pages is None else pages
    place = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((rows or len(lens), width or max(1, max(counts))), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = place[at:at + c]
        at += c
    return table, pages


def _cache(shape, dtype, kind, gen, dev):
    """Keys with a few strong channels or values, (cache, scales or None); an int8 cache is quantized per token
    and head as a program's would be."""
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16 if kind == "same" else torch.float32)
    x[..., :: 37] *= 3
    if kind == "same":
        return x.to(dtype), None
    s = (x.abs().amax(-1) / 127).clamp_min(1e-10)
    return torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["op"] == "w4a16":
        return _prepare_w4(case, s, gen, dev)
    if case["op"] == "pages":
        return _prepare_pages(case, s, gen, dev)
    dt, h, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    lens, q = _lens(case)
    s["page_table"], pages = _table(lens, page, gen, dev)
    s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    shape = (pages, h, page, d)
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    ragged = case["op"] == "prompt" or case["op"] == "write" and case["q_hi"] > 1
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=dev) if ragged else None
    s["q_most"] = max(q)
    if case["op"] == "write":
        s["k_cache"], s["v_cache"] = (torch.randn(shape, generator=gen, device=dev, dtype=dt) for _ in range(2))
        s["k"], s["v"] = (torch.randn((cu[-1], h, d), generator=gen, device=dev, dtype=dt) for _ in range(2))
        return s
    s["q"] = torch.randn((cu[-1], case["heads"], d), generator=gen, device=dev, dtype=dt)
    s["k_cache"], s["k_scale"] = _cache(shape, dt, case["kv"], gen, dev)
    s["v_cache"], s["v_scale"] = _cache(shape, dt, case["kv"], gen, dev)
    return s


def _prepare_pages(case, s, gen, dev):
    lens, n, fork = _row_lens(case), case["n"], case["what"] == "fork"
    rows = case["seqs"] + (n if fork else 0)
    width = _ceil(case["hi"] + 1, case["page"])
    table, pages = _table(lens, case["page"], gen, dev, case["pages"], width, rows)
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    refs[table[table >= 0].long()] = 1
    # the small state in one buffer, so that a pass starts from the same one with one copy
    s["start"] = torch.cat([table.reshape(-1), torch.tensor(lens + [0] * (rows - len(lens)), dtype=torch.int32, device=dev), refs])
    s["now"] = s["start"].clone()
    s["page_table"] = s["now"][: rows * width].view(rows, width)
    s["lens"] = s["now"][rows * width: rows * width + rows]
    s["refs"] = s["now"][rows * width + rows:]
    shape = (case["layers"], pages, case["kv_heads"], case["page"], case["dim"])
    s["k"], s["v"] = (torch.randn(shape, generator=gen, device=dev, dtype=DTYPES[case["dtype"]]) for _ in range(2))
    if fork:
        s["src"] = (torch.arange(n, device=dev) % case["seqs"]).to(torch.int32)
        s["dst"] = (torch.arange(n, device=dev) + case["seqs"]).to(torch.int32)
        s["counts"] = torch.ones(n, dtype=torch.int32, device=dev)
    else:
        s["ended"] = torch.randperm(case["seqs"], generator=gen, device=dev)[:n].to(torch.int32)
    return s


def _prepare_w4(case, s, gen, dev):
    m, n, k, g = case["m"], case["n"], case["k"], case["group"]
    dt = DTYPES[case["dtype"]]
    w = torch.randn((n, k // g, g), generator=gen, device=dev) * 0.02
    if case["zeros"] == "none":
        sc = (w.abs().amax(-1) / 7).half()
        code = torch.round(w / sc[..., None].float()).clamp_(-7, 7).to(torch.int32) & 15
        zeros = None
    else:
        lo, hi = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        sc = ((hi - lo) / 15).half()
        if case["zeros"] == "u4":
            z = torch.round(-lo / sc.float()).clamp_(0, 15)
            code = (torch.round(w / sc[..., None].float()) + z[..., None]).clamp_(0, 15).to(torch.int32)
            z = torch.nn.functional.pad(z.to(torch.uint8), (0, k // g % 2))
            zeros = z[:, 0::2] | z[:, 1::2] << 4
        else:
            zeros = lo.half()
            code = torch.round((w - lo[..., None]) / sc[..., None].float()).clamp_(0, 15).to(torch.int32)
    code = code.view(n, k)
    s["qweight"] = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    s["wscales"], s["wzeros"] = sc, zeros
    x = torch.randn((m, k), generator=gen, device=dev)
    x[:, torch.randperm(k, generator=gen, device=dev)[: max(1, k // 100)]] *= 20
    s["x"] = x.to(dt)
    s["bias_t"] = torch.randn(n, generator=gen, device=dev).to(dt) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------------------ a pass

def run(state):
    op = state["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_attention(s):
    return _framework().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"],
                                        cu_q=s["cu_q"], window=s["window"] or None, sinks=s["sinks"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_write(s):
    _framework().kv_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"], cu_q=s["cu_q"])
    return [s["k_cache"], s["v_cache"]]


def _own_pages(s):
    ck = _framework()
    s["now"].copy_(s["start"])
    if s["what"] == "fork":
        ck.kv_fork(s["k"], s["v"], s["page_table"], s["lens"], s["refs"], s["src"], s["dst"])
        ck.kv_grow(s["page_table"], s["lens"], s["refs"], s["dst"], s["counts"], s["page"])
        return [s["k"], s["v"], s["page_table"], s["lens"], s["refs"]]
    ck.kv_free(s["page_table"], s["lens"], s["refs"], s["ended"])
    live = ck.kv_compact(s["k"], s["v"], s["page_table"], s["refs"])
    return [s["k"], s["v"], s["page_table"], s["lens"], s["refs"], live]


def _own_w4(s):
    return _framework().w4a16_linear(s["x"], s["qweight"], s["wscales"], s["wzeros"], s["bias_t"],
                                     group_size=s["group"], convrot_groupsize=s["h"] or None)


def _gather(cache, scale, table):
    """Pages of every sequence side by side: fp32 [seqs, kv_heads, tokens, dim]."""
    at = table.clamp_min(0).long()
    x = cache[at].float()                                     # [seqs, pages, kv_heads, page, dim]
    if scale is not None:
        x = x * scale[at][..., None]
    b, w, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, w * p, d)


def _plain_attention(s):
    q, table, lens = s["q"], s["page_table"], s["kv_lens"].long()
    dev, (b, h, d) = q.device, (table.shape[0], s["kv_heads"], s["dim"])
    most, group = s["q_most"], q.shape[1] // h
    tok = torch.arange(q.shape[0], device=dev)
    if s["cu_q"] is None:
        seq, i, new = tok, torch.zeros_like(tok), torch.ones_like(lens)
    else:
        cu = s["cu_q"].long()
        seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
        i, new = tok - cu[seq], cu[1:] - cu[:-1]
    rows = torch.zeros((b, most, h, group, d), device=dev)
    rows[seq, i] = q.float().view(-1, h, group, d)
    rows = rows.permute(0, 2, 3, 1, 4).reshape(b, h, group * most, d)
    key = _gather(s["k_cache"], s["k_scale"], table)
    j = torch.arange(key.shape[2], device=dev)
    held = j < lens[:, None]                                  # [seqs, tokens]
    value = _gather(s["v_cache"], s["v_scale"], table)
    value = torch.where(held[:, None, :, None], value, torch.zeros((), device=dev))
    score = torch.matmul(rows, key.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d)).view(b, h, group, most, -1)
    at = (lens - new)[:, None] + torch.arange(most, device=dev)          # position of every query
    seen = held[:, None, :] & (j <= at[..., None])
    if s["window"]:
        seen &= (j > at[..., None] - s["window"]) | (j < s["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, h, group * most, -1), value).view(b, h, group, most, d)
    out = torch.where(seen.any(-1)[:, None, None, :, None], out / total, torch.zeros((), device=dev))
    return out.permute(0, 3, 1, 2, 4)[seq, i].reshape(q.shape).to(q.dtype)


def _plain_write(s):
    k, lens, page = s["k"], s["kv_lens"].long(), s["page"]
    tok = torch.arange(k.shape[0], device=k.device)
    if s["cu_q"] is None:
        seq, pos = tok, lens - 1
    else:
        cu = s["cu_q"].long()
        seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
        pos = lens[seq] - cu[seq + 1] + tok
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    s["k_cache"][at, :, slot] = k
    s["v_cache"][at, :, slot] = s["v"]
    return [s["k_cache"], s["v_cache"]]


def _take_free(refs, need):
    """The lowest free pages, as many as `need` says."""
    return torch.nonzero(refs == 0).view(-1)[: int(need)]


def _plain_pages(s):
    s["now"].copy_(s["start"])
    k, v, table, lens, refs, page = s["k"], s["v"], s["page_table"], s["lens"], s["refs"], s["page"]
    col = torch.arange(table.shape[1], device=k.device)
    if s["what"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        held = lens[src].long()
        full = held // page
        row = torch.where(col < full[:, None], table[src], torch.full_like(table[src], -1))
        shared = row[row >= 0].long()
        free = refs == 0
        refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
        part = held % page > 0
        new = torch.nonzero(free).view(-1)[: int(part.sum())]
        last = table[src[part], full[part]].long()
        row[part, full[part]] = new.to(torch.int32)
        table[dst] = row
        refs[new] = 1
        lens[dst] = held.to(torch.int32)
        k[:, new], v[:, new] = k[:, last], v[:, last]
        # room for the next tokens
        held, count = lens[dst].long(), s["counts"].long()
        have, want = (held + page - 1) // page, (held + count + page - 1) // page
        more = (col >= have[:, None]) & (col < want[:, None])
        new = _take_free(refs, more.sum())
        row = table[dst]
        row[more] = new.to(torch.int32)
        table[dst] = row
        refs[new] = 1
        lens[dst] = (held + count).to(torch.int32)
        return [k, v, table, lens, refs]
    ended = s["ended"].long()
    row = table[ended]
    gone = row[row >= 0].long()
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table[ended] = -1
    lens[ended] = 0
    live = refs > 0
    count = live.sum()
    low = torch.arange(refs.shape[0], device=k.device) < count
    src, dst = torch.nonzero(live & ~low).view(-1), torch.nonzero(~live & low).view(-1)
    place = torch.arange(refs.shape[0], device=k.device, dtype=torch.int32)
    place[src] = dst.to(torch.int32)
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, place[table.clamp_min(0).long()], table))
    return [k, v, table, lens, refs, count.to(torch.int32).view(1)]


def _hadamard(h, dtype, dev):
    """H_h = (H4 / 2)^(x log4 h): each radix-4 stage is y_i = (x0 + x1 + x2 + x3) / 2 - x_(3-i)."""
    one = torch.full((4, 4), 0.5, dtype=dtype, device=dev) - torch.eye(4, dtype=dtype, device=dev).flip(0)
    mat = torch.kron(one, one)
    if h >= 64:
        mat = torch.kron(mat, one)
    return torch.kron(mat, one) if h == 256 else mat


def _plain_w4(s):
    q, sc, z, g = s["qweight"].to(torch.int32), s["wscales"].float(), s["wzeros"], s["group"]
    n, k = q.shape[0], q.shape[1] * 2
    code = torch.stack([q & 15, q >> 4], dim=-1).view(n, k // g, g)
    if z is None:
        w = (code - 16 * (code > 7)).float() * sc[..., None]
    elif z.dtype == torch.uint8:
        z = torch.stack([z & 15, z >> 4], dim=-1).view(n, -1)[:, : k // g].to(torch.int32)
        w = (code - z[..., None]).float() * sc[..., None]
    else:
        w = code.float() * sc[..., None] + z.float()[..., None]
    x = s["x"].float()
    if s["h"]:
        x = torch.matmul(x.view(-1, s["h"]), _hadamard(s["h"], torch.float32, x.device)).view(x.shape)
    y = torch.matmul(x, w.view(n, k).t().contiguous())
    if s["bias_t"] is not None:
        y = y + s["bias_t"].float()
    return y.to(s["x"].dtype)


_OWN = {"decode": _own_attention, "prompt": _own_attention, "write": _own_write, "pages": _own_pages, "w4a16": _own_w4}
_PLAIN = {"decode": _plain_attention, "prompt": _plain_attention, "write": _plain_write, "pages": _plain_pages,
          "w4a16": _plain_w4}


# ------------------------------------------------------------------------------------------------ work

def _visible(length, window, sinks):
    """Keys that the query at position length - 1 sees."""
    return length if not window or length <= window else window + min(sinks, length - window)


def work(case):
    op = case["op"]
    if op == "w4a16":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        e = 4 if case["dtype"] == "fp32" else 2
        zero = {"none": 0, "u4": 0.5, "float": 2}[case["zeros"]]
        return {"bytes": n * k / 2 + n * k / g * (2 + zero) + e * (m * k + m * n + n * case["bias"]), "flops": 2 * m * n * k}
    if op == "pages":
        lens, page, n = _row_lens(case), case["page"], case["n"]
        one = 2 * 2 * case["layers"] * case["kv_heads"] * page * case["dim"]      # K and V of a page, all layers
        if case["what"] == "fork":
            src = [i % case["seqs"] for i in range(n)]
            part = [i for i in src if lens[i] % page]
            return {"bytes": one * (len(part) + len(set(part))), "flops": 0}
        # which sequences end comes from the seed: the share of live pages above the live count, on average
        used = sum(_ceil(x, page) for x in lens)
        live = used * (1 - n / case["seqs"])
        return {"bytes": 2 * one * live * (1 - live / case["pages"]), "flops": 0}
    h, d = case["kv_heads"], case["dim"]
    lens, q = _lens(case)
    if op == "write":
        return {"bytes": 2 * 2 * 2 * sum(q) * h * d, "flops": 0}
    one = h * (2 * d + 8 if case["kv"] == "int8" else 4 * d)                      # K and V of a token
    w, first = case["window"], case["sinks"]
    io = 4 * sum(q) * case["heads"] * d
    if op == "decode":
        seen = sum(_visible(x, w, first) for x in lens)
        return {"bytes": one * seen + io, "flops": 4 * case["heads"] * d * seen}
    pairs, keys = 0, 0
    for x, n in zip(lens, q):
        pairs += sum(_visible(p + 1, w, first) for p in range(x - n, x))
        keys += x if not w else min(x, w + n - 1 + first)
    return {"bytes": one * keys + io, "flops": 4 * case["heads"] * d * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "w4a16":
        return _exact_w4(s)
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(case, s)
    if case["op"] == "write":
        return _exact_write(case, s)
    return _exact_pages(case, s)


def _exact_attention(case, s):
    lens, new = _lens(case)
    d, page, group = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    first = 0
    for b, (length, n) in enumerate(zip(lens, new)):
        at = s["page_table"][b, : _ceil(length, page)].long()
        pos = torch.arange(length - n, length, device=out.device).view(-1, 1)
        j = torch.arange(length, device=out.device)
        hidden = j > pos
        if case["window"]:
            hidden |= (pos - j >= case["window"]) & (j >= case["sinks"])
        for h in range(case["kv_heads"] if length else 0):
            kk, vv = (s[c][at, h].double() for c in ("k_cache", "v_cache"))
            if case["kv"] == "int8":
                kk, vv = kk * s["k_scale"][at, h].double().unsqueeze(-1), vv * s["v_scale"][at, h].double().unsqueeze(-1)
            kk, vv = kk.reshape(-1, d)[:length], vv.reshape(-1, d)[:length]
            for g in range(h * group, (h + 1) * group):
                a = s["q"][first: first + n, g].double() @ kk.t() / math.sqrt(d)
                out[first: first + n, g] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ vv
        first += n
    return out


def _exact_write(case, s):
    lens, new = _lens(case)
    out = [s["k_cache"].double(), s["v_cache"].double()]
    first = 0
    for b, (length, n) in enumerate(zip(lens, new)):
        pos = torch.arange(length - n, length, device=out[0].device)
        at = s["page_table"][b].long()[torch.div(pos, case["page"], rounding_mode="floor")]
        for h in range(case["kv_heads"]):
            for c, x in zip(out, (s["k"], s["v"])):
                c[at, h, pos % case["page"]] = x[first: first + n, h].double()
        first += n
    return out


def _exact_pages(case, s):
    """The caches alone: which page's content ends up where, step by step (tables and counts are whole numbers)."""
    page, lens = case["page"], _row_lens(case)
    table, refs = s["page_table"].tolist(), s["refs"].tolist()
    moved = {}
    if case["what"] == "fork":
        free = [p for p, r in enumerate(refs) if r == 0]
        for i in range(case["n"]):
            full, part = divmod(lens[i % case["seqs"]], page)
            if part:
                moved[free.pop(0)] = table[i % case["seqs"]][full]
    else:
        for row in s["ended"].tolist():
            for p in table[row]:
                if p >= 0:
                    refs[p] -= 1
        live = [p for p, r in enumerate(refs) if r > 0]
        holes = [p for p in range(len(live)) if refs[p] == 0]
        moved = dict(zip(holes, (p for p in live if p >= len(live))))
    to, frm = (torch.tensor(x, dtype=torch.int64, device=s["k"].device) for x in (list(moved), list(moved.values())))
    caches = [s["k"].double(), s["v"].double()]
    for c in caches:
        for layer in c:
            layer.index_copy_(0, to, layer.index_select(0, frm))
    return caches + [None] * (3 if case["what"] == "fork" else 4)


def _exact_w4(s):
    g, (n, half) = s["group"], s["qweight"].shape
    k = 2 * half
    code = torch.empty((n, k), dtype=torch.float64, device=s["x"].device)
    code[:, 0::2], code[:, 1::2] = (s["qweight"] % 16).double(), torch.div(s["qweight"], 16, rounding_mode="floor").double()
    scale = s["wscales"].double().repeat_interleave(g, 1)
    if s["wzeros"] is None:
        code -= 16 * (code >= 8)
        shift = 0.0
    elif s["wzeros"].dtype == torch.uint8:
        z = torch.empty((n, 2 * s["wzeros"].shape[1]), dtype=torch.float64, device=code.device)
        z[:, 0::2], z[:, 1::2] = (s["wzeros"] % 16).double(), torch.div(s["wzeros"], 16, rounding_mode="floor").double()
        shift = -scale * z[:, : k // g].repeat_interleave(g, 1)
    else:
        shift = s["wzeros"].double().repeat_interleave(g, 1)
    x = s["x"].double()
    if s["h"]:
        x = x.view(x.shape[0], -1, s["h"]) @ _hadamard(s["h"], torch.float64, x.device)
        x = x.reshape(x.shape[0], k)
    y = x @ (code * scale + shift).t()
    return y if s["bias_t"] is None else y + s["bias_t"].double()
