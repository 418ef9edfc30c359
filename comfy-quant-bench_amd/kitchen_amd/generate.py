"""A small text decoder on this package's linears and paged cache, and a program that answers with it.

    python -m kitchen_amd.generate [--prompts 4] [--alternatives 2] [--tokens 32] [--int8-cache] [--temperature 0.8 --top-p 0.9]

Every layer's projections are held once, as the converters write them (uint4 codes rotated by Hadamard blocks, fp16
scale and uint4 zero-point per group of 64), and used in two ways: prompts, with rows by the thousand, are multiplied as
int8 codes, those of a norm's output made by the norm itself (rms_norm_quantize); steps of a token per sequence go through
rms_norm and w4a16_linear, whose activations stay in floating point. Keys and values live in a PagedKVCache: ragged
prompts and single tokens are turned by their positions, written to and attended in its pages, a prompt's alternatives
are forks that share its pages, which a step reads once for all of them, and when sequences end their pages are freed
and the others' moved together. Tokens are chosen by sample. Weights are random: it shows the calls and their cost, not
language."""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass

import torch

from . import _lib, kv, ops, step, weights


@dataclass
class Config:
    layers: int = 4
    hidden: int = 2048
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 128
    inner: int = 5120
    vocab: int = 4096
    window: int | None = None      # of every second layer
    sinks: int = 0
    dtype: torch.dtype = torch.bfloat16


class Linear:
    """A projection of 4-bit weights: floating activations up to `few` rows, int8 ones above."""

    GROUP, ROTATE = 64, 256

    def __init__(self, weight: torch.Tensor, few: int = 64):
        self.q, self.s, self.z = weights.quantize_w4a8_asym_weight(weight, self.GROUP, self.ROTATE)
        self.few = few

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[0] <= self.few:
            return ops.w4a16_linear(x, self.q, self.s, self.z, None, self.GROUP, self.ROTATE)
        return ops.w4a8_int8_linear(x, self.q, self.s, None, None, self.z, None, self.GROUP, self.ROTATE, x.dtype)

    def of_norm(self, delta: torch.Tensor | None, x: torch.Tensor):
        """(projection of the norm of x + delta, x + delta); without a delta, of x."""
        if x.shape[0] <= self.few:
            y, x = (step.rms_norm(x), x) if delta is None else step.rms_norm(delta, None, x)
            return self(y), x
        q, s, *h = step.rms_norm_quantize(x, convrot_groupsize=self.ROTATE) if delta is None else \
            step.rms_norm_quantize(delta, None, x, convrot_groupsize=self.ROTATE)
        xw = ops._expansion(self.q, self.z, _lib.ACT_I8, *q.shape, self.s, _lib.stream_of(q))
        y = ops.gemm_w4_group(q, s, self.q if xw is None else xw, self.s, self.z, None, self.q.shape[0], self.GROUP, _lib.ACT_I8, x.dtype)
        return y, h[0] if h else x


# Plain forms of the norm and of the turn by positions, to compare with.

def _norm(x: torch.Tensor) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def _turn(x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """Rotary positions: the halves of a head as pairs turned by pos 10000^(-2i/d)."""
    half = x.shape[-1] // 2
    a = pos[:, None].float() * 10000.0 ** (-torch.arange(half, device=x.device) / half)
    c, s = a.cos()[:, None], a.sin()[:, None]
    u, v = x.float().split(half, -1)
    return torch.cat([u * c - v * s, u * s + v * c], -1).to(x.dtype)


class Decoder:
    """Random weights of a Config with a cache for `seqs` sequences; few: rows up to which linears keep floating
    activations."""

    def __init__(self, config: Config, seqs: int, pages: int, max_tokens: int, page_size: int = 16, int8_cache: bool = False,
                 few: int = 64, seed: int = 0, device="cuda"):
        c = self.config = config
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(n, k):
            return torch.randn((n, k), generator=g, device=device) * k ** -0.5

        self.embedding = matrix(c.vocab, c.hidden).to(c.dtype)
        rows = (c.heads + 2 * c.kv_heads) * c.head_dim
        self.layers = [{"qkv": Linear(matrix(rows, c.hidden), few), "out": Linear(matrix(c.hidden, c.heads * c.head_dim), few),
                        "up": Linear(matrix(2 * c.inner, c.hidden), few), "down": Linear(matrix(c.hidden, c.inner), few)}
                       for _ in range(c.layers)]
        self.cache = kv.PagedKVCache(c.layers, pages, c.kv_heads, c.head_dim, page_size, seqs, max_tokens, c.dtype, int8_cache, device)
        self.rotary = kv.Rotary(c.head_dim, device=device)

    def _forward(self, tokens: torch.Tensor, cu_q, lens: torch.Tensor, shared: torch.Tensor | None = None) -> torch.Tensor:
        """Hidden states of new tokens whose room the cache has; it holds their keys and values afterwards. lens: the
        cache's lengths of the sequences that take part, 0 of the others, whose tokens leave no trace. shared: the plan of
        the pages that they share."""
        c = self.config
        x, delta = torch.nn.functional.embedding(tokens, self.embedding) * c.hidden ** 0.5, None
        for i, layer in enumerate(self.layers):
            y, x = layer["qkv"].of_norm(delta, x)
            q, k, v = y.view(len(tokens), -1, c.head_dim).split([c.heads, c.kv_heads, c.kv_heads], 1)
            q = self.cache.append(i, q, k, v, self.rotary, cu_q, lens=lens)
            window = c.window if i % 2 else None
            y = self.cache.attend(i, q, cu_q, window=window, sinks=c.sinks, lens=lens, shared=None if window else shared)
            y, x = layer["up"].of_norm(layer["out"](y.view(len(tokens), -1)), x)
            gate, up = y.chunk(2, -1)
            delta = layer["down"](torch.nn.functional.silu(gate) * up)
        return step.rms_norm(x) if delta is None else step.rms_norm(delta, None, x)[0]

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return torch.nn.functional.linear(x, self.embedding)

    def prompt(self, prompts: dict[int, list[int]]) -> torch.Tensor:
        """New tokens (or a chunk of them) for some of the sequences; logits [len(prompts), vocab] behind the last of each.
        Without room for all of them the cache stays as it is (cache.check() raises) and the logits say nothing."""
        if not prompts or not all(prompts.values()):
            raise ValueError("a prompt needs tokens")
        cache, dev = self.cache, self.embedding.device
        rows = sorted(prompts)
        news = [len(prompts.get(b, ())) for b in range(cache.lens.shape[0])]
        before = cache.lens.clone()
        cache.grow(rows, [news[b] for b in rows])
        cu_q = torch.tensor([0] + news, device=dev).cumsum(0).to(torch.int32)
        tokens = torch.tensor([t for b in rows for t in prompts[b]], device=dev)
        lens = cache.lens * (cache.lens > before)        # nothing is written where nothing has grown
        x = self._forward(tokens, cu_q, lens)
        return self._logits(x[(cu_q[1:][rows] - 1).long()])

    def step(self, tokens: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """A token more for the sequences `rows` (tokens [seqs], any token for the others, which keep what they hold);
        logits [seqs, vocab]. Without room for all of them the cache stays as it is (cache.check() raises)."""
        cache, before = self.cache, self.cache.lens.clone()
        cache.grow(rows, torch.ones_like(rows))
        lens = cache.lens * (cache.lens > before)        # nothing is written where nothing has grown
        return self._logits(self._forward(tokens, None, lens, cache.shared(lens) if cache.may_share() else None))


def next_tokens(logits: torch.Tensor, u: torch.Tensor, *settings) -> torch.Tensor:
    """sample's tokens as the next step takes them: a row of logits that holds no number has none (-1), and its sequence goes on
    with token 0."""
    return step.sample(logits, u, *settings).clamp_(min=0)


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--prompts", type=int, default=4)
    ap.add_argument("--alternatives", type=int, default=2, help="continuations of each prompt")
    ap.add_argument("--length", type=int, default=500, help="tokens of the longest prompt")
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--window", type=int, default=None)
    ap.add_argument("--int8-cache", action="store_true")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the likeliest token always")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    a = ap.parse_args(argv)
    config = Config(layers=a.layers, window=a.window, sinks=4 if a.window else 0)
    most, seqs = a.length + a.tokens, a.prompts * a.alternatives
    model = Decoder(config, seqs, seqs * (-(-most // 16)) + 1, most, int8_cache=a.int8_cache)
    cache, g = model.cache, torch.Generator().manual_seed(1)
    prompts = {b: torch.randint(config.vocab, (a.length * (b + 1) // a.prompts or 1,), generator=g).tolist() for b in range(a.prompts)}

    def clock():
        torch.cuda.synchronize()
        return time.perf_counter()

    t0 = clock()
    logits = model.prompt(prompts)
    cache.check()
    t1 = clock()
    # alternative i of prompt b is sequence b + i prompts and begins with the i-th best token
    cache.fork([b for _ in range(a.alternatives - 1) for b in range(a.prompts)], range(a.prompts, seqs))
    cache.check()
    tokens = logits.topk(a.alternatives).indices.t().reshape(-1)
    rows = torch.arange(seqs, dtype=torch.int32, device=tokens.device)
    answers = [tokens]
    u = torch.rand((a.tokens, seqs), generator=torch.Generator(device=tokens.device).manual_seed(2), device=tokens.device)
    t2 = clock()
    for i in range(a.tokens):
        if i == a.tokens // 2 and a.alternatives > 1:      # the last alternatives have said enough
            cache.free(rows[-a.prompts:])
            live = cache.compact()
            rows = rows[:-a.prompts]
            print(f"{int(live)} pages are held after {a.prompts} sequences ended")
        tokens = next_tokens(model.step(tokens, rows), u[i], a.temperature, a.top_k, a.top_p, a.min_p)
        answers.append(tokens)
    cache.check()
    t3 = clock()
    said = torch.stack(answers, 1).tolist()
    for b in range(seqs):
        ended = b >= seqs - a.prompts and a.alternatives > 1
        print(f"prompt {b % a.prompts}, alternative {b // a.prompts}:", *said[b][:a.tokens // 2 + 1 if ended else None])
    new = sum(map(len, prompts.values()))
    print(f"{new} prompt tokens in {1e3 * (t1 - t0):.2f} ms; {a.tokens} steps in {1e3 * (t3 - t2):.2f} ms")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
