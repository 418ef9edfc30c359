"""kitchen_amd.kv_append (queries and keys turned by their positions, keys and values into a paged cache) against numpy in 64
bits.

Tolerance. Angles are exact to 2^-32 of a turn at positions up to 2^31; cosine and sine are rounded to fp32 once, the two
products and their sum once each: a turned value is off by 3 x 2^-24 (|a| + |b|) size, then rounded once to the type
(half a step, eps / 2; fp16 below 2^-14: 2^-25), or, in an int8 cache, to half a step of max / 127. What is not turned and
values of a 16-bit cache are equal bit for bit."""
import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import step

E = 3 * 2.0 ** -24 + 2.0 ** -30


class Batch:
    """Sequences of lens tokens, `new` of them new, pages in random places of caches filled with a value."""

    def __init__(self, dev, lens, new, hq, h, d, page=16, dtype=torch.bfloat16, int8=False, seed=0, order="phtd", width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.page, self.dtype, self.int8, self.dev = lens, new, page, dtype, int8, dev
        width = width or max(1, max(-(-n // page) for n in lens))
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        # pages for the new tokens only: the earlier ones are not read
        need = [(b, j) for b, n in enumerate(lens) for j in range(max(0, n - new[b]) // page, -(-n // page))]
        self.pages = len(need) + 2
        place = torch.randperm(self.pages, generator=g)
        for (b, j), p in zip(need, place):
            table[b, j] = p
        self.table, self.kv_lens = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
        self.cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
        qkv = torch.randn((sum(new), hq + 2 * h, d), generator=g).to(dtype).to(dev)
        self.q, self.k, self.v = qkv.split([hq, h, h], 1)
        perm = ["phtd".index(c) for c in order]
        shape = (self.pages, h, page, d)

        def make(dt):
            x = torch.full(shape, 3, dtype=dt, device=dev).permute(perm).contiguous()
            return x.permute([perm.index(i) for i in range(4)])

        self.kc, self.vc = (make(torch.int8 if int8 else dtype) for _ in range(2))
        self.ks, self.vs = (torch.full(shape[:3], 9.0, device=dev) if int8 else None for _ in range(2))

    def run(self, rotary, cu="ragged", **kw):
        return ck.kv_append(self.q, self.k, self.v, self.kc, self.vc, self.table, self.kv_lens, rotary,
                            self.cu if cu == "ragged" else None, self.ks, self.vs, **kw)

    def check(self, q, rotary, **formula):
        f, size = step.frequencies(rotary.dim, **formula)
        size = rotary.size
        pos = np.concatenate([np.arange(n - m, n) for n, m in zip(self.lens, self.new)] or [[]])
        seq = np.repeat(np.arange(len(self.lens)), self.new)
        n = rotary.dim
        a, b = (np.arange(0, n, 2), np.arange(1, n, 2)) if rotary.interleaved else (np.arange(n // 2), np.arange(n // 2, n))

        def turned(x):
            x = x.double().cpu().numpy()
            y = step.turn(x, np.maximum(pos, 0), f, size, rotary.interleaved)
            y[pos < 0] = x[pos < 0]
            slack = np.zeros_like(x)
            slack[..., a] = slack[..., b] = E * size * (np.abs(x[..., a]) + np.abs(x[..., b]))
            slack[pos < 0] = 0
            return y, slack

        half = torch.finfo(self.dtype).eps / 2
        tiny = 2.0 ** -25 if self.dtype == torch.float16 else 1e-39
        y, slack = turned(self.q)
        err = np.abs(q.double().cpu().numpy() - y)
        assert (err <= slack * (1 + half) + half * np.abs(y) + tiny * (slack > 0)).all()
        assert torch.equal(q[..., n:], self.q[..., n:])
        yk, slack = turned(self.k)
        yv = self.v.double().cpu().numpy()
        kc, vc = (x.double().cpu().numpy() for x in (self.kc, self.vc))
        written = np.zeros(kc.shape[:3], dtype=bool)
        table = self.table.cpu().numpy()
        for t, (s, p) in enumerate(zip(seq, pos)):
            if p < 0 or p // self.page >= table.shape[1] or not 0 <= table[s, p // self.page] < self.pages:
                continue
            at = (table[s, p // self.page], slice(None), p % self.page)
            written[at] = True
            if self.int8:
                for got, sc, want, sl in ((kc[at], self.ks[at], yk[t], slack[t]), (vc[at], self.vs[at], yv[t], 0 * slack[t])):
                    scale = np.maximum(np.abs(want).max(-1) / 127, 1e-10)
                    ds = sl.max(-1) / 127 + 2.0 ** -23 * scale
                    assert (np.abs(sc.double().cpu().numpy() - scale) <= ds).all()
                    assert (np.abs(got - want / scale[:, None]) <= 0.5 + (sl + 127 * ds[:, None]) / scale[:, None] + 2.0 ** -16).all()
            else:
                assert (np.abs(kc[at] - yk[t]) <= slack[t] * (1 + half) + half * np.abs(yk[t]) * (slack[t] > 0) + tiny * (slack[t] > 0)).all()
                assert (vc[at] == yv[t]).all()
        assert (kc[~written] == 3).all() and (vc[~written] == 3).all()
        if self.int8:
            assert (self.ks.cpu().numpy()[~written] == 9).all() and (self.vs.cpu().numpy()[~written] == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d,dim", [(1, 1, 8, 8), (4, 4, 64, 64), (32, 8, 128, 128), (7, 1, 80, 80), (5, 5, 80, 40), (6, 2, 96, 24),
                                        (8, 2, 128, 64), (3, 1, 256, 256), (24, 8, 16, 16), (2, 2, 136, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads(gpu_device, hq, h, d, dim, interleaved, dtype):
    print(f"[append] {hq}/{h} x {d}, {dim} turned, interleaved {interleaved} {dtype}", flush=True)
    s = Batch(gpu_device, [5, 33, 0, 1, 70], [5, 2, 1, 1, 40], hq, h, d, dtype=dtype)
    r = ck.Rotary(dim, interleaved=interleaved)
    s.check(s.run(r), r)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 16, 128])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_pages_and_codes(gpu_device, page, int8, interleaved):
    print(f"[append] page {page} int8 {int8} interleaved {interleaved}", flush=True)
    for d, dim in ((128, 128), (80, 40), (64, 16)):
        s = Batch(gpu_device, [130, 1, 0, 513, 64], [60, 1, 2, 1, 64], 4, 2, d, page=page, int8=int8, order="pthd")
        r = ck.Rotary(dim, interleaved=interleaved)
        s.check(s.run(r), r)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [1, 3, 64, 700])
@pytest.mark.parametrize("int8", [False, True])
def test_single_tokens(gpu_device, seqs, int8):
    print(f"[append] {seqs} single tokens int8 {int8}", flush=True)
    lens = [0 if b % 7 == 3 else 1 + 13 * b % 500 for b in range(seqs)]
    s = Batch(gpu_device, lens, [1] * seqs, 8, 2, 64, int8=int8)
    r = ck.Rotary(64)
    s.check(s.run(r, cu=None), r)


@pytest.mark.gpu
@pytest.mark.parametrize("formula", [dict(base=500000.0), dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=8.0, original=4096),
                                     dict(scaling="yarn", factor=40.0, original=2048, base=1e6), dict(base=1.5)], ids=str)
@pytest.mark.parametrize("last", [1000, 131071, 1 << 20, (1 << 30) - 5])
def test_far_positions(gpu_device, formula, last):
    """The formula's angles at any position: exact to 1e-8 there too."""
    print(f"[append] position {last} {formula}", flush=True)
    page = 1 << 20 if last > 1 << 21 else 1024
    if page > 1024:        # a page that holds one token in reach of the test's memory: heads of 8, one page
        s = Batch(gpu_device, [last], [3], 1, 1, 8, page=page, width=1024)
        r = ck.Rotary(8, **formula)
    else:
        s = Batch(gpu_device, [last], [3], 4, 2, 128, page=page)
        r = ck.Rotary(128, **formula)
    s.check(s.run(r), r, **formula)


@pytest.mark.gpu
def test_size_is_the_programs_to_set(gpu_device):
    s = Batch(gpu_device, [300], [20], 2, 1, 64, dtype=torch.float16)
    r = ck.Rotary(64, scaling="yarn", factor=4.0, size=0.75)
    assert r.size == 0.75
    s.check(s.run(r), r, scaling="yarn", factor=4.0)


@pytest.mark.gpu
def test_equals_turning_by_zero_and_writing(gpu_device):
    """At position 0 everything stays as it is: the same bits as kv_write's."""
    lens = [1, 0, 1, 1]
    a, b = (Batch(gpu_device, lens, [1] * 4, 6, 2, 128, int8=True) for _ in range(2))
    q = a.run(ck.Rotary(128), cu=None)
    ck.kv_write(b.k, b.v, b.kc, b.vc, b.table, b.kv_lens, None, b.ks, b.vs)
    assert torch.equal(q, a.q) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
    assert torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs)


@pytest.mark.gpu
def test_in_place_and_into_other_rows(gpu_device):
    r = ck.Rotary(96, interleaved=True)
    s = Batch(gpu_device, [40, 9], [30, 9], 4, 2, 128)
    want = s.run(r)
    wide = torch.full((39, 4, 256), 7.0, dtype=torch.bfloat16, device=gpu_device)
    assert s.run(r, out=wide[..., 64:192]) is not None
    assert torch.equal(wide[..., 64:192], want) and (wide[..., :64] == 7).all() and (wide[..., 192:] == 7).all()
    q = s.q.clone()
    got = ck.kv_append(q, s.k, s.v, s.kc, s.vc, s.table, s.kv_lens, r, s.cu, out=q)
    assert got is q and torch.equal(q, want)


@pytest.mark.gpu
def test_rows_behind_the_last_sequence(gpu_device):
    """A padded batch: rows that belong to no sequence are left as they were, in the output and in the pages."""
    r = ck.Rotary(64)
    s = Batch(gpu_device, [12, 7], [5, 6], 2, 1, 64)
    cu = torch.tensor([0, 3, 8], dtype=torch.int32, device=gpu_device)
    out = torch.full(s.q.shape, 5.0, dtype=torch.bfloat16, device=gpu_device)
    ck.kv_append(s.q, s.k, s.v, s.kc, s.vc, s.table, s.kv_lens, r, cu, out=out)
    assert (out[8:] == 5).all() and not (out[:8] == 5).all()
    s.q, s.k, s.v, s.new = s.q[:8], s.k[:8], s.v[:8], [3, 5]
    s.check(out[:8], r)


@pytest.mark.gpu
def test_pages_that_are_none(gpu_device):
    """Entries out of the cache's range and positions behind the table: nothing is written, queries are turned."""
    r = ck.Rotary(64)
    s = Batch(gpu_device, [40, 40, 40], [40, 20, 4], 2, 1, 64)
    s.table[0, 1], s.table[1, 2] = 10 ** 6, -5
    s.table = s.table[:, :3]
    s.kv_lens = torch.tensor([40, 40, 60], dtype=torch.int32, device=gpu_device)
    s.lens = [40, 40, 60]
    s.check(s.run(r), r)


@pytest.mark.gpu
def test_no_numbers_stay_in_their_pairs(gpu_device):
    s = Batch(gpu_device, [9, 9], [9, 9], 2, 2, 64, dtype=torch.float16)
    s.q[3, 1, 5], s.k[4, 0, 40] = float("nan"), float("inf")
    q = s.run(ck.Rotary(64))
    bad = ~torch.isfinite(q)
    assert bad[3, 1, [5, 37]].all() and bad.sum() == 2
    page, slot = int(s.table[0, 0]), 4
    bad = ~torch.isfinite(s.kc)
    assert bad[page, 0, slot, [8, 40]].all() and bad.sum() == 2
    i8 = Batch(gpu_device, [9, 9], [9, 9], 2, 2, 64, dtype=torch.float16, int8=True)
    i8.k[4, 0, 40], i8.v[2, 1, 3] = float("inf"), float("nan")
    i8.run(ck.Rotary(64))
    page = int(i8.table[0, 0])
    assert i8.ks[page, 0, 4].isnan() and not i8.kc[page, 0, 4].any() and i8.vs[page, 1, 2].isnan()
    assert i8.ks.isnan().sum() == 1 and i8.vs.isnan().sum() == 1


@pytest.mark.gpu
def test_the_same_as_the_cache_method_in_a_graph(gpu_device):
    """PagedKVCache.append, captured and replayed with other tokens and lengths."""
    r = ck.Rotary(64)
    cache = ck.PagedKVCache(2, 40, 2, 64, 16, 3, 200, torch.bfloat16)
    cache.grow([0, 1, 2], [5, 17, 1])
    q, k, v = (torch.randn((3, n, 64), device=gpu_device).to(torch.bfloat16) for n in (4, 2, 2))
    graph = torch.cuda.CUDAGraph()
    cache.append(1, q, k, v, r)
    with torch.cuda.graph(graph):
        out = cache.append(1, q, k, v, r)
    for i in range(3):
        cache.grow([0, 1, 2], [1, 1, 1])
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=gpu_device))
        graph.replay()
        torch.cuda.synchronize()
        other = ck.PagedKVCache(2, 40, 2, 64, 16, 3, 200, torch.bfloat16)
        for name in ("page_table", "lens", "refs", "k", "v"):
            getattr(other, name).copy_(getattr(cache, name))
        other.k[1].zero_()
        want = other.append(1, q, k, v, r)
        assert torch.equal(out, want)
        n = cache.lens.tolist()
        for b in range(3):
            at = int(cache.page_table[b, (n[b] - 1) // 16]), slice(None), (n[b] - 1) % 16
            assert torch.equal(cache.k[1][at], other.k[1][at]) and torch.equal(cache.v[1][at], v[b])
    assert not cache.k[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_pages_far_into_a_cache(gpu_device, int8):
    """Offsets beyond 32 bits, in values and in bytes: what is written is what a cache of these pages alone gets."""
    r = ck.Rotary(128)
    s = Batch(gpu_device, [70, 9, 130], [70, 2, 66], 4, 4, 128, page=64, int8=int8)
    want, n = s.run(r), s.pages
    near = [x.clone() for x in (s.kc, s.vc, *((s.ks, s.vs) if int8 else ()))]
    pages = (1 << 32) // (4 * 64 * 128) + n + 5
    far = torch.arange(pages - 1, pages - 1 - n, -1, device=gpu_device)

    def spread(fill, x):
        y = torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device=gpu_device)
        y[far] = fill
        return y

    s.kc, s.vc = spread(3, s.kc), spread(3, s.vc)
    if int8:
        s.ks, s.vs = spread(9.0, s.ks), spread(9.0, s.vs)
    s.table = torch.where(s.table < 0, s.table, pages - 1 - s.table)
    assert torch.equal(s.run(r), want)
    assert all(torch.equal(x[far], y) for x, y in zip((s.kc, s.vc, *((s.ks, s.vs) if int8 else ())), near))
