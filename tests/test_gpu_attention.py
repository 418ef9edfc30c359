"""Attention over a paged cache (kitchen_amd.paged_attention) against plain loops in 64 bits.

Tolerance, for outputs of unit roundoff u (bf16 2^-8, fp16 2^-11): the output is rounded once (u |o|); the
probabilities are rounded to 16 bits before the product with V, relative u each, so the sum moves by at
most u W with W = sum_j p_j |v_j| (an int8 cache's scale is multiplied in first: the same single rounding);
the scores are fp32 sums of D exact products in any order, off by at most (D + 4) 2^-24 R with R the
largest sum_d |q_d k_jd| scale, which changes each p by a factor e^(2 err), the sums over keys likewise
(fp32, pairwise over lanes: below 2^-12 W for the lengths here). fp16 probabilities below 2^-24 of a row's
largest may vanish: at most 2^-24 of the largest |v| per key."""
import math

import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import serving

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Setup:
    """A cache with every sequence's pages in random places; slots that hold no token are NaN."""

    def __init__(self, dev, lens, hq, h, d, page=16, dtype=torch.bfloat16, int8=False, new=None, seed=0, order="phtd",
                 spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.int8, self.dtype = list(lens), new, int8, dtype
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + spare
        width = width or max(1, max(counts, default=1))
        place = torch.randperm(pages, generator=g).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, c in enumerate(counts):
            table[b, :c] = torch.tensor(place[:c], dtype=torch.int32)
            place = place[c:]
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                used[table[b, j // page], j % page] = True
        shape = (pages, h, page, d)
        k, v = (torch.randn(shape, generator=g) for _ in range(2))
        k[..., ::7] *= 3
        self.tok = len(lens) if new is None else sum(new)
        self.q = torch.randn((self.tok, hq, d), generator=g).to(dtype).to(dev)
        self.cu = None if new is None else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
        self.table, self.kv_lens = table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev)
        hole = ~used[:, None, :, None].expand(shape)
        self.ks = self.vs = None
        if int8:
            s = [(x.abs().amax(-1) / 127).clamp_min(1e-10) for x in (k, v)]
            k, v = (torch.round(x / y[..., None]).to(torch.int8) for x, y in zip((k, v), s))
            self.k64, self.v64 = (x.double() * y[..., None].double() for x, y in zip((k, v), s))
            s = [y.masked_fill(~used[:, None, :].expand(shape[:3]), math.nan) for y in s]
            self.ks, self.vs = (self._order(y[..., None], order, dev)[..., 0] for y in s)
        else:
            k, v = k.to(dtype), v.to(dtype)
            self.k64, self.v64 = k.double(), v.double()
            k, v = k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan)
        self.k, self.v = (self._order(x, order, dev) for x in (k, v))

    @staticmethod
    def _order(x, order, dev):
        """The same tensor with its dimensions (page, head, token, value) in another order in memory."""
        perm = ["phtd".index(c) for c in order]
        x = x.to(dev).permute(perm).contiguous()
        return x.permute([perm.index(i) for i in range(4)])

    def run(self, **kw):
        return ck.paged_attention(self.q, self.k, self.v, self.table, self.kv_lens, cu_q=self.cu, k_scale=self.ks,
                                  v_scale=self.vs, **kw)

    def check(self, y, q=None, **kw):
        q = self.q if q is None else q
        o, w, r = serving.attention(q.double().cpu().numpy(), self.k64.numpy(), self.v64.numpy(), self.table.cpu().numpy(),
                                    self.lens, None if self.cu is None else self.cu.cpu().numpy(), **kw)
        u, d = U[self.dtype], q.shape[2]
        err = np.abs(y.double().cpu().numpy() - o)
        vmax = float(self.v64.abs().max())
        tol = u * np.abs(o) + (u + 2 ** -11 + 2.2 * (d + 4) * 2.0 ** -24 * r[..., None]) * w \
            + max(self.lens, default=0) * 2.0 ** -24 * vmax * (self.dtype == torch.float16) + 1e-30
        tol[w == 0] = 0                        # rows that see nothing are zeros exactly
        worst = (err / np.maximum(tol, 1e-300))
        assert np.isfinite(y.float().cpu().numpy()).all()
        assert (err <= tol).all(), f"{(err > tol).mean():.3%} out, worst {worst.max():.2f} of the tolerance"


HEADS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (32, 2, 64), (34, 2, 128), (6, 2, 80), (5, 1, 8), (14, 2, 96), (4, 1, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_heads(gpu_device, hq, h, d, dtype):
    print(f"[attention] decode {hq}/{h} x {d} {dtype}", flush=True)
    s = Setup(gpu_device, [1, 0, 15, 16, 17, 333, 1024, 70], hq, h, d, dtype=dtype)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 8, 32, 128, 1024])
@pytest.mark.parametrize("int8", [False, True])
def test_decode_pages(gpu_device, page, int8):
    print(f"[attention] decode page {page} int8 {int8}", flush=True)
    s = Setup(gpu_device, [130, 1, 0, 513, 64], 8, 2, 64, page=page, int8=int8)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d", [(8, 2, 128), (3, 3, 64), (17, 1, 16), (8, 8, 256), (6, 2, 80)])
def test_decode_int8(gpu_device, hq, h, d):
    print(f"[attention] decode int8 {hq}/{h} x {d}", flush=True)
    s = Setup(gpu_device, [1, 40, 0, 700, 2049], hq, h, d, int8=True, dtype=torch.float16 if h == 3 else torch.bfloat16)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (64, 4), (100, 100), (1000, 17), (5000, 2)])
def test_decode_window(gpu_device, window, sinks):
    print(f"[attention] decode window {window} sinks {sinks}", flush=True)
    s = Setup(gpu_device, [1, 2, 63, 64, 65, 700, 0, 1500], 8, 4, 64)
    s.check(s.run(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[20011], [33000, 5], [1] * 200, [0, 0, 0], [3000] * 7])
def test_decode_lengths(gpu_device, lens):
    """One long sequence (split over its length and joined), a ragged pair, many short ones, none."""
    print(f"[attention] decode lengths {lens[:4]} x {len(lens)}", flush=True)
    s = Setup(gpu_device, lens, 4, 1, 64, page=64)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("new,past", [([1], [0]), ([77], [0]), ([16, 1, 0, 33], [0, 0, 5, 100]), ([64, 65, 63], [64, 1, 0]),
                                      ([200, 3], [1000, 500]), ([300], [0]), ([1, 1, 1], [40, 0, 9])])
@pytest.mark.parametrize("hq,h,d,dtype,int8", [(4, 2, 128, torch.bfloat16, False), (3, 1, 64, torch.float16, False),
                                               (2, 2, 80, torch.bfloat16, True), (2, 1, 256, torch.float16, False)])
def test_prompt(gpu_device, new, past, hq, h, d, dtype, int8):
    print(f"[attention] prompt {new} behind {past}, {hq}/{h} x {d} {dtype} int8 {int8}", flush=True)
    s = Setup(gpu_device, [a + b for a, b in zip(new, past)], hq, h, d, dtype=dtype, int8=int8, new=new)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (30, 4), (64, 0), (128, 64), (200, 5), (4096, 1)])
def test_prompt_window(gpu_device, window, sinks):
    print(f"[attention] prompt window {window} sinks {sinks}", flush=True)
    s = Setup(gpu_device, [500, 130, 64], 4, 2, 64, new=[400, 130, 10])
    s.check(s.run(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 8, 64, 256])
@pytest.mark.parametrize("order", ["pthd", "hptd", "tphd"])
def test_prompt_pages_and_orders(gpu_device, page, order):
    print(f"[attention] prompt page {page} order {order}", flush=True)
    s = Setup(gpu_device, [150, 70], 4, 2, 64, page=page, new=[90, 70], order=order, int8=order == "hptd")
    s.check(s.run())
    t = Setup(gpu_device, [150, 70], 4, 2, 64, page=page, order=order, int8=order == "hptd")
    t.check(t.run())


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_missing_pages(gpu_device, ragged):
    """Table entries that are no page (given back behind a window, or out of range) hold nothing."""
    s = Setup(gpu_device, [200, 90, 33], 4, 2, 64, new=[50, 90, 1] if ragged else None)
    s.table[0, 1] = -1
    s.table[0, 5:9] = 1 << 30
    s.table[1, :] = -7
    s.check(s.run())


@pytest.mark.gpu
def test_short_cache_and_table(gpu_device):
    """More new tokens than the cache holds (positions below 0 see nothing); lens past the table's width."""
    s = Setup(gpu_device, [10, 48], 4, 2, 64, new=[25, 40])
    s.check(s.run())
    s.lens[1] = 4000
    s.kv_lens.copy_(torch.tensor(s.lens))
    s.check(s.run())
    t = Setup(gpu_device, [112, 3], 4, 2, 64, new=None)
    t.lens[0] = 5000
    t.kv_lens.copy_(torch.tensor(t.lens))
    t.check(t.run())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_values_do_not_matter(gpu_device, bad, what, d):
    """Infinities and NaN in tokens that a query does not see (later ones, behind the window) leave it alone;
    queries that see them get what the formula gives."""
    s = Setup(gpu_device, [300, 90], 4, 2, d, new=[200, 90])
    page, slot = int(s.table[0, 170 // 16]), 170 % 16        # position 170: seen by 170 .. 233 of window 64
    getattr(s, what)[page, 1, slot, 3] = bad
    y = s.run(window=64, sinks=2)
    heads = torch.arange(4, device=gpu_device) >= 2
    pos = torch.arange(100, 300, device=gpu_device)
    sees = (pos >= 170) & (pos < 170 + 64)
    clean = torch.cat([~(sees[:, None] & heads), torch.ones((90, 4), dtype=torch.bool, device=gpu_device)])
    assert torch.isfinite(y[clean].float()).all()
    touched = y[~clean].float()
    if what == "v":
        assert torch.equal(torch.isfinite(touched), torch.arange(d, device=gpu_device).expand_as(touched) != 3)
    elif math.isnan(bad):
        assert torch.isnan(touched).all()
    getattr(s, what)[page, 1, slot, 3] = 0
    z = s.run(window=64, sinks=2)
    assert torch.equal(y[clean], z[clean])


@pytest.mark.gpu
def test_scores_at_the_ends(gpu_device):
    """Equal scores, scores far apart (all weight on one key), a scale of 0 and a negative one."""
    s = Setup(gpu_device, [100, 37], 4, 2, 64)
    for scale in (0.0, 40.0, -0.3, 1e-6):
        s.check(s.run(scale=scale), scale=scale)
    t = Setup(gpu_device, [100, 37], 4, 2, 64, new=[60, 37])
    for scale in (0.0, 40.0, -0.3):
        t.check(t.run(scale=scale), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_strided_queries_and_output(gpu_device, ragged):
    """q as a slice of a fused projection, out as a slice of a wider tensor (its other columns untouched), and rows
    that have to be copied first."""
    s = Setup(gpu_device, [40, 90, 7], 4, 2, 64, new=[33, 90, 7] if ragged else None)
    wide = torch.randn((s.tok, 12, 64), device=gpu_device).to(torch.bfloat16)
    wide[:, 3:7] = s.q
    out = torch.full((s.tok, 8, 64), 7.0, dtype=torch.bfloat16, device=gpu_device)
    want = s.run()
    s.q = wide[:, 3:7]
    got = s.run(out=out[:, 2:6])
    assert got.data_ptr() == out[:, 2:6].data_ptr() and torch.equal(got, want)
    assert (out[:, :2] == 7).all() and (out[:, 6:] == 7).all()
    odd = torch.zeros(s.tok * 256 + 1, dtype=torch.bfloat16, device=gpu_device)
    odd[1:] = s.q.reshape(-1)
    s.q = odd[1:].view(s.tok, 4, 64)
    assert torch.equal(s.run(), want)


@pytest.mark.gpu
def test_same_result_every_time_and_on_another_stream(gpu_device):
    s = Setup(gpu_device, [9000, 100, 4000], 8, 2, 128)
    t = Setup(gpu_device, [500, 300], 8, 2, 128, new=[400, 300])
    want = s.run(), t.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [(s.run(), t.run()) for _ in range(3)]
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.gpu
def test_in_a_graph(gpu_device):
    """Captured once, replayed with longer sequences and eager work in between."""
    s = Setup(gpu_device, [2000, 30, 700], 8, 2, 64)
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = s.run()
    for lens in ([2000, 30, 700], [5, 30, 0], [1999, 1, 650]):
        s.lens[:] = lens
        s.kv_lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        s.check(y)
        assert torch.equal(s.run(), y)


@pytest.mark.gpu
def test_caches_past_4_gib_elements(gpu_device):
    """Pages whose offsets pass 32 bits, in elements too."""
    h, d, page, pages = 8, 128, 64, (1 << 32) // (8 * 128 * 64) + 40
    big = torch.empty((pages, h, page, d), dtype=torch.bfloat16, device=gpu_device)
    s = Setup(gpu_device, [150, 70], 16, h, d, page=page, new=None)
    n = s.k.shape[0]
    big[-n:] = s.k
    s.table = torch.where(s.table >= 0, s.table + (pages - n), s.table)
    y = ck.paged_attention(s.q, big, big, s.table, s.kv_lens)
    small = ck.paged_attention(s.q, s.k, s.k, torch.where(s.table >= 0, s.table - (pages - n), s.table), s.kv_lens)
    assert torch.equal(y, small)
    q, cu = s.q.repeat(3, 1, 1), torch.tensor([0, 5, 6], dtype=torch.int32, device=gpu_device)
    y = ck.paged_attention(q, big, big, s.table, s.kv_lens, cu_q=cu)
    small = ck.paged_attention(q, s.k, s.k, torch.where(s.table >= 0, s.table - (pages - n), s.table), s.kv_lens, cu_q=cu)
    assert torch.equal(y, small)
    del big


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d", [(8, 2, 128), (3, 3, 64), (7, 1, 80), (2, 2, 256)])
@pytest.mark.parametrize("dtype,int8", [(torch.bfloat16, False), (torch.float16, False), (torch.float16, True), (torch.bfloat16, True)])
def test_few_rows_over_a_long_cache(gpu_device, hq, h, d, dtype, int8):
    print(f"[attention] prompt pieces {hq}/{h} x {d} {dtype} int8 {int8}", flush=True)
    s = Setup(gpu_device, [4099, 9, 1500, 0, 2048], hq, h, d, dtype=dtype, int8=int8, new=[3, 9, 40, 0, 1], page=64)
    for kw in ({}, {"window": 1200, "sinks": 5}, {"window": 64}):
        y = s.run(**kw)
        s.check(y, **kw)
        assert torch.equal(y, s.run(**kw))      # the counters are zeros again, the order of arrival changes nothing


@pytest.mark.gpu
def test_pieces_of_infinities_and_hidden_rows(gpu_device):
    print("[attention] prompt pieces with infinities", flush=True)
    s = Setup(gpu_device, [5000], 4, 2, 64, dtype=torch.bfloat16, new=[2], page=64)
    y = s.run()
    last = s.table[0, 4998 // 64]
    s.v[last, 1, 4999 % 64, 3] = math.inf       # seen by the second token only, in the last piece
    z = s.run()
    assert torch.equal(z[0], y[0]) and torch.isinf(z[1, 2:, 3]).all()
    z[1, 2:, 3] = y[1, 2:, 3]
    assert torch.equal(z, y)
    s.kv_lens[0] = 0                            # both tokens before the first one: nothing is seen
    assert (s.run() == 0).all()


@pytest.mark.gpu
def test_pieces_in_a_graph(gpu_device):
    print("[attention] prompt pieces in a graph", flush=True)
    s = Setup(gpu_device, [6000, 3000], 8, 2, 128, new=[5, 7], page=64)
    want = s.run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.run()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = s.run()
    for _ in range(4):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(s.run(), want)
