"""Attention of sequences that share pages (kv_shared's plan, paged_attention(shared=)) against plain loops in 64 bits over every
sequence's own table.

Tolerance as in tests/test_gpu_attention.py: the output is rounded once (u |o|); the probabilities are rounded to the
products' 16 bits, relative u each (u W, W = sum_j p_j |v_j|); scores are fp32 sums of D exact products, off by
(D + 4) 2^-24 R, which moves each p by twice that; sums over keys are fp32 (2^-11 W with the parts' joining). fp16
probabilities are held 2^6 to 2^14 times as large as they are: what vanishes is below 2^-24 of a row's largest."""
import math

import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import serving, step

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Forks:
    """Groups of sequences: groups[i] = (tokens that are shared, [every sequence's tokens beyond them, None: it has ended]); their
    rows of the table in random order. Slots that hold no token are NaN."""

    def __init__(self, dev, groups, hq, h, d, page=16, dtype=torch.bfloat16, int8=False, seed=0, order="phtd", spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.page = dtype, page
        rows = [(i, own) for i, (_, owns) in enumerate(groups) for own in owns]
        rows = [rows[i] for i in torch.randperm(len(rows), generator=g).tolist()]
        self.lens = [0 if own is None else groups[i][0] + own for i, own in rows]
        full = [n // page for n, _ in groups]
        total = sum(full) + sum(max(0, -(-n // page) - full[i]) for n, (i, own) in zip(self.lens, rows) if own is not None) + spare
        place = torch.randperm(total, generator=g).tolist()
        common = [[place.pop() for _ in range(n)] for n in full]
        width = width or max(1, max(-(-n // page) for n in self.lens))
        table = torch.full((len(rows), width), -1, dtype=torch.int32)
        used = torch.zeros(total, page, dtype=torch.bool)
        for b, (i, own) in enumerate(rows):
            if own is None:
                continue
            n = -(-self.lens[b] // page)
            entries = (common[i] + [place.pop() for _ in range(max(0, n - full[i]))])[:n]
            table[b, :n] = torch.tensor(entries, dtype=torch.int32)
            for j in range(self.lens[b]):
                used[entries[j // page], j % page] = True
        shape = (total, h, page, d)
        k, v = (torch.randn(shape, generator=g) for _ in range(2))
        k[..., ::7] *= 3
        self.q = torch.randn((len(rows), hq, d), generator=g).to(dtype).to(dev)
        self.table, self.kv_lens = table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev)
        hole = ~used[:, None, :, None].expand(shape)
        self.ks = self.vs = None
        if int8:
            s = [(x.abs().amax(-1) / 127).clamp_min(1e-10) for x in (k, v)]
            k, v = (torch.round(x / y[..., None]).to(torch.int8) for x, y in zip((k, v), s))
            self.k64, self.v64 = (x.double() * y[..., None].double() for x, y in zip((k, v), s))
            self.ks, self.vs = (self._order(y.masked_fill(~used[:, None, :].expand(shape[:3]), math.nan)[..., None], order, dev)[..., 0] for y in s)
        else:
            k, v = k.to(dtype), v.to(dtype)
            self.k64, self.v64 = k.double(), v.double()
            k, v = k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan)
        self.k, self.v = (self._order(x, order, dev) for x in (k, v))

    @staticmethod
    def _order(x, order, dev):
        perm = ["phtd".index(c) for c in order]
        x = x.to(dev).permute(perm).contiguous()
        return x.permute([perm.index(i) for i in range(4)])

    def plan(self):
        return ck.kv_shared(self.table, self.kv_lens, self.page, least=0)

    def run(self, plan=None, **kw):
        return ck.paged_attention(self.q, self.k, self.v, self.table, self.kv_lens, k_scale=self.ks, v_scale=self.vs,
                                  shared=self.plan() if plan is None else plan, **kw)

    def check(self, y, lens=None, **kw):
        lens = self.lens if lens is None else lens
        o, w, r = serving.attention(self.q.double().cpu().numpy(), self.k64.numpy(), self.v64.numpy(), self.table.cpu().numpy(), lens, None, **kw)
        u, d = U[self.dtype], self.q.shape[2]
        err = np.abs(y.double().cpu().numpy() - o)
        tol = u * np.abs(o) + (u + 2 ** -11 + 2.2 * (d + 4) * 2.0 ** -24 * r[..., None]) * w \
            + max(lens, default=0) * 2.0 ** -24 * float(self.v64.abs().max()) * (self.dtype == torch.float16) + 1e-30
        tol[w == 0] = 0
        assert np.isfinite(y.float().cpu().numpy()).all()
        assert (err <= tol).all(), f"{(err > tol).mean():.3%} out, worst {(err / np.maximum(tol, 1e-300)).max():.2f} of the tolerance"


def read(plan, b):
    """(groups, start) of a plan, as the oracle gives them."""
    p = plan.cpu().tolist()
    n, start, members, groups = p[0], p[4:4 + b], p[4 + b:4 + 2 * b], p[4 + 2 * b:4 + 4 * b]
    found = [groups[4 * i:4 * i + 4] for i in range(n)]
    for tokens, lead, first, count in found:
        assert lead == members[first]
    return [(tokens, members[first:first + count]) for tokens, lead, first, count in found], start


MIXED = [(33, [5, 1, 20, None]), (0, [7]), (64, [0, 3]), (200, [1] * 9), (16, [40, None]), (0, [None, 2, 3]), (150, [100, 0, 64])]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256])
@pytest.mark.parametrize("seed", [0, 1])
def test_plan(gpu_device, page, seed):
    s = Forks(gpu_device, MIXED, 2, 1, 8, page=page, seed=seed)
    assert read(s.plan(), len(s.lens)) == step.shared(s.table.cpu().tolist(), s.lens, page)


@pytest.mark.gpu
def test_plans_of_other_tables(gpu_device):
    """No sequence, one, entries that are no page, shared runs that end early, lengths beyond the table, thousands of rows."""
    def plan(table, lens, page):
        t = torch.tensor(table, dtype=torch.int32, device=gpu_device).view(len(lens), -1)
        got = read(ck.kv_shared(t, torch.tensor(lens, dtype=torch.int32, device=gpu_device), page), len(lens))
        assert got == step.shared(table, lens, page)
        return got

    assert ck.kv_shared(torch.zeros((0, 3), dtype=torch.int32, device=gpu_device), torch.zeros(0, dtype=torch.int32, device=gpu_device), 16).shape == (4,)
    assert plan([[3, 4]], [20], 16) == ([], [0])
    assert plan([[3, 4], [3, 5]], [20, 30], 16) == ([(16, [0, 1])], [16, 16])
    assert plan([[3, 4], [3, 4]], [20, 19], 16) == ([(19, [0, 1])], [19, 19])
    assert plan([[-1, 4], [-1, 4]], [20, 20], 16) == ([], [0, 0])
    assert plan([[3, -1, 5], [3, -1, 5]], [40, 40], 16) == ([(16, [0, 1])], [16, 16])
    assert plan([[7, 8], [7, 8]], [900, 1000], 16) == ([(32, [0, 1])], [32, 32])
    assert plan([[7, 8], [7, 8], [7, 1]], [32, -4, 0], 16) == ([], [0, 0, 0])
    g = torch.Generator().manual_seed(3)
    table = torch.randint(0, 40, (2500, 1), generator=g).repeat(1, 70)
    table[:, 65] += torch.randint(0, 3, (2500,), generator=g)
    plan(table.tolist(), torch.randint(0, 71, (2500,), generator=g).tolist(), 1)


HEADS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (32, 2, 64), (34, 2, 128), (6, 2, 80), (5, 1, 8), (14, 2, 96), (4, 1, 256), (16, 16, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads(gpu_device, hq, h, d, dtype):
    print(f"[shared] {hq}/{h} x {d} {dtype}", flush=True)
    s = Forks(gpu_device, MIXED, hq, h, d, dtype=dtype)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,h,d", [(8, 2, 128), (3, 3, 64), (17, 1, 16), (8, 8, 256), (6, 2, 80)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes(gpu_device, hq, h, d, dtype):
    print(f"[shared] int8 {hq}/{h} x {d} {dtype}", flush=True)
    s = Forks(gpu_device, MIXED, hq, h, d, dtype=dtype, int8=True)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 8, 32, 128, 1024])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("order", ["phtd", "pthd", "htpd"])
def test_pages(gpu_device, page, int8, order):
    print(f"[shared] page {page} int8 {int8} {order}", flush=True)
    s = Forks(gpu_device, [(300, [5, 200, 1]), (1030, [0, 9]), (70, [None, 3])], 8, 2, 64, page=page, int8=int8, order=order)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("members", [2, 5, 16, 17, 70])
@pytest.mark.parametrize("tokens", [1, 16, 127, 129, 5000])
def test_members(gpu_device, members, tokens):
    """Rows that fill one tile, end inside one or take several, over one piece or many."""
    print(f"[shared] {members} members of {tokens} tokens", flush=True)
    s = Forks(gpu_device, [(tokens, [i % 3 for i in range(members)])], 8, 2, 128, page=1)
    s.check(s.run())


@pytest.mark.gpu
def test_many_groups(gpu_device):
    g = torch.Generator().manual_seed(5)
    groups = [(int(torch.randint(1, 700, (1,), generator=g)), torch.randint(0, 90, (int(torch.randint(1, 7, (1,), generator=g)),), generator=g).tolist())
              for _ in range(75)]
    s = Forks(gpu_device, groups, 4, 2, 64, page=8)
    s.check(s.run())


@pytest.mark.gpu
def test_nothing_shared(gpu_device):
    """Without groups the results are the single-token kernel's, bit for bit."""
    s = Forks(gpu_device, [(0, [n]) for n in (1, 333, 17, 1024)] + [(0, [None])], 8, 2, 128)
    assert torch.equal(s.run(), ck.paged_attention(s.q, s.k, s.v, s.table, s.kv_lens))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scale(gpu_device, scale):
    s = Forks(gpu_device, MIXED, 8, 2, 64)
    s.check(s.run(scale=scale), scale=scale)


@pytest.mark.gpu
def test_pages_that_are_none(gpu_device):
    """Entries out of the cache's range, in what is shared and behind it."""
    s = Forks(gpu_device, [(128, [20, 30, 40]), (64, [50, 0])], 8, 2, 64)
    lead = s.table[:, 0].tolist()
    first = [b for b in range(5) if lead[b] == lead[0]]
    for b in first:
        s.table[b, 3] = 10 ** 6
    s.table[first[0], -1] = -1
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_plan_made_before(gpu_device, int8):
    """Sequences that have grown since, one that has ended, one that is shorter than what was shared."""
    s = Forks(gpu_device, [(100, [30, 40, 50, 60]), (40, [8, 9])], 8, 2, 64, int8=int8)
    lens = s.lens
    group = [b for b in range(6) if lens[b] > 100]
    early = [n - 5 if n else 0 for n in lens]
    s.kv_lens = torch.tensor(early, dtype=torch.int32, device=gpu_device)
    plan = s.plan()
    late = list(lens)
    late[group[1]], late[group[2]] = 0, 70
    s.kv_lens = torch.tensor(late, dtype=torch.int32, device=gpu_device)
    s.check(s.run(plan), late)


@pytest.mark.gpu
def test_no_numbers_out_of_sight(gpu_device):
    """Infinities and NaN behind a sequence's end in pages that others go on in do not reach its result (Forks fills them with NaN);
    NaN in a shared key reaches the rows that see it alone."""
    s = Forks(gpu_device, [(48, [5, 6]), (32, [9, 8])], 4, 2, 64)
    base = s.run()
    lead = s.table[:, 0].tolist()
    s.v[lead[0], 0, 3, 5] = float("nan")
    y = s.run()
    hit = [b for b in range(4) if lead[b] == lead[0]]
    bad = y.isnan()
    assert bad[hit][:, :2, 5].all() and bad.sum() == 2 * len(hit)
    other = [b for b in range(4) if b not in hit]
    assert torch.equal(y[other], base[other])


@pytest.mark.gpu
def test_out_strides_streams_and_graphs(gpu_device):
    s = Forks(gpu_device, MIXED, 8, 2, 64)
    want = s.run()
    wide = torch.full((len(s.lens), 8, 128), 7.0, dtype=torch.bfloat16, device=gpu_device)
    s.run(out=wide[..., 32:96])
    assert torch.equal(wide[..., 32:96], want) and (wide[..., :32] == 7).all() and (wide[..., 96:] == 7).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = s.plan()
        y = [s.run(plan), s.run(plan, scale=0.5)]
    for i in range(4):
        s.q.copy_(torch.randn(s.q.shape, device=gpu_device))
        graph.replay()
        eager = [s.run(), s.run(scale=0.5)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(y, eager))


@pytest.mark.gpu
def test_the_same_every_time(gpu_device):
    s = Forks(gpu_device, [(9000, [50] * 20), (300, [700] * 5)], 16, 2, 128)
    want = s.run()
    for _ in range(5):
        assert torch.equal(s.run(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [31, 32, 33, 64, 65, 97, 128, 129, 257])
@pytest.mark.parametrize("d,int8", [(64, False), (64, True), (128, False), (128, True), (256, False), (256, True), (72, False), (144, True)])
def test_rows_of_a_tile(gpu_device, rows, d, int8):
    """Groups whose rows end at every boundary between waves and tiles, over a few tiles and over many workgroups' pieces."""
    print(f"[shared] {rows} rows x {d} int8 {int8}", flush=True)
    s = Forks(gpu_device, [(200, [i % 2 for i in range(rows)]), (3000, [3] * 5)], 2, 2, d, page=8, int8=int8, dtype=torch.float16 if rows % 2 else torch.bfloat16)
    s.check(s.run())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [32, 33, 64, 65, 128, 192, 193, 256, 257, 320, 449, 512, 513, 577, 1024])
@pytest.mark.parametrize("d,int8", [(64, False), (64, True), (128, False), (128, True), (256, False), (256, True)])
def test_tiles(gpu_device, tokens, d, int8):
    """One tile to more than a ring holds, in one piece and with the next group's behind them in the same workgroup."""
    s = Forks(gpu_device, [(tokens, [1, 2, 0])] + [(tokens - 1, [2, 1])] * 9, 8, 8, d, page=1, int8=int8)
    s.check(s.run())


@pytest.mark.gpu
def test_long_and_short_groups(gpu_device):
    """Workgroups that end one group's tiles, have others whole and begin a third's; more groups than lanes."""
    groups = [(20000, [5] * 3)] + [(1 + 13 * i % 90, [i % 4, 1]) for i in range(150)] + [(7000, [60, 1, 9])]
    s = Forks(gpu_device, groups, 4, 4, 128, page=4)
    s.check(s.run())


@pytest.mark.gpu
def test_two_at_once(gpu_device):
    """Calls of two streams and of two threads at the same time do not share working space."""
    import threading
    sets = [Forks(gpu_device, [(4000, [50] * 12), (90, [3, 5])], 8, 2, 128, seed=i) for i in range(2)]
    want = [s.run() for s in sets]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(sets[i].run())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys) and len(got[0]) == len(got[1]) == 20


@pytest.mark.gpu
def test_plan_of_anything(gpu_device):
    """A plan that kv_shared did not write: whatever its numbers say, every access stays inside, and the next call is right."""
    s = Forks(gpu_device, MIXED, 8, 2, 64)
    want, plan = s.run(), s.plan()
    g = torch.Generator().manual_seed(1)
    for i in range(12):
        odd = torch.randint(-3, 40, plan.shape, generator=g, dtype=torch.int32) if i % 3 else torch.randint(-2 ** 31, 2 ** 31 - 1, plan.shape, generator=g, dtype=torch.int64).int()
        odd[0] = (i % 4) * 3
        if i % 2:
            odd[1], odd[2] = 2 ** 31 - 1, 0                 # worth sharing
        s.run(odd.to(gpu_device))
    assert torch.equal(s.run(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_pages_far_into_a_cache(gpu_device, int8):
    """Offsets beyond 32 bits, in values and in bytes: the same as in a cache that holds these pages alone."""
    s = Forks(gpu_device, [(500, [40, 0, 7]), (100, [300, 2])], 8, 4, 128, page=64, int8=int8)
    want, n = s.run(), s.k.shape[0]
    pages = (1 << 32) // (4 * 64 * 128) + n + 5
    far = torch.arange(pages - 1, pages - 1 - n, -1, device=gpu_device)

    def spread(x):
        y = torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device=gpu_device)
        y[far] = x
        return y

    s.k, s.v = spread(s.k), spread(s.v)
    if int8:
        s.ks, s.vs = spread(s.ks), spread(s.vs)
    s.table = torch.where(s.table < 0, s.table, pages - 1 - s.table)
    assert torch.equal(s.run(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_what_sharing_has_to_save(gpu_device, int8):
    """Below `least` bytes every sequence is attended by itself, bit for bit; at it the groups' are shared."""
    s = Forks(gpu_device, [(128, [5, 1, 20]), (64, [0, 3]), (0, [70])], 8, 2, 64, page=64, int8=int8)
    alone = ck.paged_attention(s.q, s.k, s.v, s.table, s.kv_lens, k_scale=s.ks, v_scale=s.vs)
    shared = s.run()
    saved = (2 * 128 + 64) * 2 * 64 * 2 * (1 if int8 else 2)
    assert saved % 1024 == 0 and not torch.equal(alone, shared)
    for least, want in ((0, shared), (saved, shared), (saved + 1024, alone), (ck.kv.LEAST_SHARED, alone), (1 << 60, alone)):
        assert torch.equal(s.run(ck.kv_shared(s.table, s.kv_lens, 64, least)), want)
    assert torch.equal(s.run(ck.kv_shared(s.table, s.kv_lens, 64)), alone)
    assert read(ck.kv_shared(s.table, s.kv_lens, 64), 6) == read(s.plan(), 6)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [7, 8, 9, 63, 64, 65, 127, 129, 705, 1023, 1024, 1025, 2047, 2048, 2049])
def test_plans_of_many_sequences(gpu_device, rows):
    g = torch.Generator().manual_seed(rows)
    table = torch.randint(-1, max(2, rows // 5), (rows, 1), generator=g).repeat(1, 9)
    table[:, 5] += torch.randint(0, 2, (rows,), generator=g)
    lens = torch.randint(0, 73, (rows,), generator=g)
    plan = ck.kv_shared(table.int().to(gpu_device), lens.int().to(gpu_device), 8, least=0)
    assert read(plan, rows) == step.shared(table.tolist(), lens.tolist(), 8)
