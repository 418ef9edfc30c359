"""The paged cache's upkeep (kv_write, kv_fork, kv_grow, kv_free, kv_compact) against plain loops: everything is
exact, bytes are copied and integers counted."""
import math
import random

import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import serving


def _layer(dev, lens, h, d, page, dtype, seed=0, fill=None, width=None):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 2
    place = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width or max(1, max(counts))), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(place[:c], dtype=torch.int32)
        place = place[c:]
    cache = [torch.full((pages, h, page, d), 3, dtype=dtype, device=dev) for _ in range(2)]
    return table, cache


def _expect(table, lens, new, page, rows, caches):
    """Every token's row into numpy copies of the caches."""
    t = 0
    for b, n in enumerate(new):
        for i in range(n):
            pos = lens[b] - n + i
            if pos >= 0 and pos // page < table.shape[1]:
                p = int(table[b, pos // page])
                if 0 <= p < caches[0].shape[0]:
                    for c, r in zip(caches, rows):
                        c[p, :, pos % page] = r[t]
            t += 1


@pytest.mark.gpu
@pytest.mark.parametrize("h,d,page", [(1, 64, 16), (8, 128, 16), (3, 80, 8), (2, 8, 1), (5, 256, 64)])
@pytest.mark.parametrize("lens,new", [([1, 17, 40, 16], None), ([30, 0, 5, 64], [30, 0, 3, 33]), ([7], [1]), ([10], [14])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write(gpu_device, h, d, page, lens, new, dtype):
    print(f"[kv] write {h}x{d} page {page} {lens} {new} {dtype}", flush=True)
    table, (kc, vc) = _layer(gpu_device, lens, h, d, page, dtype)
    n = new or [1] * len(lens)
    k, v = (torch.randn((sum(n), h, d), device=gpu_device).to(dtype) for _ in range(2))
    want = [c.view(torch.int16).cpu().numpy() for c in (kc, vc)]
    _expect(table, lens, n, page, [x.view(torch.int16).cpu().numpy() for x in (k, v)], want)
    cu = None if new is None else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=gpu_device)
    ck.kv_write(k, v, kc, vc, table.to(gpu_device), torch.tensor(lens, dtype=torch.int32, device=gpu_device), cu)
    for c, w in zip((kc, vc), want):
        assert np.array_equal(c.view(torch.int16).cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("h,d", [(1, 64), (8, 128), (3, 80), (2, 16), (5, 256), (2, 48)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_int8(gpu_device, h, d, dtype):
    print(f"[kv] write int8 {h}x{d} {dtype}", flush=True)
    lens, new = [30, 0, 5, 64], [30, 0, 3, 33]
    table, (kc, vc) = _layer(gpu_device, lens, h, d, 16, torch.int8)
    ks, vs = (torch.full(kc.shape[:3], 9.0, device=gpu_device) for _ in range(2))
    k, v = (torch.randn((sum(new), h, d), device=gpu_device) for _ in range(2))
    k[3] *= 1e-4
    k[4] = 0
    v[5, 0, 0] = 300.0
    k, v = k.to(dtype), v.to(dtype)
    codes, scales = [], []
    for x in (k, v):
        f = x.float().cpu().numpy()
        s = np.maximum(np.abs(f).max(-1) / np.float32(127), np.float32(1e-10)).astype(np.float32)
        codes.append(np.rint(f / s[..., None]).astype(np.int8))
        scales.append(s)
    want = [c.cpu().numpy() for c in (kc, vc, ks, vs)]
    _expect(table, lens, new, 16, codes + scales, want)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=gpu_device)
    ck.kv_write(k, v, kc, vc, table.to(gpu_device), torch.tensor(lens, dtype=torch.int32, device=gpu_device), cu, ks, vs)
    for c, w in zip((kc, vc, ks, vs), want):
        assert np.array_equal(c.cpu().numpy(), w)


@pytest.mark.gpu
def test_write_int8_rows_that_are_not_finite_read_back_as_nan(gpu_device):
    table, (kc, vc) = _layer(gpu_device, [3], 2, 64, 16, torch.int8)
    ks, vs = (torch.zeros(kc.shape[:3], device=gpu_device) for _ in range(2))
    k = torch.randn((3, 2, 64), device=gpu_device).to(torch.bfloat16)
    k[0, 0, 5], k[1, 1, 6], k[2, 0, 7] = math.inf, math.nan, -math.inf
    ck.kv_write(k, k, kc, vc, table.to(gpu_device), torch.tensor([3], dtype=torch.int32, device=gpu_device),
                torch.tensor([0, 3], dtype=torch.int32, device=gpu_device), ks, vs)
    p = int(table[0, 0])
    assert torch.isnan(ks[p, :, :3]).cpu().tolist() == [[True, False, True], [False, True, False]]
    assert (kc[p, 0, 0] == 0).all() and (kc[p, 1, 1] == 0).all()


@pytest.mark.gpu
def test_write_strides_and_places_that_are_not_there(gpu_device):
    """k and v as slices of a fused projection, a cache in token-major order, table entries that are no page."""
    lens = [20, 33, 8]
    table, _ = _layer(gpu_device, lens, 2, 64, 16, torch.bfloat16)
    table[1, 2] = -1
    table[2, 0] = 1 << 29
    pages = 16
    kc, vc = (torch.zeros((pages, 16, 2, 64), dtype=torch.bfloat16, device=gpu_device).transpose(1, 2) for _ in range(2))
    fused = torch.randn((3, 8, 64), device=gpu_device).to(torch.bfloat16)
    k, v = fused[:, 4:6], fused[:, 6:8]
    want = [np.zeros((pages, 2, 16, 64), dtype=np.float32) for _ in range(2)]
    _expect(table, lens, [1] * 3, 16, [x.float().cpu().numpy() for x in (k, v)], want)
    ck.kv_write(k, v, kc, vc, table.to(gpu_device), torch.tensor(lens, dtype=torch.int32, device=gpu_device))
    for c, w in zip((kc, vc), want):
        assert np.array_equal(c.float().cpu().numpy(), w)
    assert (kc != 0).any(-1).sum() == 2


def _cache(dev, int8=False, layers=3, pages=60, seqs=12, page=8, h=2, d=16, max_tokens=64, seed=1):
    c = ck.PagedKVCache(layers, pages, h, d, page, seqs, max_tokens, int8=int8, device=dev)
    g = torch.Generator().manual_seed(seed)
    for x in (c.k, c.v, c.k_scale, c.v_scale):
        if x is not None:
            x.copy_((torch.randn(x.shape, generator=g) * 50).to(x.dtype))
    return c


def _same(c, want, ks):
    assert c.page_table.cpu().tolist() == want.table
    assert c.lens.cpu().tolist() == want.lens and c.refs.cpu().tolist() == want.refs
    for x, k in zip((c.k, c.v, c.k_scale, c.v_scale), ks):
        if x is not None:
            assert torch.equal(x.cpu(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_sequence_of_calls(gpu_device, seed, int8):
    """Growing, forking, freeing and compacting in random order, calls that cannot be done among them: tables,
    lengths, counts, contents and the status as the plain loops give them after every call."""
    rng = random.Random(seed)
    layers = 1 + seed % 3
    c = _cache(gpu_device, int8=int8, layers=layers, page=[1, 4, 8][seed % 3], pages=60, h=1 + seed % 2)
    want = serving.Pages(c.page_table.cpu().tolist(), c.lens.cpu().tolist(), c.refs.cpu().tolist(), c.page_size)
    ks = [None if x is None else x.cpu().clone() for x in (c.k, c.v, c.k_scale, c.v_scale)]
    for step in range(40):
        rows = rng.sample(range(12), rng.randrange(1, 6))
        what = rng.choice(["grow", "grow", "fork", "fork", "free", "compact"])
        print(f"[kv] seed {seed} step {step} {what} {rows}", flush=True)
        want.moves, status = [], 0
        if what == "grow":
            counts = [rng.choice([0, 1, 3, 9, 20]) for _ in rows]
            if rng.random() < 0.1:
                rows = rows + [rng.choice([-1, 12, rows[0]])]
                counts.append(1)
            c.grow(rows, counts)
            status = want.grow(rows, counts)
        elif what == "fork":
            dst = [r for r in range(12) if want.lens[r] == 0][: len(rows)]
            src = [rng.choice([r for r in range(12) if r not in dst] or [0]) for _ in dst]
            if rng.random() < 0.15 and dst:
                src[0] = rng.choice([99, -5, dst[0]])
            c.fork(src, dst)
            status = want.fork(src, dst) if dst else 0
            if not dst:
                continue
        elif what == "free":
            c.free(rows + [rows[0], 99])
            want.free(rows)
        else:
            n = c.compact()
            assert int(n) == want.compact()
        if what in ("grow", "fork"):
            assert int(c.status) == status, what
            if status:
                with pytest.raises((ValueError, ck.MQError)):
                    c.check()
            else:
                c.check()
        for s, d in want.moves:
            for k in ks:
                if k is not None:
                    k[:, d] = k[:, s]
        _same(c, want, ks)


@pytest.mark.gpu
@pytest.mark.parametrize("pages,seqs", [(3000, 700), (20000, 1500)])
def test_many_pages_and_sequences(gpu_device, pages, seqs):
    """More pages than a workgroup looks at in one step, more sequences than it has threads."""
    c = ck.PagedKVCache(1, pages, 1, 8, 4, seqs, 64, device=gpu_device)
    c.k.copy_(torch.randn(c.k.shape))
    c.v.copy_(torch.randn(c.v.shape))
    ks = [c.k.cpu().clone(), c.v.cpu().clone(), None, None]
    want = serving.Pages(c.page_table.cpu().tolist(), c.lens.cpu().tolist(), c.refs.cpu().tolist(), 4)
    rng = random.Random(1)
    half = list(range(seqs // 2))
    counts = [rng.randrange(0, 13) for _ in half]
    c.grow(half, counts)
    assert want.grow(half, counts) == 0
    other = list(range(seqs // 2, seqs // 2 * 2))
    src = [rng.choice(half) for _ in other]
    c.fork(src, other)
    assert want.fork(src, other) == 0 and int(c.status) == 0
    for s, d in want.moves:
        for k in ks[:2]:
            k[:, d] = k[:, s]
    _same(c, want, ks)
    gone = rng.sample(range(seqs), seqs // 2)
    c.free(gone)
    want.free(gone)
    assert int(c.compact()) == want.compact()
    for s, d in want.moves:
        for k in ks[:2]:
            k[:, d] = k[:, s]
    _same(c, want, ks)
    c.grow(half, [50] * len(half))                      # more than 3000 pages have room for
    missing = want.grow(half, [50] * len(half))
    assert (missing > 0) == (pages == 3000) and int(c.status) == missing
    _same(c, want, ks)


@pytest.mark.gpu
def test_pages_past_4_gib(gpu_device):
    """Copies whose offsets pass 32 bits (in bytes and in 16-byte units)."""
    layers, pages, h, page, d = 2, 70, 8, 1024, 1024 // 4
    k = torch.empty((layers, pages, 8, page * 16, d), dtype=torch.bfloat16, device=gpu_device)
    v = k   # the same memory twice: both copies move the same bytes
    assert k.stride(1) * 2 * pages * layers > 1 << 33
    table = torch.full((2, 4), -1, dtype=torch.int32, device=gpu_device)
    lens, refs = (torch.zeros(n, dtype=torch.int32, device=gpu_device) for n in (2, pages))
    refs[:3] = 1
    refs[pages - 1] = 1
    table[0, 0], lens[0] = pages - 1, 100
    k[:, pages - 1] = 5
    k[:, 3] = 0
    ck.kv_fork(k, v, table, lens, refs, [0], [1])
    assert table[1].cpu().tolist() == [3, -1, -1, -1] and (k[:, 3] == 5).all()
    k[1, pages - 1, 0, 0, 0] = 6
    refs[:3] = 0
    ck.kv_compact(k, v, table, refs)
    assert table.cpu().tolist() == [[1, -1, -1, -1], [0, -1, -1, -1]] or table.cpu().tolist() == [[0, -1, -1, -1], [1, -1, -1, -1]]
    assert float(k[1, int(table[0, 0]), 0, 0, 0]) == 6
    del k, v
