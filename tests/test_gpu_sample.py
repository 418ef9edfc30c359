"""kitchen_amd.sample against plain numpy in 64 bits, row by row: tokens have to be equal. (A weight is off by 1e-9 of itself at
most, and sums are of integers: a token could only differ where u, top_p or min_p lies that close to a border of the sums.)"""
import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import step

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits(rows, vocab, dtype, seed=0, spread=2.5):
    return (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def check(dev, x, u, **kw):
    if not isinstance(u, torch.Tensor):
        u = torch.tensor(u, dtype=torch.float32)
    got = ck.sample(x.to(dev), u.to(dev), **{n: v.to(dev) if isinstance(v, torch.Tensor) else v for n, v in kw.items()})
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    rows = x.float().numpy()

    def of(name, r):
        v = kw.get(name, {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}[name])
        v = v[r].item() if isinstance(v, torch.Tensor) else v
        return v if name == "top_k" else float(np.float32(v))

    want = [step.sample(rows[r], float(u[r]), *(of(n, r) for n in ("temperature", "top_k", "top_p", "min_p")))
            for r in range(len(rows))]
    assert got.cpu().tolist() == want


def uniform(rows, seed=9):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 1023, 1024, 1025, 4096, 10007, 50000])
@pytest.mark.parametrize("dtype", TYPES)
def test_all_of_the_row(gpu_device, vocab, dtype):
    print(f"[sample] {vocab} {dtype}", flush=True)
    check(gpu_device, logits(17, vocab, dtype, vocab), uniform(17))


SETTINGS = [dict(temperature=0.0), dict(top_k=1), dict(top_k=2, temperature=3.0), dict(top_k=50, temperature=0.7),
            dict(top_k=3000, temperature=1.5), dict(top_p=0.0), dict(top_p=0.1), dict(top_p=0.9), dict(top_p=0.999, temperature=2.0),
            dict(min_p=0.05), dict(min_p=1.0), dict(min_p=2.0), dict(top_k=200, top_p=0.8), dict(top_k=40, top_p=0.95, min_p=0.1, temperature=0.8),
            dict(top_k=5000, top_p=0.99, temperature=5.0), dict(temperature=1e-3, top_p=0.5), dict(temperature=100.0, top_p=0.7),
            dict(top_k=1 << 20, top_p=1.5, min_p=-1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab,dtype", [(5003, torch.float32), (5003, torch.bfloat16), (33000, torch.float16), (131072, torch.float32)])
def test_settings(gpu_device, kw, vocab, dtype):
    print(f"[sample] {vocab} {dtype} {kw}", flush=True)
    check(gpu_device, logits(12, vocab, dtype, 3), uniform(12), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 5, 64, 300])
def test_settings_of_every_row(gpu_device, rows):
    g = torch.Generator().manual_seed(rows)
    r = torch.rand((4, rows), generator=g)
    check(gpu_device, logits(rows, 3001, torch.bfloat16, rows), uniform(rows),
          temperature=torch.where(r[0] < 0.2, 0.0, 2 * r[0]), top_k=(r[1] * 100).int() - 10,
          top_p=torch.where(r[2] < 0.2, 1.0, r[2]), min_p=r[3] / 5)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=1500, top_p=0.5), dict(top_k=100, min_p=0.5),
                                dict(temperature=0.0), dict(top_p=0.3, top_k=5)], ids=str)
@pytest.mark.parametrize("vocab", [1, 9, 3000, 40000])
def test_ties(gpu_device, kw, vocab):
    """All alike; a few values only; both zeros: ties go to the lowest index."""
    print(f"[sample] ties {vocab} {kw}", flush=True)
    g = torch.Generator().manual_seed(4)
    x = torch.stack([torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=g).float(),
                     torch.where(torch.rand(vocab, generator=g) < 0.5, -0.0, 0.0), torch.arange(vocab) % 2 * 1.0])
    check(gpu_device, x, [0.37, 0.62, 0.11, 0.93], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.0)], ids=str)
def test_rows_that_hold_no_numbers(gpu_device, kw):
    """Masks of -infinity and of the type's lowest value, NaN, +infinity, and rows where nothing is left."""
    low = torch.finfo(torch.float32).min
    x = logits(8, 700, torch.float32, 5)
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 1:] = -float("inf")
    x[3, :650] = -float("inf")
    x[4, 5:] = low
    x[5, ::3] = float("nan")
    x[6, 100], x[6, 300] = float("inf"), float("inf")
    x[7] = low
    check(gpu_device, x, [0.5, 0.5, 0.99, 0.7, 0.2, 0.4, 0.8, 0.6], **kw)


@pytest.mark.gpu
def test_random_numbers_at_the_ends(gpu_device):
    """0, just below 1, 1 and beyond, negative, NaN."""
    x = logits(8, 2000, torch.bfloat16, 6)
    u = [0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan"), 1e-38, 0.5]
    for kw in (dict(), dict(top_k=10), dict(top_p=0.4)):
        check(gpu_device, x, u, **kw)


@pytest.mark.gpu
def test_every_token_comes_as_often_as_it_should(gpu_device):
    """u over an even grid of n: a token of probability p comes n p times, give or take one."""
    n, x = 4096, logits(1, 50, torch.float32, 8)
    u = (torch.arange(n) + 0.5) / n
    token = ck.sample(x.expand(n, 50).to(gpu_device), u.to(gpu_device), temperature=1.3)
    p = torch.softmax(x[0].double() / float(np.float32(1.3)), 0)
    assert (torch.bincount(token.cpu(), minlength=50) - n * p).abs().max() <= 1


@pytest.mark.gpu
def test_strides_streams_and_graphs(gpu_device):
    x = logits(6, 9000, torch.float16, 7).to(gpu_device)
    u = uniform(6).to(gpu_device)
    part, odd = x[::2, 1:5002], x[:, ::3]
    check(gpu_device, part.cpu(), u[:3].cpu(), top_p=0.9)
    assert torch.equal(ck.sample(part, u[:3], top_p=0.9), ck.sample(part.contiguous(), u[:3], top_p=0.9))
    assert torch.equal(ck.sample(odd, u), ck.sample(odd.contiguous(), u))
    assert ck.sample(x[:0], u[:0]).shape == (0,)
    want = ck.sample(x, u, top_k=30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ck.sample(x, u, top_k=30)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    p = torch.full((6,), 0.8, device=gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ck.sample(x, u, top_k=30)
        b = ck.sample(x, u, temperature=0.7, top_p=p)
        c = ck.sample(x, u)
    for i in range(3):
        x.copy_(logits(6, 9000, torch.float16, 20 + i))
        u.copy_(uniform(6, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ck.sample(x, u, top_k=30)) and torch.equal(b, ck.sample(x, u, temperature=0.7, top_p=p))
        assert torch.equal(c, ck.sample(x, u))


ODD = [dict(), dict(top_k=9), dict(top_k=4500), dict(top_p=0.6), dict(top_k=6000, top_p=0.95, min_p=0.01), dict(min_p=0.3), dict(top_p=0.02)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", ODD, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_long_rows_of_large_batches(gpu_device, kw, dtype):
    """More rows than are cut into parts, of several blocks."""
    check(gpu_device, logits(140, 40003, dtype, 11), uniform(140), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", ODD + [dict(top_k=100000), dict(top_k=131071, top_p=0.5)], ids=str)
@pytest.mark.parametrize("vocab", [131072, 262144, 300007])
def test_thousands_alike(gpu_device, kw, vocab):
    """All alike, two values, a few hundred, and values that crowd in one bin: more to choose from than is held at once."""
    print(f"[sample] alike {vocab} {kw}", flush=True)
    g = torch.Generator().manual_seed(14)
    x = torch.stack([torch.full((vocab,), -3.5), torch.randint(0, 2, (vocab,), generator=g) * 20.0,
                     torch.randint(0, 300, (vocab,), generator=g) * 1e-6, torch.rand(vocab, generator=g) * 1e-3 - 50])
    x[3, 77] = 1.0
    check(gpu_device, x, [0.37, 0.62, 0.11, 0.93], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1e-28, 1e-10, 1e-4, 30.0, 1e4, 1e10, 1e30, float("inf")])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(top_p=0.7), dict(top_p=0.7, top_k=5000), dict(min_p=0.1)], ids=str)
def test_temperatures(gpu_device, t, kw):
    print(f"[sample] T {t} {kw}", flush=True)
    check(gpu_device, logits(6, 20011, torch.float32, 15), uniform(6), temperature=t, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e4, 6e4, 1e30, 3e38])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.7), dict(temperature=1e3, top_k=50, top_p=0.9)], ids=str)
def test_sizes_of_logits(gpu_device, dtype, size, kw):
    """Up to the type's largest, down to what is not normal."""
    big = torch.finfo(dtype).max
    x = (torch.rand((5, 9001), generator=torch.Generator().manual_seed(16)).double() * 2 - 1) * size
    x[1] = x[1].abs()
    x[2] = -x[2].abs()
    check(gpu_device, x.clamp(-big, big).to(dtype), uniform(5), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 70001])
def test_every_kind_of_nan(gpu_device, vocab):
    """Quiet and signalling, of either sign: never chosen, in rows of one part and of several."""
    bits = {torch.bfloat16: ([0x7f81, 0x7fc0, -1, -0x7f], torch.int16), torch.float16: ([0x7c01, 0x7e00, -1, -0x3ff], torch.int16),
            torch.float32: ([0x7f800001, 0x7fc00000, -1, -0x7fffff], torch.int32)}
    for dtype, (patterns, like) in bits.items():
        x = logits(4, vocab, dtype, 17)
        for i, b in enumerate(patterns):
            nan = torch.tensor([b], dtype=like).view(dtype)
            assert nan.isnan().all()
            x[i, i::2] = nan
            if i == 3:
                x[i] = nan
        for kw in (dict(), dict(top_k=5), dict(top_p=0.5), dict(temperature=0.0)):
            check(gpu_device, x, uniform(4), **kw)


@pytest.mark.gpu
def test_two_at_once(gpu_device):
    """Calls of two streams and of two threads at the same time do not share working space."""
    import threading
    x = [logits(20, 100003, torch.bfloat16, 18 + i).to(gpu_device) for i in range(2)]
    u = uniform(20).to(gpu_device)
    want = [ck.sample(y, u, top_p=0.9, top_k=800) for y in x]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got[i].append(ck.sample(x[i], u, top_p=0.9, top_k=800))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys) and len(got[0]) == len(got[1]) == 30


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [(1 << 24) - 3, 1 << 24])
def test_the_longest_rows(gpu_device, vocab):
    x = logits(1, vocab, torch.bfloat16, 21)
    check(gpu_device, x, [0.613])
    check(gpu_device, x, [0.272], top_p=0.9, temperature=0.8)
    check(gpu_device, x, [0.272], top_k=64)
