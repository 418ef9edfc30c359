"""More rows and tokens than one launch takes (2^32 threads): the same as in smaller calls."""
import pytest
import torch

import kitchen_amd as ck


@pytest.mark.gpu
def test_norms_of_many_short_rows(gpu_device):
    """2^26 rows and some, as of heads' values: 4 rows a workgroup of 256."""
    m, k = (1 << 26) + 5, 8
    x = torch.randn((1 << 20, k), device=gpu_device).to(torch.bfloat16).repeat(65, 1)[:m]
    w = torch.rand(k, device=gpu_device)
    y, (z, h), (q, s) = ck.rms_norm(x, w), ck.rms_norm(x, w, x), ck.rms_norm_quantize(x, w)
    for at in (slice(0, 1000), slice((1 << 24) - 500, (1 << 24) + 500), slice((1 << 25) - 500, (1 << 25) + 500), slice(m - 1000, m)):
        part = x[at].contiguous()
        assert torch.equal(y[at], ck.rms_norm(part, w))
        assert torch.equal(h[at], part + part) and torch.equal(z[at], ck.rms_norm(part, w, part)[0])
        c, t = ck.rms_norm_quantize(part, w)
        assert torch.equal(q[at], c) and torch.equal(s[at], t)
    n = 1 << 20
    assert all(torch.equal(y[i * n:(i + 1) * n], y[:n]) and torch.equal(q[i * n:(i + 1) * n], q[:n]) for i in range(1, m // n))


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [True, False])
def test_appends_of_many_tokens(gpu_device, ragged):
    """2^24 tokens and some: of one sequence, or one each of as many."""
    t, d, page = (1 << 24) + 3, 8, 1024 if ragged else 1
    g = torch.Generator(device=gpu_device).manual_seed(0)
    q, k, v = (torch.randn((t, 1, d), generator=g, device=gpu_device).to(torch.bfloat16) for _ in range(3))
    rotary = ck.Rotary(d)
    pages = -(-t // page)
    kc, vc = (torch.zeros((pages, 1, page, d), dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    place = torch.arange(pages, dtype=torch.int32, device=gpu_device)
    if ragged:                                          # token i at position i
        table, lens = place[None], torch.tensor([t], dtype=torch.int32, device=gpu_device)
        cu = torch.tensor([0, t], dtype=torch.int32, device=gpu_device)
    else:                                               # all at position 0
        table, lens, cu = place[:, None], torch.ones(t, dtype=torch.int32, device=gpu_device), None
    y = ck.kv_append(q, k, v, kc, vc, table, lens, rotary, cu)
    assert torch.equal(vc.view(-1, 1, d)[:t], v)
    if not ragged:
        assert torch.equal(y, q) and torch.equal(kc.view(-1, 1, d)[:t], k)
        return
    for lo in (0, (1 << 23) - 50, (1 << 23), t - 100):
        n = slice(lo, lo + 100)                         # the same tokens as the last ones of a shorter sequence
        end, few = torch.tensor([lo + 100], dtype=torch.int32, device=gpu_device), torch.tensor([0, 100], dtype=torch.int32, device=gpu_device)
        kd, vd = torch.zeros_like(kc), torch.zeros_like(vc)
        assert torch.equal(y[n], ck.kv_append(q[n], k[n], v[n], kd, vd, table, end, rotary, few))
        assert torch.equal(kc.view(-1, d)[n], kd.view(-1, d)[n])


@pytest.mark.gpu
def test_tokens_of_many_rows(gpu_device):
    """2^22 rows and some, 1024 threads each, with settings of their own."""
    rows, vocab, n = (1 << 22) + 3, 5, 1 << 14
    g = torch.Generator(device=gpu_device).manual_seed(0)
    x = torch.randn((n, vocab), generator=g, device=gpu_device).repeat(rows // n + 1, 1)[:rows].contiguous()
    u = torch.rand(n, generator=g, device=gpu_device).repeat(rows // n + 1)[:rows].contiguous()
    t = torch.rand(n, generator=g, device=gpu_device).repeat(rows // n + 1)[:rows].contiguous()
    k = torch.randint(0, 5, (n,), generator=g, device=gpu_device, dtype=torch.int32).repeat(rows // n + 1)[:rows].contiguous()
    y = ck.sample(x, u, t, k, t, t / 4)
    first = ck.sample(x[:n], u[:n], t[:n], k[:n], t[:n], t[:n] / 4)
    assert torch.equal(y, first.repeat(rows // n + 1)[:rows])
    assert torch.equal(ck.sample(x, u, 0.0), x.argmax(-1))
