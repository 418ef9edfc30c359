"""Which bits the probabilities over shared keys keep, at scores that are set one by one: the key of value 1 in the head's first
place has the score itself, in base 2. Against sums of fp64; the single-token kernel has to keep to the same bounds.

A probability is rounded to 16 bits against the row's running maximum, so the largest is exact, and the others are off by u of
themselves (fp16 ones as far as 2^-28 of the largest: they are held 2^14 times as large); the output is rounded once (u |o|). The
few sums that matter are fp32, exp2 and the scale's product too: 2^-18 of all weights."""
import math

import pytest
import torch

import kitchen_amd as ck

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHARED, PAGE = 128, 16


def check(dev, d, dtype, scores, values, exact):
    """scores, values(h) of the shared keys; exact: the key whose probability is not rounded."""
    seqs, hq, h = 3, 8, 2
    n = SHARED // PAGE
    table = torch.tensor([[*range(n), n + b] for b in range(seqs)], dtype=torch.int32, device=dev)
    lens = torch.full((seqs,), SHARED + 1, dtype=torch.int32, device=dev)
    k = torch.zeros((n + seqs, h, PAGE, d), dtype=dtype)
    v = torch.zeros_like(k)
    k[..., 0] = -60.0                                   # a sequence's own key: no weight
    k[:n, :, :, 0] = scores.view(n, 1, PAGE).to(dtype)
    v[:n] = values.view(n, PAGE, h, d).transpose(1, 2).to(dtype)
    q = torch.zeros((seqs, hq, d), dtype=dtype)
    q[..., 0] = 1.0
    p = torch.exp2(scores.to(dtype).double() - scores.max())
    x = values.to(dtype).double()
    o = (p[:, None, None] * x).sum(0) / p.sum()
    w = (p[:, None, None] * x.abs()).sum(0) / p.sum()
    rounded = w - p[exact] * x[exact].abs() / p.sum()
    tol = U[dtype] * (o.abs() * (1 + 2.0 ** -9) + rounded) + 2.0 ** -18 * w
    args = (q.to(dev), k.to(dev), v.to(dev), table, lens)
    plan = ck.kv_shared(table, lens, PAGE, least=0)
    assert plan[0] == 1
    for y in (ck.paged_attention(*args, scale=math.log(2)), ck.paged_attention(*args, scale=math.log(2), shared=plan)):
        err = (y.double().cpu().view(seqs, h, hq // h, d) - o[None, :, None]).abs()
        assert (err <= tol[None, :, None]).all(), f"{float((err / tol[None, :, None]).max()):.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("top", [5.125, 6.09375, 7.03125, 7.34375, 20.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_largest_is_exact(gpu_device, d, dtype, top):
    """Wherever it comes: behind a smaller one in the same wave's keys."""
    g = torch.Generator().manual_seed(int(top * 32))
    scores = torch.full((SHARED,), -60.0, dtype=torch.float64)
    scores[5], scores[69] = 0.0, top
    check(gpu_device, d, dtype, scores, torch.randn((SHARED, 2, d), generator=g), 69)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [-20.984375, -22.71875, -22.984375, -26.875])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_weights_of_large_values(gpu_device, d, low):
    """fp16: weights of 2^-21 to 2^-27 of the largest, whose own value is 0, keep their 11 bits."""
    g = torch.Generator().manual_seed(1)
    scores = torch.full((SHARED,), low, dtype=torch.float64)
    scores[5] = 0.0
    values = 30000 * (1 + torch.rand((SHARED, 2, d), generator=g))
    values[5] = 0
    check(gpu_device, d, torch.float16, scores, values, 5)
