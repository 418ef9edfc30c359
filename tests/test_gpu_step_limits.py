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
