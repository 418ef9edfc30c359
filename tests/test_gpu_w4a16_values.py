"""w4a16_linear's numbers: what fp32 sums of shifted codes lose."""
import pytest
import torch

import kitchen_amd as ck
from test_gpu_w4a16_tiles import exact, weights


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", ["none", "u4"])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (5, 512, 4096), (2, 4600, 4096)])
def test_fp32_rows_lose_little(gpu_device, m, n, k, zeros):
    """fp32 rows and outputs. Codes are held as 16 + c and (16 + z) sum(x) is taken off behind a group's products. For
    normal x a group's sum of (16 + c) x reaches 24 sqrt(64) = 192 (16 + c is 24 on average) where the difference is about
    4.6 sqrt(2) sqrt(64) = 52 (37 without zero-points). The exact products of 32 values are added to the sum at a time, so
    it is rounded twice in a group, at 2^-16 apart and then: errors of 2^-16 / sqrt(12) each, the sum of x times 24 as much
    once more: sqrt(3) 4.4e-6 against 37 is 2.1e-7 of the output, and half as much again is allowed for what comes behind:
    3e-7. (Codes held as 128 + c: 1150 in place of 192, rounded 8 times as coarsely.)"""
    print(f"[w4a16] precision {m}x{n}x{k} {zeros}", flush=True)
    qw, ws, wz = weights(n, k, 64, zeros, gpu_device)
    x = torch.randn((m, k), generator=torch.Generator(device=gpu_device).manual_seed(3), device=gpu_device)
    y = ck.w4a16_linear(x, qw, ws, wz)
    want = exact(x, qw, ws, wz, 64, 0)[0]
    lost = float((y.double() - want).norm() / want.norm())
    print(f"[w4a16] lost {lost:.2e}", flush=True)
    assert lost < 3e-7
