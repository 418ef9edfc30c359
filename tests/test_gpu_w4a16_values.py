"""w4a16_linear's numbers: what fp32 sums of shifted codes lose, and values that are not finite."""
import math

import pytest
import torch

import kitchen_amd as ck
from test_gpu_w4a16_tiles import check, exact, weights


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


def _plain(x, qw, ws, wz, group=64):
    """The formula as it stands, infinities and all: every weight times every x, summed in fp32."""
    n, k = qw.shape[0], 2 * qw.shape[1]
    code = torch.stack([qw & 15, qw >> 4], -1).view(n, k // group, group).float()
    s = ws.float()[..., None]
    if wz is None:
        w = (code - 16 * (code > 7)) * s
    elif wz.dtype == torch.uint8:
        w = (code - torch.stack([wz & 15, wz >> 4], -1).view(n, -1)[:, : k // group, None].float()) * s
    else:
        w = code * s + wz.float()[..., None]
    return (x.float()[:, None, :] * w.view(1, n, k)).sum(-1)


def _same_kind(y, want, finite_too=True):
    y, want = y.float(), want.float()
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isposinf(), want.isposinf()) and torch.equal(y.isneginf(), want.isneginf())
    if finite_too:
        at = want.isfinite()
        assert ((y - want).abs()[at] <= 2.0 ** -7 * want.abs()[at] + 1e-3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", ["none", "u4", "float"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 300, 448), (3, 64, 8192), (2, 17000, 256), (6, 4500, 1024), (9, 40, 16384)])
def test_infinities_keep_their_sign(gpu_device, m, n, k, dtype, zeros):
    """x with an infinity: the output is one where that weight is not 0 (of the weight's sign), NaN where it is; two of
    one column with other signs, or a NaN, make NaN; other rows do not change."""
    print(f"[w4a16] infinities {m}x{n}x{k} {dtype} {zeros}", flush=True)
    qw, ws, wz = weights(n, k, 64, zeros, gpu_device, seed=2)
    x = torch.randn((m, k), generator=torch.Generator(device=gpu_device).manual_seed(5), device=gpu_device).to(dtype)
    want = ck.w4a16_linear(x, qw, ws, wz)
    for places in ({5: math.inf}, {k - 1: -math.inf}, {70: math.inf, k - 9: math.inf}, {3: math.nan}):
        z = x.clone()
        for at, v in places.items():
            z[m // 2, at] = v
        y = ck.w4a16_linear(z, qw, ws, wz)
        _same_kind(y, _plain(z, qw, ws, wz))
        others = torch.arange(m, device=gpu_device) != m // 2
        assert torch.equal(y[others], want[others])


@pytest.mark.gpu
@pytest.mark.parametrize("k", [320, 512])
def test_scales_that_are_not_finite(gpu_device, k):
    """An infinite or NaN scale or zero-point stays in its column and gives what the formula gives."""
    for dtype in (torch.bfloat16, torch.float16):
        qw, ws, wz = weights(40, k, 64, "float", gpu_device)
        x = torch.randn((3, k), device=gpu_device).abs().to(dtype)
        want = ck.w4a16_linear(x, qw, ws, wz)
        ws, wz = ws.clone(), wz.clone()
        ws[3, -1], ws[9, 0], wz[20, -1] = math.inf, math.nan, -math.inf
        qw[3, -32:] |= 0x11                          # no code of 0 there: infinity times 0 is NaN
        y = ck.w4a16_linear(x, qw, ws, wz)
        keep = torch.ones(40, dtype=torch.bool, device=gpu_device)
        keep[[3, 9, 20]] = False
        assert torch.equal(y[:, keep], want[:, keep])
        _same_kind(y[:, ~keep], _plain(x, qw, ws, wz)[:, ~keep], finite_too=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_finite_values(gpu_device, dtype):
    """Products that fit fp32 though 16 + c times x would not."""
    qw, ws, _ = weights(48, 256, 64, "none", gpu_device)
    x = torch.zeros((2, 256), dtype=dtype, device=gpu_device)
    x[0, 7], x[1] = 2.0 ** 126, 1.0
    y = ck.w4a16_linear(x, qw, ws)
    _same_kind(y, _plain(x, qw, ws, None))


@pytest.mark.gpu
def test_more_rows_than_a_grid_has(gpu_device):
    """75000 groups of rows: more than 65535, which some launches are limited to."""
    qw, ws, wz = weights(16, 64, 64, "u4", gpu_device)
    x = torch.randn((600000, 64), device=gpu_device).to(torch.bfloat16)
    check(ck.w4a16_linear(x, qw, ws, wz, None, 64, 64), x, qw, ws, wz, 64, 64)


@pytest.mark.gpu
def test_weights_at_any_place(gpu_device):
    """Packed weights that begin between 16-byte boundaries, and one row of them for every column."""
    qw, ws, wz = weights(50, 512, 64, "u4", gpu_device)
    x = torch.randn((2, 512), device=gpu_device).to(torch.bfloat16)
    want = ck.w4a16_linear(x, qw, ws, wz)
    for shift in (1, 8):
        flat = torch.zeros(50 * 256 + shift, dtype=torch.uint8, device=gpu_device)
        flat[shift:] = qw.reshape(-1)
        assert torch.equal(ck.w4a16_linear(x, flat[shift:].view(50, 256), ws, wz), want)
    one = qw[:1].expand(50, 256)
    assert torch.equal(ck.w4a16_linear(x, one, ws, wz), ck.w4a16_linear(x, one.contiguous(), ws, wz))
