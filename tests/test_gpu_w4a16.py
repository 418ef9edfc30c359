"""Linears with 4-bit weights and floating-point activations (kitchen_amd.w4a16_linear) against 64 bits.

Tolerance for outputs of unit roundoff u: one rounding of the output (u |y|), and fp32 sums of K products in any
order, of the codes shifted by up to 144 and of the zero-points' part apart: a relative error of at most
(K / 64 + 40) 2^-24 of the sum of the parts' magnitudes (a group of 64 is summed first, then the groups; the
spread of the oracle holds |w| + 24 s per weight, a sixth of the shifted codes' 144, hence the factor 6)."""
import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import serving

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _weights(n, k, group, zeros, dev, seed=0, sdt=torch.float16):
    g = torch.Generator().manual_seed(seed)
    qw = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    ws = (torch.rand((n, k // group), generator=g) * 0.02 + 0.001).to(sdt)
    wz = None
    if zeros == "u4":
        wz = torch.randint(0, 256, (n, (k // group + 1) // 2), generator=g, dtype=torch.uint8)
    elif zeros == "float":
        wz = (-torch.rand((n, k // group), generator=g) * 0.1).to(sdt)
    return qw.to(dev), ws.to(dev), None if wz is None else wz.to(dev)


def _check(x, qw, ws, wz, bias, y, group, block):
    z = None if wz is None else wz.cpu().numpy() if wz.dtype == torch.uint8 else wz.double().cpu().numpy()
    want, spread = serving.w4a16_linear(x.double().cpu().numpy(), qw.cpu().numpy(), ws.double().cpu().numpy(), z,
                                        None if bias is None else bias.double().cpu().numpy(), group, block)
    k = x.shape[-1]
    tol = U[y.dtype] * np.abs(want) + 6 * (k / 64 + 40) * 2.0 ** -24 * spread + 1e-30
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= tol).all(), f"worst {(err / tol).max():.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", ["none", "u4", "float"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,group,block", [(1, 256, 512, 64, 0), (1, 1000, 3072, 64, 256), (2, 33, 320, 64, 64),
                                               (3, 16, 64, 64, 0), (5, 130, 1056, 32, 16), (16, 257, 1024, 128, 256),
                                               (17, 64, 448, 64, 64), (33, 48, 256, 128, 0), (1, 1, 32, 32, 16),
                                               (70, 20, 192, 64, 0), (4, 4096, 4096, 64, 0)])
def test_against_64_bits(gpu_device, m, n, k, group, block, dtype, zeros):
    print(f"[w4a16] {m}x{n}x{k} group {group} block {block} {dtype} {zeros}", flush=True)
    qw, ws, wz = _weights(n, k, group, zeros, gpu_device)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(m)).to(dtype).to(gpu_device)
    x[:, : k // 50] *= 20
    bias = torch.randn(n, device=gpu_device).to(dtype) if m % 2 else None
    y = ck.w4a16_linear(x, qw, ws, wz, bias, group, block or None)
    assert y.dtype == dtype
    _check(x, qw, ws, wz, bias, y, group, block)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [32768, 16384, 12288])
@pytest.mark.parametrize("m", [1, 16, 40])
def test_long_rows(gpu_device, k, m):
    print(f"[w4a16] {m}x64x{k}", flush=True)
    qw, ws, wz = _weights(64, k, 64, "u4", gpu_device)
    x = torch.randn((m, k), device=gpu_device).to(torch.bfloat16)
    _check(x, qw, ws, wz, None, ck.w4a16_linear(x, qw, ws, wz, convrot_groupsize=256), 64, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group,dtype", [(16, 4500, 16384, 64, torch.bfloat16), (16, 4500, 8192, 32, torch.float16),
                                               (4, 10000, 32768, 32, torch.float32), (9, 8300, 4096, 128, torch.float16)])
def test_many_columns(gpu_device, m, n, k, group, dtype):
    """More columns than the compute units take at once, rows that do not fit LDS together with their scales."""
    print(f"[w4a16] {m}x{n}x{k} group {group} {dtype}", flush=True)
    qw, ws, wz = _weights(n, k, group, "float" if group == 128 else "u4", gpu_device)
    x = torch.randn((m, k), device=gpu_device).to(dtype)
    y = ck.w4a16_linear(x, qw, ws, wz, group_size=group)
    at = torch.cat([torch.arange(40), torch.arange(n // 2, n // 2 + 40), torch.arange(n - 40, n)]).to(gpu_device)
    _check(x, qw[at], ws[at], wz[at], None, y[:, at], group, 0)
    assert torch.isfinite(y.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group,zeros,dtype", [(1, 100, 8192, 64, "none", torch.bfloat16), (3, 333, 5120, 128, "float", torch.float16),
                                                     (4, 2000, 4160, 64, "u4", torch.float16), (2, 40, 9000 // 32 * 32, 32, "u4", torch.bfloat16),
                                                     (1, 17, 32768, 128, "u4", torch.float32)])
def test_few_columns_of_long_rows(gpu_device, m, n, k, group, zeros, dtype):
    print(f"[w4a16] {m}x{n}x{k} group {group} {zeros} {dtype}", flush=True)
    qw, ws, wz = _weights(n, k, group, zeros, gpu_device)
    x = torch.randn((m, k), device=gpu_device).to(dtype)
    _check(x, qw, ws, wz, None, ck.w4a16_linear(x, qw, ws, wz, group_size=group), group, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sdt", [torch.bfloat16, torch.float32])
def test_types(gpu_device, out, sdt):
    qw, ws, wz = _weights(100, 512, 64, "float", gpu_device, sdt=sdt)
    x = torch.randn((3, 7, 512), device=gpu_device).to(torch.bfloat16)
    bias = torch.randn(100, device=gpu_device)
    y = ck.w4a16_linear(x, qw.view(torch.int8), ws, wz, bias, out_dtype=out)
    assert y.shape == (3, 7, 100) and y.dtype == out
    _check(x.view(21, 512), qw, ws, wz, bias, y.view(21, 100), 64, 0)


@pytest.mark.gpu
def test_strides(gpu_device):
    """Weights and scales as slices of wider tensors, rows of x that have to be copied."""
    qw, ws, wz = _weights(50, 512, 64, "u4", gpu_device)
    x = torch.randn((2, 512), device=gpu_device).to(torch.bfloat16)
    want = ck.w4a16_linear(x, qw, ws, wz)
    wide = torch.zeros((50, 512), dtype=torch.uint8, device=gpu_device)
    wide[:, 64:320] = qw
    sw = torch.zeros((50, 20), dtype=torch.float16, device=gpu_device)
    sw[:, 3:11] = ws
    assert torch.equal(ck.w4a16_linear(x, wide[:, 64:320], sw[:, 3:11], wz), want)
    wide[:, 7:263] = qw
    assert torch.equal(ck.w4a16_linear(x, wide[:, 7:263], sw[:, 3:11], wz), want)
    odd = torch.zeros(1025, dtype=torch.bfloat16, device=gpu_device)
    odd[1:] = x.reshape(-1)
    assert torch.equal(ck.w4a16_linear(odd[1:].view(2, 512), qw, ws, wz), want)
    assert torch.equal(ck.w4a16_linear(x.t().contiguous().t(), qw, ws, wz), want)


@pytest.mark.gpu
def test_converted_checkpoint(gpu_device):
    """The weights of the framework's own quantizers: the linear agrees with the float weight to what 4 bits leave."""
    g = torch.Generator(device=gpu_device).manual_seed(1)
    w = torch.randn((512, 1024), generator=g, device=gpu_device) * 0.02
    x = torch.randn((4, 1024), generator=g, device=gpu_device).to(torch.bfloat16)
    want = x.float() @ w.t()
    for make, zero in ((ck.quantize_w4a8_asym_weight, True), (ck.quantize_w4a4_group_weight, False)):
        q = make(w, 64, 256)
        y = ck.w4a16_linear(x, q[0], q[1], q[2] if zero else None, convrot_groupsize=256)
        assert float((y.float() - want).norm() / want.norm()) < 0.15
        _check(x, q[0].view(torch.uint8), q[1], q[2].view(torch.uint8) if zero else None, None, y, 64, 256)


@pytest.mark.gpu
def test_values_that_are_not_finite(gpu_device):
    """An infinity in one row of x stays in that row; a NaN scale stays in its column."""
    qw, ws, _ = _weights(64, 256, 64, "none", gpu_device)
    x = torch.randn((3, 256), device=gpu_device).to(torch.bfloat16)
    want = ck.w4a16_linear(x, qw, ws)
    x2, ws2 = x.clone(), ws.clone()
    x2[1, 5] = float("inf")
    y = ck.w4a16_linear(x2, qw, ws)
    assert torch.equal(y[[0, 2]], want[[0, 2]]) and not torch.isfinite(y[1].float()).any()
    ws2[7, 1] = float("nan")
    y = ck.w4a16_linear(x, qw, ws2)
    keep = torch.arange(64, device=gpu_device) != 7
    assert torch.equal(y[:, keep], want[:, keep]) and torch.isnan(y[:, 7].float()).all()


@pytest.mark.gpu
def test_every_time_the_same_and_on_another_stream(gpu_device):
    qw, ws, wz = _weights(500, 2048, 64, "u4", gpu_device)
    x = torch.randn((2, 2048), device=gpu_device).to(torch.bfloat16)
    want = ck.w4a16_linear(x, qw, ws, wz, convrot_groupsize=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ck.w4a16_linear(x, qw, ws, wz, convrot_groupsize=64) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
