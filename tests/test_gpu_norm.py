"""kitchen_amd.rms_norm and rms_norm_quantize against the formula in 64 bits.

Tolerance. h is one fp32 addition rounded to the rows' type: equal to torch's. A row's squares are summed in fp32, at most
64 in one lane and ten additions behind them, each off by 2^-24 of the sum so far: mean off by at most 74 x 2^-24, its root
by half of that; root, division, two products and the epsilon's addition 2^-24 each: y is off by E |y| with
E = 42 x 2^-24 before it is rounded once (half a step, eps / 2; a fp16 below 2^-14 half a step of 2^-24). The rotation's
stages are sums of three additions and a fused product each, four stages: a rotated value is off by (E + 16 x 2^-24) A
with A the sum of its block's |y| over the root of the block's size (A = |y| without one). Codes are within half a
step of z / s, plus what z and s are off by."""
import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import step

E = 42 * 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def rows(m, k, dtype, dev, seed=0, pitch=None, shift=0):
    """[m, k] with a few strong channels, its rows `pitch` apart, `shift` elements into its memory."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    x[:, :: 41] *= 15
    pitch = pitch or k
    mem = torch.full((m * pitch + shift,), float("nan"), dtype=dtype, device=dev)
    y = mem[shift:].view(m, pitch)[:, :k]
    y.copy_(x)
    return y


def check_float(y, h, w, dtype, eps=1e-6):
    want = step.rms_norm(h.double().cpu().numpy(), None if w is None else w.double().cpu().numpy(), eps)
    err = np.abs(y.double().cpu().numpy() - want)
    tol = (torch.finfo(dtype).eps / 2 * (1 + E) + E) * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    assert (err <= tol).all(), f"{(err > tol).mean():.2%} out, worst {(err / tol).max():.2f}"


def check_codes(q, s, h, w, block, eps=1e-6):
    y = step.rms_norm(h.double().cpu().numpy(), None if w is None else w.double().cpu().numpy(), eps)
    z, scale = step.quantize(y, block)
    m, k = y.shape
    a = np.abs(y)
    if block:
        a = np.repeat(np.abs(y).reshape(m, -1, block).sum(-1) / block ** 0.5, block, axis=1)
    dz = (E + (16 * 2.0 ** -24 if block else 0)) * a
    ds = dz.max(-1) / 127 + 2.0 ** -23 * scale
    s = s.double().cpu().numpy()
    assert (np.abs(s - scale) <= ds).all()
    off = np.abs(q.double().cpu().numpy() - z / scale[:, None])
    assert (off <= 0.5 + (dz + 127 * ds[:, None]) / scale[:, None] + 2.0 ** -16).all(), off.max()
    assert q.abs().max() <= 127


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 63), (4, 64), (7, 511), (3, 512), (2, 513), (9, 1000), (1, 2048), (66, 4096), (2, 5121),
          (3, 8192), (2, 8193), (1, 16384), (2, 20001), (1, 32768)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(gpu_device, m, k, dtype, residual):
    print(f"[norm] {m} x {k} {dtype} residual {residual}", flush=True)
    x = rows(m, k, dtype, gpu_device, 1)
    w = (1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(2))).to(dtype).to(gpu_device)
    if not residual:
        check_float(ck.rms_norm(x, w), x, w, dtype)
        return
    r = rows(m, k, dtype, gpu_device, 3)
    y, h = ck.rms_norm(x, w, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_float(y, h, w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_codes(gpu_device, m, k, dtype):
    print(f"[norm] codes {m} x {k} {dtype}", flush=True)
    x, r = rows(m, k, dtype, gpu_device, 1), rows(m, k, dtype, gpu_device, 3)
    w = (1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(2))).to(gpu_device)
    q, s, h = ck.rms_norm_quantize(x, w, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_codes(q, s, h, w, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [16, 64, 256])
@pytest.mark.parametrize("m,blocks", [(1, 1), (3, 3), (5, 4), (2, 5), (70, 20), (2, 33), (1, 64), (2, 127)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotated_codes(gpu_device, m, blocks, block, dtype):
    k = block * blocks
    print(f"[norm] codes {m} x {k} rotated by {block} {dtype}", flush=True)
    x = rows(m, k, dtype, gpu_device, 5)
    w = (1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(2))).to(torch.bfloat16).to(gpu_device)
    q, s = ck.rms_norm_quantize(x, w, convrot_groupsize=block)
    check_codes(q, s, x, w, block)


@pytest.mark.gpu
def test_rotated_codes_of_the_longest_rows(gpu_device):
    x = rows(2, 32768, torch.float32, gpu_device, 5)
    q, s = ck.rms_norm_quantize(x, None, x, convrot_groupsize=256)[:2]
    check_codes(q, s, x + x, None, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch,shift", [(1030, 0), (1027, 1), (1024, 3), (2048, 8)])
def test_rows_anywhere(gpu_device, dtype, pitch, shift):
    """Rows at any address that their type allows, a weight that begins there too."""
    print(f"[norm] pitch {pitch} shift {shift} {dtype}", flush=True)
    x, r = rows(5, 1024, dtype, gpu_device, 1, pitch, shift), rows(5, 1024, dtype, gpu_device, 2, pitch, shift)
    w = rows(1, 1024, dtype, gpu_device, 3, None, shift)[0]
    y, h = ck.rms_norm(x, w, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_float(y, h, w, dtype)
    q, s, h = ck.rms_norm_quantize(x, w, r, convrot_groupsize=64)
    check_codes(q, s, h, w, 64)


@pytest.mark.gpu
def test_shapes_and_strides(gpu_device):
    """More dimensions, an expanded residual, a transposed input, no rows."""
    x = torch.randn((3, 5, 96), device=gpu_device).to(torch.bfloat16)
    one = torch.randn((1, 5, 96), device=gpu_device).to(torch.bfloat16)
    y, h = ck.rms_norm(x, None, one.expand(3, 5, 96))
    assert y.shape == x.shape and h.shape == x.shape
    assert torch.equal(h, (x.float() + one.float()).to(torch.bfloat16))
    check_float(y.view(-1, 96), h.view(-1, 96), None, torch.bfloat16)
    q, s, h2 = ck.rms_norm_quantize(x, None, one.expand(3, 5, 96))
    assert q.shape == (15, 96) and torch.equal(h, h2)
    t = torch.randn((96, 7), device=gpu_device).t()
    check_float(ck.rms_norm(t), t, None, torch.float32)
    assert ck.rms_norm(x[:0]).shape == (0, 5, 96)
    q, s = ck.rms_norm_quantize(x[:0])
    assert q.shape == (0, 96) and s.shape == (0,)


@pytest.mark.gpu
def test_values_at_the_ends(gpu_device):
    """Zeros, the smallest and largest values, and rows that hold what is no number: alone in their row."""
    x = torch.ones((6, 300), device=gpu_device)
    x[0] = 0
    x[1] = 1e-30
    x[2] = 1e17
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y = ck.rms_norm(x, eps=1e-6)
    assert not y[0].any() and torch.allclose(y[1], torch.full_like(y[1], 1e-27), rtol=1e-5)
    assert torch.allclose(y[2], torch.ones_like(y[2]), rtol=1e-5) and torch.allclose(y[5], torch.ones_like(y[5]), rtol=1e-5)
    assert y[3].isnan().all() and y[4, 9].isnan()
    for block in (None, 256):
        z = x if block is None else torch.cat([x, x], 1)[:, :512].contiguous()
        q, s = ck.rms_norm_quantize(z, convrot_groupsize=block)
        assert (s[3:5].isnan()).all() and not q[3:5].any() and not q[0].any()
        assert torch.isfinite(s[[0, 1, 2, 5]]).all() and s[0] == torch.tensor(1e-10)
    check_codes(*ck.rms_norm_quantize(x[5:]), x[5:], None, 0)


@pytest.mark.gpu
def test_codes_run_in_the_linear(gpu_device):
    """Codes of the fused call and of norm, rotation and quantizer one by one give the linear nearly the same: the latter round
    the norm to 16 bits in between (2^-8 each, of random signs)."""
    from kitchen_amd import weights

    w = torch.randn((512, 1024), device=gpu_device)
    qd, sc, z = weights.quantize_w4a8_asym_weight(w, 64, 256)
    x, r = rows(9, 1024, torch.bfloat16, gpu_device, 1), rows(9, 1024, torch.bfloat16, gpu_device, 2)
    q, s, h = ck.rms_norm_quantize(x, None, r, convrot_groupsize=256)
    got = ck.gemm_w4_group(q, s, qd, sc, z, None, 512).float()
    want = ck.w4a8_int8_linear(ck.rms_norm(x, None, r)[0], qd, sc, None, None, z).float()
    assert (got - want).norm() < 0.01 * want.norm()


@pytest.mark.gpu
def test_streams_and_graphs(gpu_device):
    x, r = rows(33, 777, torch.float16, gpu_device, 1), rows(33, 777, torch.float16, gpu_device, 2)
    want = ck.rms_norm(x, None, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ck.rms_norm(x, None, r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = ck.rms_norm(x, None, r)
        q, s = ck.rms_norm_quantize(y)
    for i in range(3):
        x.copy_(rows(33, 777, torch.float16, gpu_device, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        wy, wh = ck.rms_norm(x, None, r)
        wq, ws = ck.rms_norm_quantize(wy)
        assert torch.equal(y, wy) and torch.equal(h, wh) and torch.equal(q, wq) and torch.equal(s, ws)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(1023, 520), (1024, 512), (1024, 513), (1025, 1537), (1100, 2570), (1030, 5000), (1024, 8191), (1500, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(gpu_device, m, k, dtype):
    """Where a wave has two pieces of a row instead of one, odd numbers of waves, rows that share a workgroup and its last one."""
    print(f"[norm] {m} x {k} {dtype}", flush=True)
    x, r = rows(m, k, dtype, gpu_device, 1), rows(m, k, dtype, gpu_device, 3)
    y, h = ck.rms_norm(x, None, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_float(y, h, None, dtype)
    q, s = ck.rms_norm_quantize(x)
    check_codes(q, s, x, None, 0)
    if k > 16:
        k = k // 16 * 16
        q, s = ck.rms_norm_quantize(x[:, :k], convrot_groupsize=16)
        check_codes(q, s, x[:, :k], None, 16)
