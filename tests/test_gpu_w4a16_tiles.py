"""w4a16_linear where a workgroup goes through several column tiles: every column against 64 bits, at row lengths whose
wave shares are and are not whole rounds of the kernel's ring of loads.

Tolerance for outputs of unit roundoff u: one rounding of the output (u |y|); fp32 sums over a group and then over the
groups, of codes that are held shifted by at most 32 (so of terms up to |x| s (|c| + 32)): a relative error of at
most (group + K / group + 40) 2^-24 of the terms' magnitudes; rotated rows for a 16-bit output are held to 16 bits of
each value, the two parts cut off: 2^-15 of the products' magnitudes, and the rotation rounds in fp32."""
import pytest
import torch

import kitchen_amd as ck
from oracle import hadamard

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def weights(n, k, group, zeros, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    qw = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8, device=dev)
    ws = (torch.rand((n, k // group), generator=g, device=dev) * 0.02 + 0.001).half()
    if zeros == "u4":
        wz = torch.randint(0, 256, (n, (k // group + 1) // 2), generator=g, dtype=torch.uint8, device=dev)
    else:
        wz = (-torch.rand((n, k // group), generator=g, device=dev) * 0.1).half() if zeros == "float" else None
    return qw, ws, wz


def exact(x, qw, ws, wz, group, block):
    """(y, spread) in 64 bits; spread: sum |x'| |w|; terms: sum |x'| (|w| + 32 s)."""
    n, k = qw.shape[0], 2 * qw.shape[1]
    x = x.double()
    if block:
        h = torch.from_numpy(hadamard.hadamard(block)).to(x)
        x = (x.reshape(-1, block) @ h).view(x.shape)
    code = torch.stack([qw & 15, qw >> 4], -1).view(n, k // group, group).double()
    s = ws.double()[..., None]
    if wz is None:
        w = (code - 16 * (code > 7)) * s
    elif wz.dtype == torch.uint8:
        w = (code - torch.stack([wz & 15, wz >> 4], -1).view(n, -1)[:, : k // group, None].double()) * s
    else:
        w = code * s + wz.double()[..., None]
    terms = (w.abs() + 32 * s).view(n, k)
    w = w.view(n, k)
    return x @ w.t(), x.abs() @ w.abs().t(), x.abs() @ terms.t()


def check(y, x, qw, ws, wz, group, block):
    k = x.shape[1]
    want, spread, terms = exact(x, qw, ws, wz, group, block)
    tol = U[y.dtype] * want.abs() + (group + k / group + 40) * 2.0 ** -24 * terms + (2.0 ** -15 * spread if block else 0) + 1e-30
    out = (y.double() - want).abs() > tol
    assert not out.any(), f"{int(out.any(0).sum())} of {y.shape[1]} columns, the first {int(out.any(0).nonzero()[0])}"


FORMS = [(5, torch.bfloat16, 0), (8, torch.float16, 0), (16, torch.bfloat16, 0), (3, torch.bfloat16, 256), (8, torch.float16, 64),
         (2, torch.float32, 0), (5, torch.float32, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4500, 18432])
@pytest.mark.parametrize("k", [256, 1024, 2048, 2560, 3072, 3648, 4096, 5120, 7168])
@pytest.mark.parametrize("m,dtype,block", FORMS)
def test_every_column_of_several_tiles(gpu_device, m, dtype, block, k, n):
    block = block if block and k % block == 0 else 0
    for zeros in ("none", "u4", "float"):
        print(f"[w4a16] {m}x{n}x{k} block {block} {dtype} {zeros}", flush=True)
        qw, ws, wz = weights(n, k, 64, zeros, gpu_device)
        x = torch.randn((m, k), generator=torch.Generator(device=gpu_device).manual_seed(m), device=gpu_device).to(dtype)
        check(ck.w4a16_linear(x, qw, ws, wz, None, 64, block or None), x, qw, ws, wz, 64, block)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group,dtype", [(16, 8300, 1152, 128, torch.float16), (7, 9000, 1056, 32, torch.bfloat16),
                                               (16, 12300, 640, 32, torch.float32), (40, 5000, 1664, 128, torch.bfloat16)])
def test_other_groups(gpu_device, m, n, k, group, dtype):
    print(f"[w4a16] {m}x{n}x{k} group {group} {dtype}", flush=True)
    qw, ws, wz = weights(n, k, group, "u4", gpu_device)
    x = torch.randn((m, k), device=gpu_device).to(dtype)
    check(ck.w4a16_linear(x, qw, ws, wz, None, group), x, qw, ws, wz, group, 0)
