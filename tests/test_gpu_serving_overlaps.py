"""One row of a table, of scales or of zero-points expanded to all gives what its copies give."""
import pytest
import torch

import kitchen_amd as ck
from test_gpu_attention import Setup
from test_gpu_w4a16_tiles import weights


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_sequences_of_one_table(gpu_device, ragged):
    s = Setup(gpu_device, [200, 0, 0], 4, 2, 64, new=[50, 0, 0] if ragged else None)
    new = [5, 30, 1]
    q = torch.randn((sum(new) if ragged else 3, 4, 64), device=gpu_device).to(torch.bfloat16)
    cu = torch.tensor([0, 5, 35, 36], dtype=torch.int32, device=gpu_device) if ragged else None
    lens = torch.tensor([200, 77, 9], dtype=torch.int32, device=gpu_device)
    one = s.table[:1].expand(3, -1)
    assert torch.equal(ck.paged_attention(q, s.k, s.v, one, lens, cu), ck.paged_attention(q, s.k, s.v, one.contiguous(), lens, cu))


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", ["u4", "float"])
def test_columns_of_one_scale(gpu_device, zeros):
    qw, ws, wz = weights(300, 512, 64, zeros, gpu_device)
    x = torch.randn((3, 512), device=gpu_device).to(torch.bfloat16)
    s, z = ws[:1].expand(300, -1), wz[:1].expand(300, -1)
    assert torch.equal(ck.w4a16_linear(x, qw, s, z), ck.w4a16_linear(x, qw, s.contiguous(), z.contiguous()))
