"""Attention arguments at their edges: both forms (one token a sequence, ragged chunks) give the same answer."""
import math

import pytest
import torch

from test_gpu_attention import Setup


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("d", [64, 80])
def test_a_scale_of_nan(gpu_device, d, int8):
    """softmax of NaN is NaN: in every row that sees a key, in no row that sees none."""
    for new in (None, [60, 40, 0], [1, 3, 0]):
        s = Setup(gpu_device, [100, 37, 0], 4, 2, d, new=new, int8=int8, dtype=torch.float16)
        y = s.run(scale=math.nan)
        pos = torch.tensor(s.lens, device=gpu_device) - 1 if new is None else \
            torch.cat([torch.arange(n - m, n) for n, m in zip(s.lens, new)]).to(gpu_device)
        assert y[pos >= 0].isnan().all() and (y[pos < 0] == 0).all()


@pytest.mark.gpu
def test_a_scale_of_nan_over_a_long_cache(gpu_device):
    """Pieces that are joined, and rows behind a window without a page."""
    s = Setup(gpu_device, [5000, 4000], 4, 2, 64, new=[2, 3], page=64)
    s.table[1] = -1
    y = s.run(scale=math.nan)
    assert y[:2].isnan().all() and (y[2:] == 0).all()
    t = Setup(gpu_device, [5000, 4000], 4, 2, 64, page=64)
    t.table[1] = -1
    y = t.run(scale=math.nan)
    assert y[0].isnan().all() and (y[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [math.inf, 2.0 ** -120])
def test_scales_at_the_ends_of_the_range(gpu_device, scale):
    """An infinite scale: weight on the largest score if it is not 0; one too small to tell: the mean."""
    s = Setup(gpu_device, [50, 9], 2, 2, 64, new=[50, 9])
    t = Setup(gpu_device, [50, 9], 2, 2, 64)
    y, z = s.run(scale=scale), t.run(scale=scale)
    assert s.q.shape[0] == 59
    if math.isinf(scale):
        assert y[0].isnan().all() and z.isnan().all()      # the largest is infinite: infinity less itself
    else:
        s.check(y, scale=scale)
        t.check(z, scale=scale)
