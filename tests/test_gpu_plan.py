"""What a plan of shared pages (kv_shared) says beside its groups, and what the attention makes of it."""
import pytest
import torch

import kitchen_amd as ck
from kitchen_amd import _lib
from test_gpu_shared import MIXED, Forks, read


def plan_of(s, page, least):
    """From the library's entry point itself."""
    plan = torch.zeros(ck.kv._plan_ints(len(s.lens)), dtype=torch.int32, device=s.table.device)
    _lib.call("mq_kv_shared", s.table.data_ptr(), s.table.stride(0), *s.table.shape, s.kv_lens.data_ptr(), page, least, plan.data_ptr(),
              _lib.stream_of(s.table))
    return plan


@pytest.mark.gpu
def test_what_can_never_be_saved(gpu_device):
    """Any number of bytes is a least one: from 2^41 on, which no plan holds, nothing is ever shared."""
    s = Forks(gpu_device, [(128, [5, 1, 20]), (64, [0, 3]), (0, [70])], 8, 2, 64, page=64)
    alone = ck.paged_attention(s.q, s.k, s.v, s.table, s.kv_lens)
    shared = s.run()
    assert not torch.equal(alone, shared)
    for least in (-1, -(1 << 62), 0, 1023):
        assert torch.equal(s.run(plan_of(s, 64, least)), shared), least
    for least in ((1 << 41) - 1024, (1 << 41) - 1, 1 << 41, (1 << 41) + 1, 1 << 42, 1 << 62, (1 << 63) - 1):
        plan = plan_of(s, 64, least)
        assert torch.equal(s.run(plan), alone), least
        plan[1] = 2 ** 31 - 1                           # as if everything were saved
        assert torch.equal(s.run(plan), alone), least
    for least in (1 << 60, 1 << 70):
        assert torch.equal(s.run(ck.kv_shared(s.table, s.kv_lens, 64, least)), alone)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_plan_of_another_page_size(gpu_device, int8):
    """It counts tokens in pages that are not the cache's; those of larger ones would take every sequence's own for the lead's."""
    s = Forks(gpu_device, [(200, [30, 9, 61]), (40, [1, 0])], 8, 2, 64, page=16, int8=int8)
    alone = ck.paged_attention(s.q, s.k, s.v, s.table, s.kv_lens, k_scale=s.ks, v_scale=s.vs)
    assert not torch.equal(s.run(), alone)
    for page in (1, 4, 8, 32, 64, 1024):
        plan = plan_of(s, page, 0)
        assert read(plan, len(s.lens))[0]               # there are groups
        y = s.run(plan)
        assert torch.equal(y, alone), page
        s.check(y)


@pytest.mark.gpu
def test_plan_of_anything_of_this_page_size(gpu_device):
    """A plan that kv_shared did not write and that shares by what its head says: every access stays inside, and the next call is
    right."""
    s = Forks(gpu_device, MIXED, 8, 2, 64)
    want, plan = s.run(), s.plan()
    assert plan[3] == 4
    g = torch.Generator().manual_seed(2)
    for i in range(16):
        odd = torch.randint(-3, 40, plan.shape, generator=g, dtype=torch.int32) if i % 3 else torch.randint(-2 ** 31, 2 ** 31 - 1, plan.shape, generator=g, dtype=torch.int64).int()
        odd[0], odd[1], odd[2], odd[3] = (i % 4) * 3, 2 ** 31 - 1, 0, 4
        s.run(odd.to(gpu_device))
    assert torch.equal(s.run(), want)
