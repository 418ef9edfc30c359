"""kv_grow with more sequences and pages than it looks at in one step: the status is that of the whole call."""
import pytest
import torch

import kitchen_amd as ck


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [False, True])
def test_grow_counts_every_sequence(gpu_device, bad):
    """2500 sequences of which the first thousand need more pages than there are; a bad one among the last."""
    print(f"[kv] grow 2500 bad {bad}", flush=True)
    c = ck.PagedKVCache(1, 600, 1, 8, 4, 2500, 64, device=gpu_device)
    counts = [1 + i % 7 for i in range(2500)]
    if bad:
        counts[2400] = 65
    c.grow(range(2500), counts)
    assert int(c.status) == (-1 if bad else sum(-(-n // 4) for n in counts) - 600)
    assert not c.lens.any() and not c.refs.any() and (c.page_table == -1).all()


@pytest.mark.gpu
def test_grow_by_more_pages_than_32_bits_count(gpu_device):
    """1024 sequences of 2^22 one-token pages each: 2^32 pages, of which there are 4."""
    print("[kv] grow 2^32 pages", flush=True)
    table = torch.empty((1024, 1 << 22), dtype=torch.int32, device=gpu_device)
    table[:, :8] = -1
    lens, refs, status = (torch.zeros(n, dtype=torch.int32, device=gpu_device) for n in (1024, 4, 1))
    for more in (0, 1):                              # 2^32, and one more
        counts = [1 << 22] * 1024
        counts[-1] += more - 1
        lens[-1] = 1 - more
        ck.kv_grow(table, lens, refs, range(1024), counts, 1, status)
        assert int(status) == 0x7fffffff
        assert lens[:-1].sum() == 0 and int(lens[-1]) == 1 - more and not refs.any() and (table[:, :8] == -1).all()


@pytest.mark.gpu
def test_a_call_for_no_sequence_is_done(gpu_device):
    """The status of a growth or fork of nothing is 0, whatever the one before it was."""
    c = ck.PagedKVCache(1, 2, 1, 8, 4, 3, 64, device=gpu_device)
    for call in (lambda: c.grow([], []), lambda: c.fork([], [])):
        c.grow([0], [60])
        assert int(c.status) == 13
        call()
        assert int(c.status) == 0
        c.check()
