"""Tables, scales and zero-points whose rows overlap in memory (one row expanded to all): what the library is told is
inside the tensors. CPU: the calls into the library are recorded."""
import pytest
import torch

from kitchen_amd import _lib, kv, ops


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "stream_of_device", lambda dev: 0)
    monkeypatch.setattr(kv, "_device_of", lambda t, what: t.device)
    monkeypatch.setattr(ops, "_as_2d", lambda x, k: x)
    return seen


def test_an_expanded_table_is_copied(calls):
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    cache = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    lens = torch.ones(3, dtype=torch.int32)
    one = torch.zeros((1, 4), dtype=torch.int32)
    for table, own in ((one.expand(3, 4), False), (torch.zeros((3, 4), dtype=torch.int32), True),
                       (torch.zeros((3, 9), dtype=torch.int32)[:, :4], True),
                       (torch.zeros(20, dtype=torch.int32).as_strided((3, 4), (2, 1)), False)):
        calls.clear()
        kv.kv_write(k, k, cache, cache, table, lens)
        name, args = calls[0]
        at, ld = args[23], args[24]
        assert name == "mq_kv_write" and ld >= 4
        assert (at == table.data_ptr()) == own and (ld == table.stride(0) or not own)


def test_an_expanded_table_is_not_written(calls):
    table, lens, refs = torch.zeros((1, 4), dtype=torch.int32).expand(3, 4), torch.ones(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
    cache = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    for call in (lambda: kv.kv_grow(table, lens, refs, [0], [1], 16), lambda: kv.kv_free(table, lens, refs, [0]),
                 lambda: kv.kv_fork(cache, cache, table, lens, refs, [0], [1]), lambda: kv.kv_compact(cache, cache, table, refs)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert not calls


@pytest.mark.parametrize("floating", [False, True])
def test_expanded_scales_and_zero_points_are_copied(calls, floating):
    x = torch.zeros((2, 512), dtype=torch.bfloat16)
    qw = torch.zeros((7, 256), dtype=torch.uint8)
    one = torch.ones((1, 8), dtype=torch.float16)
    zero = one if floating else torch.zeros((1, 4), dtype=torch.uint8)
    ops.w4a16_linear(x, qw, one.expand(7, 8), zero.expand(7, zero.shape[1]))
    name, args = calls[0]
    ws, ldws, wz, ldwz = args[6], args[8], args[9], args[12]
    assert name == "mq_linear_w4a16" and ldws == 8 and ldwz == zero.shape[1]
    assert ws != one.data_ptr() and wz != zero.data_ptr()
    calls.clear()
    s, z = torch.ones((7, 8), dtype=torch.float16), torch.zeros((7, zero.shape[1]), dtype=zero.dtype)
    ops.w4a16_linear(x, qw, s, z)
    assert calls[0][1][6] == s.data_ptr() and calls[0][1][9] == z.data_ptr()
