"""The host side of the calls around a step's linears, on the CPU: what settings, classes and shapes they take, and what is handed
to the library. Host tensors stand for device tensors and nothing is launched."""
import ctypes
import math

import pytest
import torch

import kitchen_amd as ck
from kitchen_amd import _lib, kv
from test_step_cpu import host  # noqa: F401  (the library's calls, recorded)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_top_k_of_any_whole_number_type(host, dtype):
    """The kernel reads int32: every type of whole numbers comes as that, int64 beyond its range at its end."""
    from kitchen_amd import step

    values = [0, 5, 100] if dtype is torch.uint8 else [-1, 5, 100]
    _, _, got = step._setting(torch.tensor(values, dtype=dtype), "top_k", 3, torch.int32, torch.device("cpu"))
    assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == values
    strided = torch.tensor([v for x in values for v in (x, 1)], dtype=dtype)[::2]
    assert step._setting(strided, "top_k", 3, torch.int32, torch.device("cpu"))[2].tolist() == values
    ck.sample(torch.zeros((3, 50)), torch.zeros(3), top_k=torch.tensor(values, dtype=dtype))
    assert host[-1][0] == "mq_sample"
    if dtype is torch.int64:
        far = step._setting(torch.tensor([1 << 40, -(1 << 40), 3]), "top_k", 3, torch.int32, torch.device("cpu"))[2]
        assert far.tolist() == [(1 << 31) - 1, -1, 3]


def test_outputs_are_plain_tensors(host, monkeypatch):
    """The outputs are the library's own buffers, not the class of what goes in."""
    class Tagged(torch.Tensor):
        pass

    def tagged(t):
        return t.as_subclass(Tagged)

    x, w = tagged(torch.zeros((3, 64), dtype=torch.bfloat16)), tagged(torch.ones(64))
    norms = [ck.rms_norm(x, w), *ck.rms_norm(x, w, x), *ck.rms_norm_quantize(x, w, x), ck.rms_norm(x[:, ::2]),
             ck.rms_norm(torch.nn.Parameter(torch.zeros(3, 64)))]
    q = tagged(torch.zeros((3, 8, 64), dtype=torch.bfloat16))
    cache, table, lens = torch.zeros((5, 8, 16, 64), dtype=torch.bfloat16), torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    turned = ck.kv_append(q, q, q, cache, cache, table, lens, ck.Rotary(64, device="cpu"))
    monkeypatch.setattr(kv, "_ATTN_WS", {(None, 3, 8, 8, 64, 3, True, False): (0, 0)})
    attended = ck.paged_attention(q, cache, cache, table, lens, shared=ck.kv_shared(tagged(table), tagged(lens), 16))
    token = ck.sample(tagged(torch.zeros((3, 50))), tagged(torch.zeros(3)))
    for y in (*norms, turned, attended, token):
        assert type(y) is torch.Tensor and not y.requires_grad
    assert [(type(y), y.dtype, y.shape) for y in (ck.rms_norm(x[:2, :32]), turned)] == \
        [(torch.Tensor, torch.bfloat16, (2, 32)), (torch.Tensor, torch.bfloat16, (3, 8, 64))]


@pytest.mark.parametrize("shape", [(0,), (3, 0), (2, 3, 0), (2, 0, 5, 0)])
def test_rows_without_values_are_refused(host, shape):
    for call in (ck.rms_norm, ck.rms_norm_quantize):
        for residual in (None, torch.zeros(shape)):
            with pytest.raises(ValueError, match="rows of 1 to"):
                call(torch.zeros(shape), residual=residual)
    assert not host and ck.rms_norm(torch.zeros((2, 0, 5))).shape == (2, 0, 5) and not host


def test_yarn_of_shorter_contexts_keeps_the_size():
    """The size makes up for scores over longer contexts: 0.1 ln(factor) + 1 above 1, else 1."""
    from oracle import step

    for factor, size in ((0.25, 1.0), (0.999, 1.0), (1.0, 1.0), (math.e, 1.1), (math.exp(10), 2.0)):
        r = ck.Rotary(64, scaling="yarn", factor=factor, device="cpu")
        assert math.isclose(r.size, size) and math.isclose(step.frequencies(64, scaling="yarn", factor=factor)[1], size)
    assert ck.Rotary(64, scaling="yarn", factor=0.25, size=0.7, device="cpu").size == 0.7
    assert ck.Rotary(64, scaling="linear", factor=8.0, device="cpu").size == 1.0
