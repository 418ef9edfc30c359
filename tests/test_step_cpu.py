"""Refusals of the calls around a step's linears (norms, turned tokens, shared pages, sampling) and the plain loops they are
tested against. CPU only: every call fails its checks or is empty, so nothing is launched."""
import ctypes
import math

import numpy as np
import pytest
import torch

import kitchen_amd as ck
from kitchen_amd import _lib, kv
from oracle import step

A = 1 << 20   # a fake aligned address: never dereferenced

NORM = dict(x=A, dtype=0, ldx=64, r=A, ldr=64, w=A, w_dtype=2, eps=1e-6, h=A, ldh=64, y=A, ldy=64, M=3, K=64, stream=None)
QUANT = dict(x=A, dtype=0, ldx=64, r=A, ldr=64, w=A, w_dtype=2, eps=1e-6, block=0, h=A, ldh=64, q=A, ldq=64, s=A, M=3, K=64,
             stream=None)
APPEND = dict(q=A, q_token=1024, q_head=128, out=A, o_token=1024, o_head=128, Hq=8, k=A, k_token=512, k_head=128, v=A, v_token=512,
              v_head=128, dtype=0, T=3, H=4, D=128, kc=A, vc=A, cdt=0, c_page=8192, c_head=2048, c_token=128, ks=None, vs=None,
              s_page=0, s_head=0, s_token=0, pages=9, page=16, table=A, ld=4, B=3, width=4, lens=A, cu=None, freq=A, turn=128,
              interleaved=0, size=1.0, stream=None)
PLAN = dict(table=A, ld=4, rows=3, width=4, lens=A, page=16, least=0, plan=A, stream=None)
SHARED = dict(q=A, q_token=1024, q_head=128, dtype=0, B=3, Hq=8, H=4, D=128, kc=A, vc=A, cdt=0, c_page=8192, c_head=2048,
              c_token=128, ks=None, vs=None, s_page=0, s_head=0, s_token=0, pages=9, page=16, table=A, ld=4, width=4,
              lens=A, plan=A, scale=0.1, out=A, out_token=1024, out_head=128, work=A, work_bytes=1 << 30, counters=A, stream=None)
SAMPLE = dict(x=A, dtype=0, ld=100, rows=3, V=100, u=A, t=None, t1=1.0, k=None, k1=0, p=None, p1=1.0, m=None, m1=0.0, token=A,
              work=None, work_bytes=0, stream=None)

REFUSED = [
    ("mq_rms_norm", NORM, dict(dtype=3), "input type"), ("mq_rms_norm", NORM, dict(w_dtype=-1), "weight type"),
    ("mq_rms_norm", NORM, dict(K=0), "bad shape"), ("mq_rms_norm", NORM, dict(M=-1), "bad shape"),
    ("mq_rms_norm", NORM, dict(ldx=63), "strides"), ("mq_rms_norm", NORM, dict(ldy=63), "strides"),
    ("mq_rms_norm", NORM, dict(ldr=0), "strides"), ("mq_rms_norm", NORM, dict(ldh=1), "strides"),
    ("mq_rms_norm", NORM, dict(x=None), "null"), ("mq_rms_norm", NORM, dict(h=None), "null"), ("mq_rms_norm", NORM, dict(y=None), "null"),
    ("mq_rms_norm", NORM, dict(x=A + 1), "aligned"), ("mq_rms_norm", NORM, dict(w=A + 2), "aligned"),
    ("mq_rms_norm", NORM, dict(dtype=2, r=A + 2), "aligned"),
    ("mq_rms_norm_quant", QUANT, dict(block=32), "group size"), ("mq_rms_norm_quant", QUANT, dict(block=256), "not a multiple"),
    ("mq_rms_norm_quant", QUANT, dict(s=None), "scale"), ("mq_rms_norm_quant", QUANT, dict(q=None), "null"),
    ("mq_rms_norm_quant", QUANT, dict(ldq=60), "strides"),
    ("mq_kv_append", APPEND, dict(dtype=2), "type"), ("mq_kv_append", APPEND, dict(turn=136), "turned"),
    ("mq_kv_append", APPEND, dict(turn=12), "turned"), ("mq_kv_append", APPEND, dict(turn=-8), "turned"),
    ("mq_kv_append", APPEND, dict(freq=None), "frequencies"), ("mq_kv_append", APPEND, dict(freq=A + 4), "frequencies"),
    ("mq_kv_append", APPEND, dict(q=None), "q and out"), ("mq_kv_append", APPEND, dict(o_head=129), "q and out"),
    ("mq_kv_append", APPEND, dict(k=A + 8), "k and v"), ("mq_kv_append", APPEND, dict(Hq=-1), "heads"),
    ("mq_kv_append", APPEND, dict(T=4), "without cu_q"), ("mq_kv_append", APPEND, dict(cdt=3), "scales"),
    ("mq_kv_append", APPEND, dict(page=12), "power of two"), ("mq_kv_append", APPEND, dict(lens=None), "lens"),
    ("mq_kv_shared", PLAN, dict(page=0), "power of two"), ("mq_kv_shared", PLAN, dict(plan=None), "plan"),
    ("mq_kv_shared", PLAN, dict(lens=None), "lens"), ("mq_kv_shared", PLAN, dict(table=None), "page_table"),
    ("mq_kv_shared", PLAN, dict(ld=3), "page_table"), ("mq_kv_shared", PLAN, dict(rows=-1), "bad shape"),
    ("mq_kv_shared", PLAN, dict(width=1 << 28, ld=1 << 28), "too many tokens"),
    ("mq_paged_attention_shared", SHARED, dict(Hq=6), "query heads"), ("mq_paged_attention_shared", SHARED, dict(plan=None), "plan"),
    ("mq_paged_attention_shared", SHARED, dict(plan=A + 2), "plan"), ("mq_paged_attention_shared", SHARED, dict(work_bytes=64), "workspace"),
    ("mq_paged_attention_shared", SHARED, dict(work=None), "workspace"), ("mq_paged_attention_shared", SHARED, dict(counters=None), "counters"),
    ("mq_paged_attention_shared", SHARED, dict(q=None), "16-byte"), ("mq_paged_attention_shared", SHARED, dict(out_token=4), "16 bytes"),
    ("mq_paged_attention_shared", SHARED, dict(D=260), "head width"), ("mq_paged_attention_shared", SHARED, dict(dtype=2), "type"),
    ("mq_paged_attention_shared", SHARED, dict(width=1 << 30, ld=1 << 30, page=1024), "too many tokens"),
    ("mq_sample", SAMPLE, dict(dtype=3), "unknown type"), ("mq_sample", SAMPLE, dict(V=0), "bad shape"),
    ("mq_sample", SAMPLE, dict(rows=-1), "bad shape"), ("mq_sample", SAMPLE, dict(ld=99), "row stride"),
    ("mq_sample", SAMPLE, dict(u=None), "null"), ("mq_sample", SAMPLE, dict(token=None), "null"),
    ("mq_sample", SAMPLE, dict(t=A + 2), "aligned"), ("mq_sample", SAMPLE, dict(token=A + 4), "aligned"),
    ("mq_sample", SAMPLE, dict(V=1 << 20, ld=1 << 20), "workspace"), ("mq_sample", SAMPLE, dict(V=1 << 20, ld=1 << 20, work=A + 4, work_bytes=1 << 40), "workspace"),
]


@pytest.mark.parametrize("name,good,bad,message", REFUSED, ids=[f"{r[0]}-{'-'.join(r[2])}" for r in REFUSED])
def test_refused_before_launch(name, good, bad, message):
    _lib.load()
    args = list({**good, **bad}.values())
    with pytest.raises(ValueError, match=message):
        _lib.call(name, *args)
    slow = getattr(_lib.load(), name)
    assert slow(*args) == -1 and message in _lib.load().mq_last_error().decode()


@pytest.mark.parametrize("name,args", [("mq_rms_norm", dict(NORM, K=32769, ldx=32769, ldr=32769, ldh=32769, ldy=32769)),
                                       ("mq_rms_norm_quant", dict(QUANT, K=40960, ldx=40960, ldr=40960, ldh=40960, ldq=40960)),
                                       ("mq_sample", dict(SAMPLE, V=(1 << 24) + 1, ld=1 << 25))])
def test_too_long_rows_are_unsupported(name, args):
    with pytest.raises(ck.MQError, match="exceeds"):
        _lib.call(name, *args.values())


EMPTY = [("mq_rms_norm", NORM, dict(M=0)), ("mq_rms_norm_quant", QUANT, dict(M=0)), ("mq_kv_append", APPEND, dict(T=0, B=0)),
         ("mq_paged_attention_shared", SHARED, dict(B=0)), ("mq_sample", SAMPLE, dict(rows=0))]


@pytest.mark.parametrize("name,good,empty", EMPTY)
def test_empty_calls_do_nothing_and_the_fast_calls_take_what_ctypes_takes(name, good, empty):
    """Pointers may be None and nothing else may; floats are numbers of any kind."""
    lib = _lib.load()
    args, kinds = list({**good, **empty}.values()), _lib._SIGNATURES[name][0]
    assert name in _lib.FAST_ENTRIES and len(args) == len(kinds)
    _lib.call(name, *args)
    for i, kind in enumerate(kinds):
        one = args[:i] + [None] + args[i + 1:]
        if kind is ctypes.c_void_p:
            assert _lib._entries[name](*one) == getattr(lib, name)(*one)
        else:
            with pytest.raises(TypeError):
                _lib._entries[name](*one)
            if kind is ctypes.c_float:
                for x in (1, 0.25, True):
                    assert _lib._entries[name](*args[:i], x, *args[i + 1:]) == 0
    with pytest.raises(TypeError, match="arguments"):
        _lib._entries[name](*args[:-1])


def test_host_tensors_are_refused():
    x, i = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    cache, table = torch.zeros((3, 4, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 2), dtype=torch.int32)
    rotary = ck.Rotary(64, device="cpu")
    for call in (lambda: ck.rms_norm(x), lambda: ck.rms_norm_quantize(x), lambda: ck.sample(x[0], torch.zeros(4)),
                 lambda: ck.kv_append(x, x, x, cache, cache, table, i, rotary), lambda: ck.kv_shared(table, i, 16)):
        with pytest.raises(ValueError, match="device tensor"):
            call()


@pytest.fixture
def host(monkeypatch):
    """The Python checks on host tensors; calls into the library are recorded."""
    from kitchen_amd import step as module

    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "stream_of_device", lambda dev: 0)
    monkeypatch.setattr(kv, "_device_of", lambda t, what: t.device)
    monkeypatch.setattr(kv, "_scratch", lambda n, dev, stream: torch.zeros(4))
    monkeypatch.setattr(kv, "_counters", lambda n, dev, stream: torch.zeros(4, dtype=torch.int32))
    monkeypatch.setattr(module, "_device_check", lambda t, what: None)
    monkeypatch.setattr(module, "_SAMPLE_WS", {(None, 3, 50): 0})
    return seen


def refused(match, f, *args, **kw):
    with pytest.raises(ValueError, match=match):
        f(*args, **kw)


def test_norm_arguments(host):
    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    refused("bfloat16, float16 or float32", ck.rms_norm, x.double())
    refused("at least one dimension", ck.rms_norm, x[0, 0])
    refused("residual must be", ck.rms_norm, x, None, x.float())
    refused("residual must be", ck.rms_norm, x, None, x[:2])
    refused("residual must be", ck.rms_norm, x, None, torch.empty((3, 64), dtype=torch.bfloat16, device="meta"))
    refused("weight must be", ck.rms_norm, x, torch.zeros(63))
    refused("weight must be", ck.rms_norm, x, torch.zeros(64, dtype=torch.int8))
    refused("weight must be", ck.rms_norm, x, torch.zeros(64, device="meta"))
    refused("32768", ck.rms_norm, torch.zeros((1, 32769)))
    refused("1 to", ck.rms_norm, torch.zeros((3, 0)))
    refused("convrot_groupsize must", ck.rms_norm_quantize, x, convrot_groupsize=32)
    refused("not divisible", ck.rms_norm_quantize, x, convrot_groupsize=256)
    assert not host
    # rows that overlap or are not contiguous are copied
    for t in (x[:1].expand(3, 64), torch.zeros((64, 3), dtype=torch.bfloat16).t(), torch.zeros((3, 128), dtype=torch.bfloat16)[:, ::2]):
        host.clear()
        ck.rms_norm(t)
        assert host[0][1][0] != t.data_ptr() and host[0][1][2] == 64
    ck.rms_norm(torch.zeros((3, 99), dtype=torch.bfloat16)[:, 1:65])
    assert host[-1][1][2] == 99


def test_sample_arguments(host):
    x, u = torch.zeros((3, 50)), torch.zeros(3)
    refused("logits must be", ck.sample, x[0], u[:1])
    refused("logits must be", ck.sample, x.double(), u)
    refused("1 to", ck.sample, x[:, :0], u)
    refused("u must be", ck.sample, x, u.double())
    refused("u must be", ck.sample, x, u[:2])
    refused("u must be", ck.sample, x, torch.zeros(3, device="meta"))
    refused("temperature must be", ck.sample, x, u, torch.ones(2))
    refused("top_k must be", ck.sample, x, u, top_k=torch.ones(3))
    refused("top_p must be", ck.sample, x, u, top_p=torch.ones(3, dtype=torch.int32))
    refused("min_p must be", ck.sample, x, u, min_p=torch.ones((3, 1)))
    refused("min_p must be", ck.sample, x, u, min_p=torch.ones(3, device="meta"))
    assert not host
    ck.sample(x, u, torch.ones(3, dtype=torch.float16), torch.tensor([1 << 40, -5, 7]), 0.5, torch.ones(3, dtype=torch.float64))
    args = host[0][1]
    assert args[6] is not None and args[8] is not None and args[10] is None and args[11] == 0.5 and args[12] is not None


def test_append_arguments(host):
    q, k = torch.zeros((3, 8, 64), dtype=torch.bfloat16), torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    cache, table, lens = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    r = ck.Rotary(64, device="cpu")

    def call(q=q, k=k, v=k, kc=cache, vc=cache, table=table, lens=lens, r=r, **kw):
        return ck.kv_append(q, k, v, kc, vc, table, lens, r, **kw)

    refused("k and v must be alike", call, v=k[:2])
    refused("k and v must be alike", call, v=k.half())
    refused("q must be", call, q=q[:2])
    refused("q must be", call, q=q.half())
    refused("q must be", call, q=q[..., :32])
    refused("values to turn", call, r=ck.Rotary(128, device="cpu"))
    refused("frequencies are on", call, r=ck.Rotary(64, device="meta"))
    refused("caches of", call, kc=cache[:, :1], vc=cache[:, :1])
    refused("page_table must", call, table=table.long())
    refused("kv_lens must", call, lens=lens[:2])
    refused("cu_q must", call, cu_q=lens)
    refused("out must be", call, out=q.half())
    refused("out must be", call, out=torch.zeros((3, 8, 65), dtype=torch.bfloat16)[..., 1:])
    refused("scales are for", call, k_scale=cache[..., 0].float())
    assert not host
    assert call().shape == q.shape and host[0][0] == "mq_kv_append"


def test_shared_arguments(host, monkeypatch):
    q = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    cache, table, lens = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    refused("page_table must be", ck.kv_shared, table.long(), lens, 16)
    refused("kv_lens must be", ck.kv_shared, table, lens[:2], 16)
    refused("kv_lens must be", ck.kv_shared, table, lens.long(), 16)
    assert not host
    plan = ck.kv_shared(table[:1].expand(3, 2), lens, 16)
    assert plan.shape == (_lib.load().mq_kv_shared_ints(3),) and host[0][1][0] != table.data_ptr()
    cu = torch.zeros(4, dtype=torch.int32)
    for kw in (dict(cu_q=cu), dict(window=5)):
        refused("one new token per sequence", ck.paged_attention, q, cache, cache, table, lens, shared=plan, **kw)
    for bad in (plan[:-1], plan.long(), torch.zeros(plan.shape, dtype=torch.int32, device="meta")):
        refused("kv_shared's plan", ck.paged_attention, q, cache, cache, table, lens, shared=bad)
    assert len(host) == 1


def test_rotary_arguments_and_frequencies():
    for bad in (dict(dim=12), dict(dim=0), dict(dim=264), dict(base=1.0), dict(factor=0.0), dict(beta_fast=1.0), dict(original=0)):
        refused("must be", ck.Rotary, **dict(dict(dim=64, device="cpu"), **bad))
    refused("scaling must be", ck.Rotary, 64, scaling="longer", device="cpu")
    for kw in (dict(), dict(base=1e6), dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=8.0, original=4096),
               dict(scaling="yarn", factor=40.0, original=2048, base=5e5)):
        for dim in (8, 64, 80, 128, 256):
            f, size = step.frequencies(dim, **kw)
            r = ck.Rotary(dim, device="cpu", **kw)
            got = r.turns.numpy().view(np.uint64).astype(np.float64) / 2.0 ** 64 * 2 * math.pi
            # fp64 formulas (some roundings of 2^-53 each), then a fraction rounded to 2^-64 of a turn: half of that is
            # pi 2^-64 = 1.7e-19 radians a position
            assert np.allclose(got, f, rtol=1e-13, atol=2e-19) and math.isclose(r.size, size)
    assert ck.Rotary(64, scaling="yarn", factor=2.0, size=1.5, device="cpu").size == 1.5


def test_plain_sampling_is_the_softmax():
    rng = np.random.default_rng(0)
    x = rng.normal(size=40)
    p = np.exp(x / 0.7) / np.exp(x / 0.7).sum()
    got = np.bincount([step.sample(x, (i + 0.5) / 20000, 0.7) for i in range(20000)], minlength=40)
    assert np.abs(got - 20000 * p).max() <= 1
    best = np.argsort(-x)
    assert {step.sample(x, u, 0.7, top_k=5) for u in np.linspace(0, 0.999, 400)} == set(best[:5].tolist())
    n = int(np.searchsorted(np.cumsum(p[best]), 0.6)) + 1
    assert {step.sample(x, u, 0.7, top_p=0.6) for u in np.linspace(0, 0.999, 2000)} == set(best[:n].tolist())
    assert {step.sample(x, u, 0.7, min_p=0.5) for u in np.linspace(0, 0.999, 2000)} == set(np.flatnonzero(p >= 0.5 * p.max()).tolist())
    assert step.sample([1.0, 3.0, 3.0], 0.9, 0.0) == 1 and step.sample([-np.inf, np.nan], 0.5) == -1


def test_plain_turn_is_a_rotation():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(4, 2, 24))
    f, _ = step.frequencies(16)
    for interleaved in (False, True):
        y = step.turn(x, [0, 1, 5, 9], f, 1.0, interleaved)
        assert np.allclose(y[0], x[0]) and np.allclose(y[..., 16:], x[..., 16:])
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
        # scores depend on the distance of two positions only
        a = step.turn(x[:1], [7], f, 1.0, interleaved) * step.turn(x[1:2], [3], f, 1.0, interleaved)
        b = step.turn(x[:1], [104], f, 1.0, interleaved) * step.turn(x[1:2], [100], f, 1.0, interleaved)
        assert np.allclose(a.sum(-1), b.sum(-1))
