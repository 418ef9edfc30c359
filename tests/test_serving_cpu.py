"""Refusals of the token-generation calls and the plain loops they are tested against. CPU only: every call fails
its checks or is empty, so nothing is launched."""
import ctypes

import numpy as np
import pytest
import torch

import kitchen_amd as ck
from kitchen_amd import _lib
from oracle import serving

A = 1 << 20   # a fake aligned address: never dereferenced

WRITE = dict(k=A, k_token=512, k_head=128, v=A, v_token=512, v_head=128, dtype=0, T=3, H=4, D=128, kc=A, vc=A, cdt=0,
             c_page=8192, c_head=2048, c_token=128, ks=None, vs=None, s_page=0, s_head=0, s_token=0, pages=9, page=16,
             table=A, ld=4, B=3, width=4, lens=A, cu=None, stream=None)
ATTN = dict(q=A, q_token=1024, q_head=128, dtype=0, T=3, Hq=8, H=4, D=128, kc=A, vc=A, cdt=0, c_page=8192, c_head=2048,
            c_token=128, ks=None, vs=None, s_page=0, s_head=0, s_token=0, pages=9, page=16, table=A, ld=4, B=3, width=4,
            lens=A, cu=None, scale=0.1, window=0, sinks=0, out=A, out_token=1024, out_head=128, work=None, work_bytes=0,
            counters=None, stream=None)
GROW = dict(table=A, ld=4, rows=3, width=4, lens=A, refs=A, pages=9, page=16, seqs=A, counts=A, n=2, status=None, work=A,
            work_bytes=1 << 20, stream=None)
FORK = dict(k=A, v=A, layers=2, layer_bytes=1 << 16, pitch=4096, bytes=4096, ks=None, vs=None, sl=0, sp=0, sb=0, table=A, ld=4,
            rows=3, width=4, lens=A, refs=A, pages=9, page=16, src=A, dst=A, n=2, status=None, work=A, work_bytes=1 << 20,
            stream=None)
FREE = dict(table=A, ld=4, rows=3, width=4, lens=A, refs=A, pages=9, seqs=A, n=2, stream=None)
COMPACT = dict(k=A, v=A, layers=2, layer_bytes=1 << 16, pitch=4096, bytes=4096, ks=None, vs=None, sl=0, sp=0, sb=0, table=A,
               ld=4, rows=3, width=4, refs=A, pages=9, live=A, work=A, work_bytes=1 << 20, stream=None)
W4 = dict(x=A, x_dtype=0, ldx=512, hblock=0, qw=A, ldw=256, ws=A, s_dtype=1, ldws=8, wz=None, zero=0, z_dtype=0, ldwz=0,
          group=64, bias=None, bias_dtype=0, y=A, y_dtype=0, ldy=64, M=2, N=64, K=512, stream=None)

REFUSED = [
    ("mq_kv_write", WRITE, dict(dtype=2), "type"), ("mq_kv_write", WRITE, dict(cdt=1), "cache must have"),
    ("mq_kv_write", WRITE, dict(D=260), "head width"), ("mq_kv_write", WRITE, dict(D=100), "head width"),
    ("mq_kv_write", WRITE, dict(D=136, cdt=3), "multiple of 16"), ("mq_kv_write", WRITE, dict(page=12), "power of two"),
    ("mq_kv_write", WRITE, dict(page=0), "power of two"), ("mq_kv_write", WRITE, dict(T=4), "without cu_q"),
    ("mq_kv_write", WRITE, dict(lens=None), "lens"), ("mq_kv_write", WRITE, dict(table=None), "page_table"),
    ("mq_kv_write", WRITE, dict(ld=3), "page_table"), ("mq_kv_write", WRITE, dict(kc=A + 8), "16-byte"),
    ("mq_kv_write", WRITE, dict(c_token=132), "16 bytes"), ("mq_kv_write", WRITE, dict(cdt=3), "scales"),
    ("mq_kv_write", WRITE, dict(k=None), "k and v"), ("mq_kv_write", WRITE, dict(v_head=4), "k and v"),
    ("mq_kv_write", WRITE, dict(H=0), "bad shape"), ("mq_kv_write", WRITE, dict(c_page=-8192), "negative"),
    ("mq_paged_attention", ATTN, dict(Hq=6), "query heads"), ("mq_paged_attention", ATTN, dict(window=-1), "window"),
    ("mq_paged_attention", ATTN, dict(sinks=-1), "sinks"), ("mq_paged_attention", ATTN, dict(q=A + 2), "16-byte"),
    ("mq_paged_attention", ATTN, dict(out_head=130), "16 bytes"), ("mq_paged_attention", ATTN, dict(dtype=2), "type"),
    ("mq_paged_attention", ATTN, dict(width=1 << 30, ld=1 << 30, page=1024), "too many tokens"),
    ("mq_kv_grow", GROW, dict(page=3), "power of two"), ("mq_kv_grow", GROW, dict(seqs=None), "sequences"),
    ("mq_kv_grow", GROW, dict(work_bytes=8), "workspace"), ("mq_kv_grow", GROW, dict(work=A + 4), "workspace"),
    ("mq_kv_grow", GROW, dict(refs=None), "refs"), ("mq_kv_grow", GROW, dict(n=-1), "bad shape"),
    ("mq_kv_fork", FORK, dict(k=None), "caches"), ("mq_kv_fork", FORK, dict(bytes=4098), "multiples of 4"),
    ("mq_kv_fork", FORK, dict(pitch=2048), "overlapping"), ("mq_kv_fork", FORK, dict(ks=A), "both caches"),
    ("mq_kv_fork", FORK, dict(src=None), "src and dst"), ("mq_kv_fork", FORK, dict(work=None), "workspace"),
    ("mq_kv_free", FREE, dict(seqs=None), "sequences"), ("mq_kv_free", FREE, dict(lens=None), "lens"),
    ("mq_kv_compact", COMPACT, dict(live=None), "live"), ("mq_kv_compact", COMPACT, dict(work_bytes=0), "workspace"),
    ("mq_kv_compact", COMPACT, dict(table=None), "page_table"),
    ("mq_linear_w4a16", W4, dict(group=48), "group size"), ("mq_linear_w4a16", W4, dict(K=320, hblock=256), "convrot"),
    ("mq_linear_w4a16", W4, dict(K=96), "group size"), ("mq_linear_w4a16", W4, dict(hblock=32), "convrot"),
    ("mq_linear_w4a16", W4, dict(zero=1), "null operand"), ("mq_linear_w4a16", W4, dict(zero=3), "zero-point rule"),
    ("mq_linear_w4a16", W4, dict(zero=1, wz=A, ldwz=3), "ldwz"), ("mq_linear_w4a16", W4, dict(zero=2, wz=A, ldwz=7), "ldwz"),
    ("mq_linear_w4a16", W4, dict(ldx=516), "ldx"), ("mq_linear_w4a16", W4, dict(ldw=264), "ldw"),
    ("mq_linear_w4a16", W4, dict(ldws=7), "ldws"), ("mq_linear_w4a16", W4, dict(ldy=63), "ldy"),
    ("mq_linear_w4a16", W4, dict(x=A + 4), "16-byte"), ("mq_linear_w4a16", W4, dict(s_dtype=3), "scale type"),
    ("mq_linear_w4a16", W4, dict(y_dtype=4), "output type"), ("mq_linear_w4a16", W4, dict(x_dtype=3), "input type"),
]


@pytest.mark.parametrize("name,good,bad,message", REFUSED, ids=[f"{r[0]}-{'-'.join(r[2])}" for r in REFUSED])
def test_refused_before_launch(name, good, bad, message):
    _lib.load()
    args = list({**good, **bad}.values())
    with pytest.raises(ValueError, match=message):
        _lib.call(name, *args)
    slow = getattr(_lib.load(), name)
    assert slow(*args) == -1 and message in _lib.load().mq_last_error().decode()


def test_too_long_rows_are_unsupported():
    with pytest.raises(ck.MQError, match="32768"):
        _lib.call("mq_linear_w4a16", *{**W4, "K": 65536, "ldx": 65536, "ldw": 32768, "ldws": 1024}.values())


@pytest.mark.parametrize("name,good,empty", [("mq_kv_write", WRITE, dict(T=0, B=0)), ("mq_kv_write", WRITE, dict(pages=0)),
                                             ("mq_paged_attention", ATTN, dict(T=0, B=0)), ("mq_kv_grow", GROW, dict(n=0)),
                                             ("mq_kv_fork", FORK, dict(n=0)), ("mq_kv_free", FREE, dict(n=0)),
                                             ("mq_linear_w4a16", W4, dict(M=0)), ("mq_linear_w4a16", W4, dict(N=0))])
def test_empty_calls_do_nothing(name, good, empty):
    _lib.call(name, *{**good, **empty}.values())


@pytest.mark.parametrize("name", ["mq_kv_write", "mq_paged_attention", "mq_kv_grow", "mq_linear_w4a16"])
def test_the_fast_calls_take_what_ctypes_takes(name):
    """Pointers may be None and nothing else may; the scale is a number of any kind."""
    lib = _lib.load()
    good = {"mq_kv_write": dict(WRITE, T=0, B=0), "mq_paged_attention": dict(ATTN, T=0, B=0), "mq_kv_grow": dict(GROW, n=0),
            "mq_linear_w4a16": dict(W4, M=0)}[name]
    args = list(good.values())
    kinds = _lib._SIGNATURES[name][0]
    assert len(args) == len(kinds)
    for i, kind in enumerate(kinds):
        one = args[:i] + [None] + args[i + 1:]
        if kind is ctypes.c_void_p:
            assert _lib._entries[name](*one) == getattr(lib, name)(*one)
        else:
            with pytest.raises(TypeError):
                _lib._entries[name](*one)
    if name == "mq_paged_attention":
        for scale in (1, 0.25, True):
            assert _lib._entries[name](*{**good, "scale": scale}.values()) == 0
    with pytest.raises(TypeError, match="arguments"):
        _lib._entries[name](*args[:-1])


def test_host_tensors_are_refused():
    x, i = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    cache = torch.zeros((3, 4, 16, 64), dtype=torch.bfloat16)
    table = torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ck.paged_attention(x, cache, cache, table, i)
    with pytest.raises(ValueError, match="device tensor"):
        ck.kv_write(x, x, cache, cache, table, i)
    for call in (lambda: ck.kv_grow(table, i, i, [0], [1], 16), lambda: ck.kv_free(table, i, i, [0]),
                 lambda: ck.kv_fork(cache, cache, table, i, i, [0], [1]), lambda: ck.kv_compact(cache, cache, table, i)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    with pytest.raises(ValueError, match="GPU"):
        ck.w4a16_linear(torch.zeros(1, 64), torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 1)))


def test_w4a16_arguments():
    x, q, s = torch.zeros((1, 128)), torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 2))
    with pytest.raises(ValueError, match="qweight K"):
        ck.w4a16_linear(torch.zeros(1, 64), q, s)
    with pytest.raises(ValueError, match="group_size"):
        ck.w4a16_linear(x, q, s, group_size=16)
    with pytest.raises(ValueError, match="convrot_groupsize"):
        ck.w4a16_linear(x, q, s, convrot_groupsize=256)
    with pytest.raises(ValueError, match="8-bit"):
        ck.w4a16_linear(x, q.float(), s)


def test_plain_attention_is_softmax():
    """The oracle's loops against the textbook product on one contiguous sequence."""
    rng = np.random.default_rng(0)
    q, kv = rng.normal(size=(5, 2, 8)), rng.normal(size=(2, 3, 1, 4, 8))
    table = [[2, 0]]
    o, _, _ = serving.attention(q, kv[0], kv[1], table, [7], [0, 5], window=3, sinks=1)
    k, v = (np.concatenate([c[2, 0], c[0, 0]])[:7] for c in kv)
    for t in range(5):
        see = [j for j in range(t + 3) if j > t + 2 - 3 or j < 1]
        for h in range(2):
            p = np.exp(k[see] @ q[t, h] / 8 ** 0.5)
            assert np.allclose(o[t, h], p @ v[see] / p.sum())


def test_plain_pages_keep_what_sequences_hold():
    p = serving.Pages([[-1] * 4 for _ in range(4)], [0] * 4, [0] * 9, 4)
    assert p.grow([0, 1], [6, 9]) == 0 and p.table[:2] == [[0, 1, -1, -1], [2, 3, 4, -1]]
    assert p.fork([1, 0], [2, 3]) == 0 and p.moves == [(4, 5), (1, 6)] and p.refs[2:4] == [2, 2] and p.refs[0] == 2
    assert p.grow([2], [8]) == -1 and p.grow([2], [7]) == 0 and p.table[2] == [2, 3, 5, 7] and p.lens[2] == 16
    p.free([1])
    assert p.refs[4] == 0 and p.refs[2] == 1
    n = p.compact()
    assert sorted(x for r in p.table for x in r if x >= 0) and max(x for r in p.table for x in r) == n - 1
