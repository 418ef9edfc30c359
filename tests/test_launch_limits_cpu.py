"""Calls whose one launch would have more threads than the runtime counts (2^32: it leaves workgroups out without an error) are
refused before it. CPU only: nothing is launched."""
import pytest

from kitchen_amd import _lib
from test_serving_cpu import A, WRITE

QUANTIZE = dict(w=A, dtype=0, N=3, K=64, ldw=64, hblock=0, format=_lib.WFMT_I8_ROW, q=A, ldq=64, scale=A, ld_scale=0, zero=None,
                ld_zero=0, stream=None)
REFUSED = [("mq_kv_write", WRITE, dict(T=1 << 28, B=1 << 28, H=1), "too many rows"),                 # 16 threads a row
           ("mq_kv_write", WRITE, dict(T=1 << 26, B=1 << 26, H=4), "too many rows"),
           ("mq_kv_write", WRITE, dict(T=(1 << 30) + 1, B=(1 << 30) + 1, H=4, D=8), "too many rows"),
           ("mq_kv_write", WRITE, dict(T=(1 << 31) - 1, B=(1 << 31) - 1, H=(1 << 31) - 1), "too many rows"),
           ("mq_quantize_weight", QUANTIZE, dict(N=1 << 24), "N too large"),
           ("mq_quantize_weight", QUANTIZE, dict(N=1 << 24, format=_lib.WFMT_I4_ROW), "N too large")]


@pytest.mark.parametrize("name,good,bad,message", REFUSED)
def test_refused_before_launch(name, good, bad, message):
    args = list({**good, **bad}.values())
    with pytest.raises(ValueError, match=message):
        _lib.call(name, *args)
