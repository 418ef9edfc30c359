"""What a step of token generation does between its linears and behind them, executed by libmq.so on the current HIP
stream: norms with the residual's addition, in floating point or as the int8 codes that the linears multiply, and
the choice of the next token. (No counterpart in the reference, whose models run in the programs that call it.)

    y, x = ck.rms_norm(delta, weight, x)                    # x + delta and its norm
    q, s, x = ck.rms_norm_quantize(delta, weight, x, convrot_groupsize=256)
    y = ck.gemm_w4_group(q, s, qdata, scales, zeros, None, n)
    token = ck.sample(logits, u, temperature=0.8, top_p=0.9)

Every call raises ValueError for tensors whose shapes, types, strides or devices do not fit; no call waits for the device or
reads from it.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .ops import CONVROT_GROUPSIZES, FLOAT_TYPES, _scratch

MOST_COLUMNS = 32768
_SAMPLE_WS: dict = {}


def _device_check(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise ValueError(f"kitchen_amd ops run on the GPU: {what} must be a device tensor")


def _rows(x: torch.Tensor, what: str, like: torch.Tensor | None = None) -> torch.Tensor:
    """[M, K] with contiguous rows behind each other (copied where they are not)."""
    if like is None:
        _device_check(x, what)
    if x.dtype not in FLOAT_TYPES:
        raise ValueError(f"{what} must be bfloat16, float16 or float32, got {x.dtype}")
    if like is not None and (x.shape != like.shape or x.dtype != like.dtype or x.device != like.device):
        raise ValueError(f"{what} must be {like.dtype} {list(like.shape)} on {like.device}, got {x.dtype} {list(x.shape)} on {x.device}")
    if x.dim() == 0:
        raise ValueError(f"{what} needs at least one dimension")
    k = x.shape[-1]
    if x.dim() != 2:
        # (rows of no values: how many is not -1's to say)
        x = x.reshape(-1 if k else math.prod(x.shape[:-1]), k)
    s0, s1 = x.stride()
    if (s1 != 1 and k > 1) or (x.shape[0] > 1 and s0 < k):
        x = x.contiguous()
    return x


def _new(x: torch.Tensor) -> torch.Tensor:
    """Contiguous, of x's shape, a plain tensor whatever x's class (empty_like keeps the class; a call with one argument is half a
    microsecond shorter)."""
    if type(x) is torch.Tensor and x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _norm_args(x, weight, residual, eps):
    x2 = _rows(x, "x")
    m, k = x2.shape
    if not 0 < k <= MOST_COLUMNS:
        raise ValueError(f"rows of 1 to {MOST_COLUMNS} values, got {k}")
    if weight is not None:
        if weight.shape != (k,) or weight.dtype not in FLOAT_TYPES or weight.device != x2.device:
            raise ValueError(f"weight must be floating-point [{k}] on {x2.device}, got {weight.dtype} {list(weight.shape)} on {weight.device}")
        weight = weight.contiguous()
    r2 = None if residual is None else _rows(residual, "residual", x)
    h = None if residual is None else _new(x)
    args = (x2.data_ptr(), _lib.DTYPE_CODE[x2.dtype], x2.stride(0), None if r2 is None else r2.data_ptr(),
            0 if r2 is None else r2.stride(0), None if weight is None else weight.data_ptr(),
            _lib.DT_BF16 if weight is None else _lib.DTYPE_CODE[weight.dtype], float(eps))
    # what is passed by address stays alive until the call is made
    return x2, m, k, h, args, (None if h is None else h.data_ptr(), k), (r2, weight)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """y = h * weight / sqrt(mean(h^2) + eps) over the last dimension of h = x (+ residual, rounded to x's type), computed in
    fp32 and rounded once to x's type. x: bfloat16, float16 or float32 of any strides, rows of up to 32768 values; weight: floating [K],
    None for ones. Returns y, or with a residual (y, h), both contiguous in x's shape."""
    x2, m, k, h, args, hargs, _keep = _norm_args(x, weight, residual, eps)
    y = _new(x)
    if m:
        _lib.call("mq_rms_norm", *args, *hargs, y.data_ptr(), k, m, k, _lib.stream_of_device(x2.device))
    return y if h is None else (y, h)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
                      convrot_groupsize: int | None = None):
    """rms_norm's y, not rounded in between, as rotate_quantize's int8 codes: rotated by H per block of convrot_groupsize (None:
    not), scale = max(absmax / 127, 1e-10) per row, codes rne(y / scale). Returns (q int8 [M, K], scale float32 [M]),
    and with a residual h in x's shape behind them. A row with an infinity or NaN gets codes 0 and scale NaN."""
    if convrot_groupsize and convrot_groupsize not in CONVROT_GROUPSIZES:
        raise ValueError(f"convrot_groupsize must be one of {CONVROT_GROUPSIZES} or None, got {convrot_groupsize}")
    x2, m, k, h, args, hargs, _keep = _norm_args(x, weight, residual, eps)
    if convrot_groupsize and k % convrot_groupsize:
        raise ValueError(f"Input K={k} is not divisible by convrot_groupsize={convrot_groupsize}")
    q = torch.empty((m, k), dtype=torch.int8, device=x2.device)
    s = torch.empty((m,), dtype=torch.float32, device=x2.device)
    if m:
        _lib.call("mq_rms_norm_quant", *args, int(convrot_groupsize or 0), *hargs, q.data_ptr(), k, s.data_ptr(), m, k,
                  _lib.stream_of_device(x2.device))
    return (q, s) if h is None else (q, s, h)


def _setting(value, name: str, rows: int, dtype, device):
    """(pointer or None, value) of a setting: a number for all rows, or a tensor [rows]."""
    if not isinstance(value, torch.Tensor):
        return None, value, None
    if value.shape != (rows,) or value.device != device:
        raise ValueError(f"{name} must be a number or [{rows}] on {device}, got {list(value.shape)} on {value.device}")
    if (value.dtype == dtype) if dtype is torch.int32 else value.is_floating_point():
        value = value.to(dtype).contiguous()
    elif dtype is torch.int32 and value.dtype in (torch.int64, torch.int16, torch.uint8, torch.int8):
        # (the bounds are no numbers of the smaller types)
        value = (value.clamp(-1, (1 << 31) - 1) if value.dtype is torch.int64 else value).to(dtype).contiguous()
    else:
        raise ValueError(f"{name} must be {'whole numbers' if dtype is torch.int32 else 'floating-point'}, got {value.dtype}")
    return value.data_ptr(), 0, value


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """The next token of every row of logits [rows, V] (bfloat16, float16 or float32, V <= 2^24) for its random number u (float32
    [rows], in [0, 1)): int64 [rows].

    Weights are exp((l - max l) / temperature). In the order of l (descending, ties by index) the first top_k are kept (0: all), of
    those the shortest leading part whose weight reaches top_p of theirs (>= 1: all), of those the ones of weight >= min_p; the
    token is the first, in the order of its number, whose kept weight up to it exceeds u times all kept weight. temperature 0: the first
    largest logit. Each setting is a number or a tensor [rows]. Logits that are NaN count as -infinity; where +infinities
    are, only they have weight; a row of -infinities gives -1. The same inputs always give the same tokens."""
    _device_check(logits, "logits")
    if logits.dim() != 2 or logits.dtype not in FLOAT_TYPES:
        raise ValueError(f"logits must be bfloat16, float16 or float32 [rows, V], got {logits.dtype} {list(logits.shape)}")
    rows, vocab = logits.shape
    if not 0 < vocab <= 1 << 24:
        raise ValueError(f"rows of 1 to {1 << 24} logits, got {vocab}")
    dev = logits.device
    if u.shape != (rows,) or u.dtype != torch.float32 or u.device != dev:
        raise ValueError(f"u must be float32 [{rows}] on {dev}, got {u.dtype} {list(u.shape)} on {u.device}")
    x, u = _rows(logits, "logits"), u.contiguous()
    t = _setting(temperature, "temperature", rows, torch.float32, dev)
    k = _setting(top_k, "top_k", rows, torch.int32, dev)
    p = _setting(top_p, "top_p", rows, torch.float32, dev)
    least = _setting(min_p, "min_p", rows, torch.float32, dev)
    token = torch.empty(rows, dtype=torch.int64, device=dev)
    if rows:
        stream, key = _lib.stream_of_device(dev), (dev.index, rows, vocab)
        nbytes = _SAMPLE_WS.get(key)
        if nbytes is None:
            with torch.cuda.device(dev):
                nbytes = int(_lib.load().mq_sample_workspace_bytes(rows, vocab))
            if len(_SAMPLE_WS) > 4096:
                _SAMPLE_WS.clear()
            _SAMPLE_WS[key] = nbytes
        work = _scratch(nbytes, dev, stream) if nbytes else None
        _lib.call("mq_sample", x.data_ptr(), _lib.DTYPE_CODE[x.dtype], x.stride(0), rows, vocab, u.data_ptr(), t[0], float(t[1]),
                  k[0], min(max(int(k[1]), -1), 1 << 24), p[0], float(p[1]), least[0], float(least[1]), token.data_ptr(),
                  None if work is None else work.data_ptr(), nbytes, stream)
    return token
