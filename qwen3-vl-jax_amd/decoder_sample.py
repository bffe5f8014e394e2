"""The next token of rows of logits, on the GPU.

    tokens = sample_tokens(logits, u, temperature=0.7, top_k=20, top_p=0.8)          # [rows, vocab], one random number a row

Settings are numbers for all rows, or device tensors with one value a row, which a captured graph reads at every replay. What a
row gives depends on its logits, its settings and its random number alone, bit for bit.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

from . import capi
from .decoder_attn import _elsewhere, _forward_ad, _no_gradient, _qdtype, _stream, _torch, _workspace, _written


def _setting(value, what: str, rows: int, device, dtype, low, high):
    """(pointer, number) of a setting as the entry takes it."""
    torch = _torch()
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"{what} is {value.dtype}, expected {dtype}")
        if value.device != device:
            raise ValueError(f"{what} on {value.device}, logits on {device}")
        if value.shape != (rows,) or not value.is_contiguous():
            raise ValueError(f"{what} must be a number or contiguous ({rows},), not {tuple(value.shape)}")
        return value.data_ptr(), 0
    if dtype == torch.int32:
        if value != int(value) or not low <= value <= high:
            raise ValueError(f"{what} {value}: a whole number from {low} to {high}")
        return None, int(value)
    value = float(value)
    if not low <= value <= high or not math.isfinite(value):
        raise ValueError(f"{what} {value}: a number from {low:g}" + (f" to {high:g}" if math.isfinite(high) else ""))
    return None, value


@functools.lru_cache(maxsize=256)
def _sample_bytes(rows: int) -> int:
    nb = C.c_size_t()
    capi.check(capi.load().qvl_sample_workspace_size(rows, C.byref(nb)), "qvl_sample_workspace_size")
    return nb.value


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """The next token (int64 [B]) of each row of logits [B, V] (float32 or bfloat16, contiguous rows, V up to 2^18), by its random
    number u [B] (float32, uniform in [0, 1); others, and NaN, count as 0 or as just below 1). With z = (x - max x) / temperature a
    token weighs e^z, as a whole number of 2^-44. In the order of falling logits (equal ones: rising index) the first top_k are kept
    (0: all), of them those before which less than top_p of their sum lies (1: all), of them those of at least min_p times the largest
    weight (0: all). The token is the first whose sum of kept weights up to it, by index, is over u times their whole sum.
    Temperature 0: the largest logit, of the lowest index. Tokens of -infinity are never chosen; a row of them alone, or with a NaN or
    +infinity, gives -1. Each setting is a number, or a tensor [B] beside the logits (float32; top_k int32)."""
    torch = _torch()
    if len(logits.shape) != 2:
        raise ValueError(f"logits must be [rows, vocab], not {tuple(logits.shape)}")
    B, V = logits.shape
    dt, device = _qdtype(logits.dtype), logits.device
    if logits.stride(1) != 1 and V > 1:
        raise ValueError("logits: the last axis must be contiguous")
    if logits.requires_grad or _forward_ad()._current_level >= 0:
        _no_gradient(logits, "logits")
    for t, what, want in ((u, "u", torch.float32),) + (() if out is None else ((out, "out", torch.int64),)):
        if t.dtype != want:
            raise TypeError(f"{what} is {t.dtype}, expected {want}")
        if t.device != device:
            raise ValueError(f"{what} on {t.device}, logits on {device}")
        if t.shape != (B,) or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous ({B},), not {tuple(t.shape)}")
    settings = (*_setting(temperature, "temperature", B, device, torch.float32, 0.0, math.inf),
                *_setting(top_k, "top_k", B, device, torch.int32, 0, 2 ** 31 - 1),
                *_setting(top_p, "top_p", B, device, torch.float32, 0.0, 1.0),
                *_setting(min_p, "min_p", B, device, torch.float32, 0.0, 1.0))
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=device)
    if _elsewhere(device):
        with torch.cuda.device(device):
            return sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, out=out)
    nb = _sample_bytes(B)
    ws = _workspace(nb, logits)
    capi.check(capi.load().qvl_sample_tokens(_stream(device), dt, logits.data_ptr(), logits.stride(0) if B > 1 else 0, B, V,
                                             u.data_ptr(), *settings, out.data_ptr(), None if ws is None else ws.data_ptr(), nb),
               "qvl_sample_tokens")
    _written()((out,))
    return out
