"""What a text decoder layer computes between its qkv Dense and its output Dense, on the GPU.

After `decoder_io.inject_vision` a prompt's hidden rows go through the decoder's layers. In each of them, on torch device
tensors [rows, heads, head_dim] (any row and head strides of whole 16 bytes), float32 or bfloat16:

    rotary = TextRotary.from_spec(spec.text)                             # once
    plan = CausalPlan(q_lens, k_lens, k_starts, num_heads=..., ...)      # once per prefill, for all layers
    q, k_cache, v_cache = qk_norm_rotary(q, k, v, q_norm, k_norm, positions, rotary, k_cache=k_cache, v_cache=v_cache,
                                         rows=rows)
    out = causal_attention(q, k_cache, v_cache, plan)                    # the prompt
    out = decode_attention(q, k_cache, v_cache, k_start, k_len, max_len=...)       # then token by token
    out = prefix_attention(q, k_cache, v_cache, k_start, k_len, prefix_start, prefix_len, cu_groups, max_len=...,
                           max_prefix=...)                               # where sequences share an image's tokens

Everything runs on the tensors' device and its current stream; nothing synchronises. Workspaces come from torch's
allocator with every call, so calls on several streams and captured graphs share none. No operator has a gradient: a tensor
that requires one is refused while gradients are recorded, and one that carries a forward-mode tangent always.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Sequence

import numpy as np

from . import capi


@functools.lru_cache(maxsize=None)
def _torch():
    import torch
    return torch


@functools.lru_cache(maxsize=None)
def _forward_ad():
    import torch.autograd.forward_ad
    return torch.autograd.forward_ad


def _qdtype(dtype):
    torch = _torch()
    if dtype == torch.bfloat16:
        return capi.QVL_DTYPE_BF16
    if dtype == torch.float32:
        return capi.QVL_DTYPE_F32
    raise TypeError(f"unsupported dtype {dtype} (bfloat16 or float32)")


def _device(device):
    torch = _torch()
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"device {d}: the decoder operators run on the GPU")
    return torch.device("cuda", torch.cuda.current_device()) if d.index is None else d


def _no_gradient(t, what: str):
    """For a tensor that requires a gradient, or inside a forward-mode dual_level."""
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{what} requires a gradient: the decoder operators have none (call them under torch.no_grad())")
    if _forward_ad().unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} carries a tangent: the decoder operators have no forward-mode gradient")


def _heads_view(t, what: str, like, heads: Optional[int] = None, written: bool = False):
    """(pointer, row stride, head stride) of a [rows, heads, head_dim] tensor, checked against `like`: q's (dtype, device,
    head_dim), and whether a forward-mode dual_level is entered."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{what} must be [rows, heads, head_dim], not {tuple(shape)}")
    rows, n, dim = shape
    row, head, one = t.stride()
    if one != 1 and dim > 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    if t.dtype != like[0]:
        raise TypeError(f"{what} is {t.dtype}, q is {like[0]}")
    if t.device != like[1]:
        raise ValueError(f"{what} on {t.device}, q on {like[1]}")
    if dim != like[2]:
        raise ValueError(f"{what}: head_dim {dim}, q has {like[2]}")
    if heads is not None and n != heads:
        raise ValueError(f"{what}: {n} heads, expected {heads}")
    if t.requires_grad or like[3]:
        _no_gradient(t, what)
    # the stride of an axis of one entry is never used: torch may hold any value there
    if rows < 2:
        row = 0
    if n < 2:
        head = 0
    if written and row < head * n and rows > 0 and n > 0:   # (rows of whole, separate heads need no further look)
        inner, outer, count = (head, row, n) if n > 1 and (rows == 1 or head <= row) else (row, head, rows)
        if (n > 1 or rows > 1) and (inner < dim or (n > 1 and rows > 1 and outer < inner * (count - 1) + dim)):
            raise ValueError(f"{what}: its rows and heads lie over one another (strides {t.stride()})")
    elif written and (rows > 1 or n > 1) and (head < dim if n > 1 else row < dim):
        raise ValueError(f"{what}: its rows and heads lie over one another (strides {t.stride()})")
    return t.data_ptr(), row, head


def _like(q):
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"q must be [rows, heads, head_dim], not {tuple(shape)}")
    return q.dtype, q.device, shape[2], _forward_ad()._current_level >= 0


def _word(t, what: str, like, dtype, shape):
    """Pointer of a contiguous device tensor beside q."""
    if t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}, expected {dtype}")
    if t.device != like[1]:
        raise ValueError(f"{what} on {t.device}, q on {like[1]}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {shape}, not {tuple(t.shape)}")
    return t.data_ptr()


def _elsewhere(device) -> bool:
    """Whether the tensors lie on another device than the current one: the operator then calls itself with theirs current
    (a kernel goes to the current device)."""
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: the decoder operators run on the GPU")
    return device.index != _torch()._C._cuda_getDevice()


def _stream(device) -> int:
    return _torch()._C._cuda_getCurrentRawStream(device.index)   # current_stream(device).cuda_stream, 1.5 us cheaper


@functools.lru_cache(maxsize=None)
def _written():
    """Called with the tensors that a kernel wrote through pointers: autograd's check of what other operations saved looks at
    their versions."""
    return _torch()._C._increment_version                          # torch.autograd.graph.increment_version, for a tuple


def _streams_of(device) -> set:
    """The streams that torch's allocator knows a tensor made now to be used on: the current one."""
    return {_stream(device)}


def _read_on(t, streams: set, stream: int):
    """t, of an object that may go before the kernel that reads it has run, is read on `stream`, none of `streams`: its memory is
    not handed out again before that work is through."""
    t.record_stream(_torch().cuda.current_stream(t.device))
    streams.add(stream)


class TextRotary:
    """The rotation of `qk_norm_rotary`: frequencies theta^(-2j/head_dim), j < head_dim/2, each following the t, h or w
    position (`section`: how many follow which, one axis after the other or interleaved). Like a CausalPlan, it has to
    outlive the graphs that captured a call with it."""

    def __init__(self, head_dim: int, theta: float, section: Sequence[int], interleaved: bool = True, device="cuda"):
        torch = _torch()
        if len(section) != 3:
            raise ValueError(f"section {tuple(section)}: expected the counts of t, h and w")
        self.head_dim, self.theta = int(head_dim), float(theta)
        self.section, self.interleaved = tuple(int(s) for s in section), bool(interleaved)
        table = np.zeros((max(self.head_dim // 2, 0), 2), np.uint64)
        sec = (C.c_int32 * 3)(*self.section)
        capi.check(capi.load().qvl_text_rotary_table(self.head_dim, self.theta, sec, int(self.interleaved),
                                                     table.ctypes.data), "qvl_text_rotary_table")
        self.table = torch.from_numpy(table.view(np.int64)).to(_device(device))
        self._streams = _streams_of(self.table.device)

    @classmethod
    def from_spec(cls, text, device="cuda"):
        """The rotation of a TextBackboneSpec (model.py:67-81)."""
        if text.rope_scaling_factor not in (None, 1, 1.0):
            raise ValueError(f"rope_scaling factor {text.rope_scaling_factor} is not supported")
        return cls(text.head_dim, text.rope_theta, tuple(text.rope_section), text.mrope_interleaved, device)


def qk_norm_rotary(q, k, v, q_norm, k_norm, positions, rotary: TextRotary, *, eps: float = 1e-6, k_cache=None,
                   v_cache=None, rows=None, q_out=None):
    """Per-head RMSNorm of q [N, Hq, D] and k [N, Hkv, D] (weights q_norm, k_norm float32 [D]) and the rotation by
    `positions` (int32 [3, N] for t, h, w, or [N] for text), one pass. Returns (q, k, v): without a cache new tensors q
    and k and v itself; with k_cache, v_cache [R, Hkv, D] and rows (int64 [N]), token n's key and value go to row
    rows[n] of the caches, which are returned (a row outside [0, R) is dropped; rows should differ). q_out, if given,
    takes q (it may be q itself). Outputs lie over no other input."""
    torch = _torch()
    like = _like(q)
    N, Hq, D = q.shape
    qv = _heads_view(q, "q", like)
    kv = _heads_view(k, "k", like)
    Hkv = k.shape[1]
    if k.shape[0] != N or (v is not None and v.shape[0] != N):
        raise ValueError(f"q has {N} tokens, k {k.shape[0]}" + ("" if v is None else f", v {v.shape[0]}"))
    table = rotary.table
    if D != rotary.head_dim:
        raise ValueError(f"head_dim {D}, the rotation is made for {rotary.head_dim}")
    if table.device != like[1]:
        raise ValueError(f"the rotation on {table.device}, q on {q.device}")
    qw, kw = _word(q_norm, "q_norm", like, torch.float32, (D,)), _word(k_norm, "k_norm", like, torch.float32, (D,))
    if q_norm.requires_grad or k_norm.requires_grad or like[3]:
        _no_gradient(q_norm, "q_norm")
        _no_gradient(k_norm, "k_norm")
    if positions.dim() == 1:
        pos, pos_stride = _word(positions, "positions", like, torch.int32, (N,)), 0
    else:
        pos, pos_stride = _word(positions, "positions", like, torch.int32, (3, N)), N
    if q_out is None:
        q_out = q.new_empty((N, Hq, D))
    elif q_out.shape[0] != N:
        raise ValueError(f"q_out has {q_out.shape[0]} rows for {N} tokens")
    qo = _heads_view(q_out, "q_out", like, Hq, True)
    if (k_cache is None) != (v_cache is None) or (k_cache is None) != (rows is None):
        raise ValueError("k_cache, v_cache and rows come together")
    if k_cache is None:
        k_cache, out_rows, prow = q.new_empty((N, Hkv, D)), N, None
        vv = vo = (None, 0, 0)
    else:
        if v is None:
            raise ValueError("v_cache without v")
        vv = _heads_view(v, "v", like, Hkv)
        vo = _heads_view(v_cache, "v_cache", like, Hkv, True)
        out_rows, prow = k_cache.shape[0], _word(rows, "rows", like, torch.int64, (N,))
        if v_cache.shape[0] != out_rows:
            raise ValueError(f"k_cache has {out_rows} rows, v_cache {v_cache.shape[0]}")
        if out_rows == 0:
            raise ValueError("the caches have no rows")
    ko = _heads_view(k_cache, "k_cache", like, Hkv, True)
    if _elsewhere(like[1]):
        with torch.cuda.device(like[1]):
            return qk_norm_rotary(q, k, v, q_norm, k_norm, positions, rotary, eps=eps, k_cache=None if rows is None else k_cache,
                                  v_cache=v_cache, rows=rows, q_out=q_out)
    stream = _stream(like[1])
    if stream not in rotary._streams:
        _read_on(table, rotary._streams, stream)
    capi.check(capi.load().qvl_qk_norm_rotary(
        stream, _qdtype(like[0]), *qv, *kv, *vv, qw, kw, float(eps), pos, pos_stride, table.data_ptr(), prow, out_rows,
        *qo, *ko, *vo, N, Hq, Hkv, D), "qvl_qk_norm_rotary")
    _written()((q_out, k_cache) if v_cache is None else (q_out, k_cache, v_cache))
    return q_out, k_cache, v if v_cache is None else v_cache


class CausalPlan:
    """The work list of `causal_attention` for one packed prefill: sequence i brings q_lens[i] new tokens and has k_lens[i]
    keys (default q_lens), the new ones among them, in cache rows from k_starts[i] (default: one sequence after the other).
    Made on the host once and used by every layer, on any stream. A graph that captured a call reads the list at every
    replay: the plan has to outlive it. tile_rows: 0, or the kernel's tile height (128, or 256 in bfloat16)."""

    def __init__(self, q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None,
                 k_starts: Optional[Sequence[int]] = None, *, num_heads: int, num_kv_heads: int, head_dim: int, dtype,
                 device="cuda", tile_rows: int = 0):
        torch = _torch()
        device = _device(device)
        new = np.ascontiguousarray(q_lens, np.int64).reshape(-1)
        keys = new if k_lens is None else np.ascontiguousarray(k_lens, np.int64).reshape(-1)
        first = (np.concatenate([[0], np.cumsum(keys)[:-1]]).astype(np.int64) if k_starts is None and len(keys) else
                 np.ascontiguousarray([] if k_starts is None else k_starts, np.int64).reshape(-1))
        if not len(new) == len(keys) == len(first):
            raise ValueError(f"{len(new)} query lengths, {len(keys)} key lengths, {len(first)} starts")
        self.num_heads, self.num_kv_heads, self.head_dim = int(num_heads), int(num_kv_heads), int(head_dim)
        self.dtype, self.device = dtype, device
        self.n_tokens = int(new.sum())
        self.kv_rows = int((first + keys).max()) if len(keys) else 0     # rows the caches must have
        lib = capi.load()
        n_cus = torch.cuda.get_device_properties(device).multi_processor_count
        p64 = lambda a: a.ctypes.data_as(C.POINTER(C.c_int64))
        n, parts, joins, rows = C.c_int64(), C.c_int64(), C.c_int64(), C.c_int32(int(tile_rows))
        for entries in (4096, None):                # room for most lists; the call says how much one needs
            entries = entries or n.value + joins.value
            items = np.zeros((entries, capi.QVL_CAUSAL_ITEM_WORDS), np.int32)
            rc = lib.qvl_causal_worklist(len(new), p64(new), p64(keys), p64(first), self.num_heads, self.num_kv_heads,
                                         self.head_dim, _qdtype(dtype), n_cus, C.byref(rows),
                                         items.ctypes.data_as(C.POINTER(C.c_int32)), entries, C.byref(n), C.byref(parts), C.byref(joins))
            if rc == capi.QVL_OK or n.value + joins.value <= entries:
                break
        capi.check(rc, "qvl_causal_worklist")
        items = items[:max(n.value + joins.value, 1)]
        self.n_items, self.n_parts, self.n_joins, self.tile_rows = n.value, parts.value, joins.value, rows.value
        nb = C.c_size_t()
        capi.check(lib.qvl_causal_workspace_size(self.head_dim, self.tile_rows, self.n_parts, C.byref(nb)),
                   "qvl_causal_workspace_size")
        self.workspace_bytes = nb.value
        self.items = torch.from_numpy(items).to(device)
        self._streams = _streams_of(device)


def _attention_views(q, k, v, out, like):
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape:
        raise ValueError(f"out {tuple(out.shape)}, q {tuple(q.shape)}")
    qv, kv = _heads_view(q, "q", like), _heads_view(k, "k", like)
    vv = _heads_view(v, "v", like, k.shape[1])
    if k.shape[0] != v.shape[0]:
        raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
    return qv + kv + vv, _heads_view(out, "out", like, q.shape[1], True), out


def _workspace(nbytes: int, q):
    return q.new_empty(nbytes, dtype=_torch().uint8) if nbytes else None


def _scale(scale, head_dim: int) -> float:
    return float(head_dim) ** -0.5 if scale is None else float(scale)


def causal_attention(q, k, v, plan: CausalPlan, *, scale: Optional[float] = None, out=None):
    """softmax(scale q k^T) v of a packed prefill: q [N, Hq, D] holds the plan's new tokens one sequence after the other
    (rows past them are left as they are in `out`), k and v [R, Hkv, D] the caches (or the prompt's own keys and values).
    Token t of a sequence sees its keys up to itself; scale defaults to D^-0.5. `out`, here and below, lies over no input."""
    like = _like(q)
    views, ov, out = _attention_views(q, k, v, out, like)
    N, Hq, D = q.shape
    if (Hq, k.shape[1], D, like[0]) != (plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.dtype):
        raise ValueError(f"q of {Hq} heads, k of {k.shape[1]}, head_dim {D}, {q.dtype}: the plan is for "
                         f"{plan.num_heads}, {plan.num_kv_heads}, {plan.head_dim}, {plan.dtype}")
    if like[1] != plan.device:
        raise ValueError(f"q on {q.device}, the plan on {plan.device}")
    rows = k.shape[0]
    if N < plan.n_tokens or rows < plan.kv_rows:
        raise ValueError(f"{N} tokens and {rows} cache rows; the plan needs {plan.n_tokens} and {plan.kv_rows}")
    if _elsewhere(like[1]):
        with _torch().cuda.device(like[1]):
            return causal_attention(q, k, v, plan, scale=scale, out=out)
    ws = _workspace(plan.workspace_bytes, q)
    stream = _stream(like[1])
    if stream not in plan._streams:
        _read_on(plan.items, plan._streams, stream)
    capi.check(capi.load().qvl_causal_attention(
        stream, _qdtype(like[0]), *views, rows, plan.tile_rows, plan.items.data_ptr(), plan.n_items, plan.n_parts,
        plan.n_joins, _scale(scale, D), *ov, N, Hq, plan.num_kv_heads, D, None if ws is None else ws.data_ptr(),
        plan.workspace_bytes), "qvl_causal_attention")
    _written()((out,))
    return out


@functools.lru_cache(maxsize=256)
def _decode_bytes(device_index, *sizes) -> int:
    """qvl_decode_workspace_size: the same for the same sizes on the same (current) device."""
    nb = C.c_size_t()
    capi.check(capi.load().qvl_decode_workspace_size(*sizes, C.byref(nb)), "qvl_decode_workspace_size")
    return nb.value


def _decode(q, k, v, k_start, k_len, max_len, cu_q, groups, scale, out):
    torch = _torch()
    like = _like(q)
    views, ov, out = _attention_views(q, k, v, out, like)
    N, Hq, D = q.shape
    rows, Hkv = k.shape[0], k.shape[1]
    n_seqs = k_start.numel()
    ks = _word(k_start, "k_start", like, torch.int64, (n_seqs,))
    kl = _word(k_len, "k_len", like, torch.int32, (n_seqs,))
    cq = None if cu_q is None else _word(cu_q, "cu_q", like, torch.int32, (n_seqs + 1,))
    cg = ps = pl = None
    n_groups = max_prefix = 0
    if groups is not None:
        prefix_start, prefix_len, cu_groups, max_prefix = groups
        n_groups = prefix_start.numel()
        ps = _word(prefix_start, "prefix_start", like, torch.int64, (n_groups,))
        pl = _word(prefix_len, "prefix_len", like, torch.int32, (n_groups,))
        cg = _word(cu_groups, "cu_groups", like, torch.int32, (n_groups + 1,))
    dt, max_len, max_prefix = _qdtype(like[0]), int(max_len), int(max_prefix)
    if _elsewhere(like[1]):
        with torch.cuda.device(like[1]):
            return _decode(q, k, v, k_start, k_len, max_len, cu_q, groups, scale, out)
    nb = _decode_bytes(like[1].index, N, n_seqs, max_len, n_groups, max_prefix, Hq, Hkv, D, dt)
    ws = _workspace(nb, q)
    capi.check(capi.load().qvl_decode_attention(
        _stream(like[1]), dt, *views, rows, cq, n_seqs, ks, kl, max_len, cg, n_groups, ps, pl, max_prefix, _scale(scale, D), *ov, N,
        Hq, Hkv, D, None if ws is None else ws.data_ptr(), nb), "qvl_decode_attention")
    _written()((out,))
    return out


def decode_attention(q, k, v, k_start, k_len, *, max_len: int, cu_q=None, scale: Optional[float] = None, out=None):
    """Attention of new tokens over the caches k, v [R, Hkv, D]: sequence i's keys are the k_len[i] (int32) rows from
    k_start[i] (int64), its new tokens' own at their end. q [N, Hq, D] holds one token per sequence, or tokens
    cu_q[i]..cu_q[i+1] (int32 [n + 1]). The lengths are read on the device; max_len, the longest the launch is laid out
    for, only sets how far the keys are split over the GPU."""
    return _decode(q, k, v, k_start, k_len, max_len, cu_q, None, scale, out)


def prefix_attention(q, k, v, k_start, k_len, prefix_start, prefix_len, cu_groups, *, max_len: int, max_prefix: int,
                     cu_q=None, scale: Optional[float] = None, out=None):
    """`decode_attention` of sequences that share prefixes: every token of sequences cu_groups[g]..cu_groups[g+1] (int32
    [G + 1], never falling) also sees the prefix_len[g] (int32) cache rows from prefix_start[g]
    (int64), which lie in the cache once and are read once for the group. Sequences of no group have no prefix."""
    return _decode(q, k, v, k_start, k_len, max_len, cu_q, (prefix_start, prefix_len, cu_groups, max_prefix), scale, out)
