"""The text decoder's cache in pages and 4 bits a value, on the GPU: what a decoder layer does with it in place of rows.

A `PagedCache` holds pages of keys and values for one layer, 4.25 bits a value (a bf16 scale for each 64 values of a head, and for each value
a sign and one of the numbers 0, .5, 1, 1.5, 2, 3, 4, 6). Sequences own pages of it, named by a page table (int32
[sequences, pages], a line's first k_len tokens in order); the table and the lengths lie on the device and may change
between calls, or between the replays of a graph:

    cache = PagedCache(n_pages, page_rows, num_kv_heads, head_dim)                                       # once a layer
    q = qk_norm_rotary_paged(q, k, v, q_norm, k_norm, positions, rotary, cache, page_table, k_len)       # new tokens into their pages
    out = paged_attention(q, cache, page_table, k_len, max_len=...)                                      # token by token
    k, v = unpack_paged(cache, page_table, k_len, k_start, k, v, max_len=...)                            # a prompt after a history:
    out = causal_attention(q, k, v, plan)                                                                # decoder_attn's

The conventions of `decoder_attn` hold: tensors [rows, heads, head_dim] in float32 or bfloat16 with any row and head strides of
whole 16 bytes, the current stream of the tensors' device, workspaces from torch's allocator with every call, no gradients.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

from . import capi
from .decoder_attn import (TextRotary, _device, _elsewhere, _heads_view, _like, _no_gradient, _qdtype, _read_on, _scale, _stream, _torch,
                           _word, _workspace, _written)


class PagedCache:
    """Pages of `page_rows` tokens (a power of two, 16 to 4096) for one layer's keys and values, in `data` (uint8; what a page
    holds is this library's own layout). Pages may be copied or moved as bytes: page p is data[p]."""

    def __init__(self, n_pages: int, page_rows: int, num_kv_heads: int, head_dim: int, device="cuda"):
        self.n_pages, self.page_rows = int(n_pages), int(page_rows)
        self.num_kv_heads, self.head_dim = int(num_kv_heads), int(head_dim)
        nb = C.c_size_t()
        capi.check(capi.load().qvl_paged_cache_size(self.n_pages, self.page_rows, self.num_kv_heads, self.head_dim, C.byref(nb)),
                   "qvl_paged_cache_size")
        self.page_bytes = nb.value // self.n_pages if self.n_pages else 0
        torch = _torch()
        self._data = torch.zeros((self.n_pages, self.page_bytes), dtype=torch.uint8, device=_device(device))

    @property
    def data(self):
        return self._data


def _pages(cache: PagedCache, page_table, k_len, like, heads: Optional[int] = None):
    """The cache, the page table and the sequences' lengths as the entries take them: (cache and table arguments, number of
    sequences, k_len's pointer)."""
    data = cache._data
    if data.device != like[1]:
        raise ValueError(f"the cache on {data.device}, q on {like[1]}")
    if data.shape != (cache.n_pages, cache.page_bytes) or not data.is_contiguous():
        raise ValueError(f"the cache's data {tuple(data.shape)} is not its {cache.n_pages} pages of {cache.page_bytes} bytes any more")
    if like[2] != cache.head_dim:
        raise ValueError(f"head_dim {like[2]}, the cache has {cache.head_dim}")
    if heads is not None and heads != cache.num_kv_heads:
        raise ValueError(f"{heads} key/value heads, the cache has {cache.num_kv_heads}")
    shape, stride = page_table.shape, page_table.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"page_table must be [sequences, pages] with a contiguous last axis, not {tuple(shape)}")
    int32 = _torch().int32
    if page_table.dtype != int32:
        raise TypeError(f"page_table is {page_table.dtype}, expected torch.int32")
    if page_table.device != like[1]:
        raise ValueError(f"page_table on {page_table.device}, q on {like[1]}")
    n = shape[0]
    # (data's address with every call: a copy of the cache has pages of its own)
    return ((data.data_ptr(), cache.n_pages, cache.page_rows, page_table.data_ptr(), shape[1], stride[0] if n > 1 else 0), n,
            _word(k_len, "k_len", like, int32, (n,)))


def _cu(cu_q, like, n_seqs: int, n_tokens: int):
    if cu_q is None:
        if n_tokens != n_seqs:
            raise ValueError(f"{n_tokens} tokens of {n_seqs} sequences without cu_q")
        return None
    return _word(cu_q, "cu_q", like, _torch().int32, (n_seqs + 1,))


def qk_norm_rotary_paged(q, k, v, q_norm, k_norm, positions, rotary: TextRotary, cache: PagedCache, page_table, k_len, *,
                         eps: float = 1e-6, cu_q=None, q_out=None):
    """`decoder_attn.qk_norm_rotary` with keys and values to pages: sequence i's new tokens (one, token i; or tokens
    cu_q[i]..cu_q[i+1], int32 [n + 1]) are the last of its k_len[i] (int32). Returns q; q_out, if given, takes it (it may be q
    itself). A token whose place is in no page is dropped, one of no sequence leaves its row of q_out as it is. A key is
    normalised, rotated and brought to 4 bits in float64: another order of a sum could move a code only where the quotient lies within some
    1e-15 of a border between two."""
    torch = _torch()
    like = _like(q)
    N, Hq, D = q.shape
    qv, kv = _heads_view(q, "q", like), _heads_view(k, "k", like)
    Hkv = k.shape[1]
    vv = _heads_view(v, "v", like, Hkv)
    if k.shape[0] != N or v.shape[0] != N:
        raise ValueError(f"q has {N} tokens, k {k.shape[0]}, v {v.shape[0]}")
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
    pages, n_seqs, lens = _pages(cache, page_table, k_len, like, Hkv)
    cu = _cu(cu_q, like, n_seqs, N)
    if q_out is None:
        q_out = q.new_empty((N, Hq, D))
    elif q_out.shape[0] != N:
        raise ValueError(f"q_out has {q_out.shape[0]} rows for {N} tokens")
    qo = _heads_view(q_out, "q_out", like, Hq, True)
    if _elsewhere(like[1]):
        with torch.cuda.device(like[1]):
            return qk_norm_rotary_paged(q, k, v, q_norm, k_norm, positions, rotary, cache, page_table, k_len, eps=eps, cu_q=cu_q,
                                        q_out=q_out)
    stream = _stream(like[1])
    if stream not in rotary._streams:
        _read_on(table, rotary._streams, stream)
    capi.check(capi.load().qvl_paged_append(
        stream, _qdtype(like[0]), *qv, *kv, *vv, qw, kw, float(eps), pos, pos_stride, table.data_ptr(), *pages, cu, n_seqs, lens, *qo,
        N, Hq, Hkv, D), "qvl_paged_append")
    _written()((q_out, cache.data))
    return q_out


def append_paged(k, v, cache: PagedCache, page_table, k_len, *, cu_q=None):
    """Keys and values [N, Hkv, D] of new tokens into their pages as they are (a prefill's, rotated already, or those of a cache of
    rows); the sequences' state as in `qk_norm_rotary_paged`. Values that `unpack_paged` gave in float32 come back bit
    for bit where a group's scale is 0, NaN or a normal number (2^-126 on) and six times it a float32: not for groups whose largest value is
    under 6 2^-126 or over 3.399e38, which may come back as other multiples, zeros or, from infinities at the top, NaN."""
    like = _like(k)
    N, Hkv, D = k.shape
    kv, vv = _heads_view(k, "k", like), _heads_view(v, "v", like, Hkv)
    if v.shape[0] != N:
        raise ValueError(f"k has {N} tokens, v {v.shape[0]}")
    pages, n_seqs, lens = _pages(cache, page_table, k_len, like, Hkv)
    cu = _cu(cu_q, like, n_seqs, N)
    if _elsewhere(like[1]):
        with _torch().cuda.device(like[1]):
            return append_paged(k, v, cache, page_table, k_len, cu_q=cu_q)
    capi.check(capi.load().qvl_paged_append(
        _stream(like[1]), _qdtype(like[0]), None, 0, 0, *kv, *vv, None, None, 0.0, None, 0, None, *pages, cu, n_seqs, lens, None, 0, 0,
        N, 0, Hkv, D), "qvl_paged_append")
    _written()((cache.data,))


def unpack_paged(cache: PagedCache, page_table, k_len, k_start, k, v, *, max_len: int, first=None):
    """The keys and values that pages stand for, as rows of k and v [R, Hkv, D]: tokens first[i] (int32; None: 0) to k_len[i] of
    sequence i, token t as row k_start[i] + t - first[i] (k_start int64; of a negative first the tokens before 0 are none), rounded to
    their dtype once. Rows outside [0, R) are dropped, tokens in no page are NaN.
    max_len, the most tokens of a sequence, only lays the launch out. Returns (k, v)."""
    torch = _torch()
    like = _like(k)
    R, Hkv, D = k.shape
    kv, vv = _heads_view(k, "k", like, None, True), _heads_view(v, "v", like, Hkv, True)
    if v.shape[0] != R:
        raise ValueError(f"k has {R} rows, v {v.shape[0]}")
    pages, n_seqs, lens = _pages(cache, page_table, k_len, like, Hkv)
    start = _word(k_start, "k_start", like, torch.int64, (n_seqs,))
    begin = None if first is None else _word(first, "first", like, torch.int32, (n_seqs,))
    if _elsewhere(like[1]):
        with torch.cuda.device(like[1]):
            return unpack_paged(cache, page_table, k_len, k_start, k, v, max_len=max_len, first=first)
    capi.check(capi.load().qvl_paged_unpack(
        _stream(like[1]), _qdtype(like[0]), *pages, n_seqs, begin, lens, int(max_len), start, *kv, *vv, R, Hkv, D), "qvl_paged_unpack")
    _written()((k, v))
    return k, v


@functools.lru_cache(maxsize=256)
def _paged_bytes(device_index, *sizes) -> int:
    """qvl_paged_attention_workspace_size: the same for the same sizes on the same (current) device."""
    nb = C.c_size_t()
    capi.check(capi.load().qvl_paged_attention_workspace_size(*sizes, C.byref(nb)), "qvl_paged_attention_workspace_size")
    return nb.value


def paged_attention(q, cache: PagedCache, page_table, k_len, *, max_len: int, cu_q=None, scale: Optional[float] = None, out=None):
    """`decoder_attn.decode_attention` over pages: sequence i's keys are its first k_len[i] (int32) tokens, its new tokens' own
    at their end. q [N, Hq, D] holds one token per sequence, or tokens cu_q[i]..cu_q[i+1] (int32 [n + 1]). max_len, the longest
    the launch is laid out for, only sets how far the keys are split over the GPU. `out` lies over no input."""
    like = _like(q)
    N, Hq, D = q.shape
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape:
        raise ValueError(f"out {tuple(out.shape)}, q {tuple(q.shape)}")
    qv, ov = _heads_view(q, "q", like), _heads_view(out, "out", like, Hq, True)
    pages, n_seqs, lens = _pages(cache, page_table, k_len, like)
    cu, max_len, Hkv = _cu(cu_q, like, n_seqs, N), int(max_len), cache.num_kv_heads
    if _elsewhere(like[1]):
        with _torch().cuda.device(like[1]):
            return paged_attention(q, cache, page_table, k_len, max_len=max_len, cu_q=cu_q, scale=scale, out=out)
    nb = _paged_bytes(like[1].index, N, n_seqs, max_len, Hq, Hkv, D)
    ws = _workspace(nb, q)
    capi.check(capi.load().qvl_paged_attention(
        _stream(like[1]), _qdtype(like[0]), *qv, *pages, cu, n_seqs, lens, max_len, _scale(scale, D), *ov, N, Hq, Hkv, D,
        None if ws is None else ws.data_ptr(), nb), "qvl_paged_attention")
    _written()((out,))
    return out
