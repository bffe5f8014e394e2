"""The paged cache and the choice of tokens without a GPU: what the entries and the host layer refuse, and what they tell the streams
and autograd. (Nothing is launched.)"""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

BF, F32 = torch.bfloat16, torch.float32
P = 1 << 20                                      # stands for an aligned pointer; nothing reads it
VIEW = (P, 1024, 128)


@pytest.fixture()
def lib(pkg):
    return pkg.capi.load()


@pytest.fixture(scope="module")
def codes(pkg):
    """The error codes by their names in the header."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "qvl_vision.h").read_text()
    return {k: int(v) for k, v in re.findall(r"#define (QVL_ERR_[A-Z_]+) \((-\d+)\)", text)}


@pytest.mark.parametrize("pages,rows,heads,dim,want", [
    (3, 64, 8, 128, 3 * 8 * 4 * 2176), (1, 16, 1, 64, 1088), (7, 4096, 3, 64, 7 * 3 * 256 * 1088), (0, 16, 2, 128, 0)])
def test_cache_sizes(lib, pages, rows, heads, dim, want):
    nb = C.c_size_t(1)
    assert lib.qvl_paged_cache_size(pages, rows, heads, dim, C.byref(nb)) == 0 and nb.value == want


@pytest.mark.parametrize("pages,rows,heads,dim,name", [
    (1, 8, 1, 64, "UNSUPPORTED"), (1, 48, 1, 64, "UNSUPPORTED"), (1, 8192, 1, 64, "UNSUPPORTED"), (1, 0, 1, 64, "UNSUPPORTED"),
    (1, 16, 1, 96, "UNSUPPORTED"), (-1, 16, 1, 64, "INVALID_ARG"), (1, 16, 0, 64, "INVALID_ARG"), (1 << 31, 16, 1, 64, "UNSUPPORTED"),
    (1, 16, 4097, 64, "UNSUPPORTED")])
def test_cache_sizes_refused(lib, codes, pages, rows, heads, dim, name):
    nb = C.c_size_t()
    assert lib.qvl_paged_cache_size(pages, rows, heads, dim, C.byref(nb)) == codes["QVL_ERR_" + name]
    assert lib.qvl_paged_cache_size(1, 16, 1, 64, None) == codes["QVL_ERR_INVALID_ARG"]


def append(lib, **kw):
    a = dict(dtype=1, q=VIEW, k=VIEW, v=VIEW, qn=P, kn=P, eps=1e-6, pos=P, stride=0, table=P, cache=P, pages=4, rows=16, pt=P, width=2,
             pts=2, cu=P, n=2, len=P, out=VIEW, N=3, hq=8, hkv=2, D=128)
    a.update(kw)
    return lib.qvl_paged_append(None, a["dtype"], *a["q"], *a["k"], *a["v"], a["qn"], a["kn"], a["eps"], a["pos"], a["stride"], a["table"],
                                a["cache"], a["pages"], a["rows"], a["pt"], a["width"], a["pts"], a["cu"], a["n"], a["len"], *a["out"], a["N"],
                                a["hq"], a["hkv"], a["D"])


BAD_PAGES = [(dict(D=72), "UNSUPPORTED"), (dict(rows=24), "UNSUPPORTED"), (dict(pages=-1), "INVALID_ARG"), (dict(cache=None), "INVALID_ARG"),
             (dict(pt=None), "INVALID_ARG"), (dict(cache=P + 32), "MISALIGNED"), (dict(pt=P + 2), "MISALIGNED"), (dict(pts=-1), "INVALID_ARG"),
             (dict(n=65536), "UNSUPPORTED"), (dict(n=-1), "INVALID_ARG"), (dict(len=None), "INVALID_ARG"), (dict(len=P + 2), "MISALIGNED"),
             (dict(dtype=7), "UNSUPPORTED"), (dict(hkv=0), "INVALID_ARG")]


@pytest.mark.parametrize("kw,name", BAD_PAGES + [
    (dict(N=-1), "INVALID_ARG"), (dict(N=1 << 30), "UNSUPPORTED"), (dict(cu=None), "INVALID_ARG"), (dict(k=(None, 1024, 128)), "INVALID_ARG"),
    (dict(v=(None, 1024, 128)), "INVALID_ARG"), (dict(out=(None, 1024, 128)), "INVALID_ARG"), (dict(qn=None), "INVALID_ARG"),
    (dict(kn=None), "INVALID_ARG"), (dict(pos=None), "INVALID_ARG"), (dict(table=None), "INVALID_ARG"), (dict(table=P + 4), "MISALIGNED"),
    (dict(q=(P + 8, 1024, 128)), "MISALIGNED"), (dict(k=(P, 1028, 128)), "MISALIGNED"), (dict(v=(P, 1024, -8)), "INVALID_ARG"),
    (dict(hq=0), "INVALID_ARG"), (dict(hq=5000), "UNSUPPORTED"), (dict(eps=float("nan")), "INVALID_ARG"), (dict(eps=-1.0), "INVALID_ARG"),
    (dict(stride=-1), "INVALID_ARG"), (dict(cu=P + 1), "MISALIGNED")])
def test_append_refused(lib, codes, kw, name):
    assert append(lib, **kw) == codes["QVL_ERR_" + name], lib.qvl_last_error()


def test_append_of_nothing(lib):
    assert append(lib, N=0) == 0 and append(lib, n=0) == 0 and append(lib, N=0, n=0, cu=None, len=None) == 0


def unpack(lib, **kw):
    a = dict(dtype=1, cache=P, pages=4, rows=16, pt=P, width=2, pts=2, n=2, first=None, len=P, max_len=5, start=P, k=VIEW, v=VIEW, R=9, hkv=2,
             D=128)
    a.update(kw)
    return lib.qvl_paged_unpack(None, a["dtype"], a["cache"], a["pages"], a["rows"], a["pt"], a["width"], a["pts"], a["n"], a["first"], a["len"],
                                a["max_len"], a["start"], *a["k"], *a["v"], a["R"], a["hkv"], a["D"])


@pytest.mark.parametrize("kw,name", BAD_PAGES + [
    (dict(max_len=-1), "INVALID_ARG"), (dict(R=-1), "INVALID_ARG"), (dict(start=None), "INVALID_ARG"), (dict(start=P + 4), "MISALIGNED"),
    (dict(first=P + 1), "MISALIGNED"), (dict(k=(None, 0, 0)), "INVALID_ARG"), (dict(v=(P, 1025, 128)), "MISALIGNED"),
    (dict(max_len=1 << 30), "UNSUPPORTED")])
def test_unpack_refused(lib, codes, kw, name):
    assert unpack(lib, **kw) == codes["QVL_ERR_" + name], lib.qvl_last_error()
    assert unpack(lib, n=0) == 0 and unpack(lib, R=0) == 0


def attend(lib, **kw):
    a = dict(dtype=1, q=VIEW, cache=P, pages=4, rows=16, pt=P, width=2, pts=2, cu=P, n=2, len=P, max_len=5, scale=0.1, out=VIEW, N=3, hq=8, hkv=2,
             D=128, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.qvl_paged_attention(None, a["dtype"], *a["q"], a["cache"], a["pages"], a["rows"], a["pt"], a["width"], a["pts"], a["cu"], a["n"],
                                   a["len"], a["max_len"], a["scale"], *a["out"], a["N"], a["hq"], a["hkv"], a["D"], a["ws"], a["bytes"])


@pytest.mark.parametrize("kw,name", [c for c in BAD_PAGES if "len" not in c[0]] + [
    (dict(hq=7), "INVALID_ARG"), (dict(hq=8192), "UNSUPPORTED"), (dict(N=-1), "INVALID_ARG"), (dict(N=1 << 29), "UNSUPPORTED"),
    (dict(scale=0.0), "INVALID_ARG"), (dict(scale=float("inf")), "INVALID_ARG"), (dict(scale=float("nan")), "INVALID_ARG"),
    (dict(q=(None, 1024, 128)), "INVALID_ARG"), (dict(out=(P + 4, 1024, 128)), "MISALIGNED"), (dict(q=(P, 1024, 100)), "MISALIGNED"),
    (dict(max_len=-1), "INVALID_ARG"), (dict(max_len=1 << 31), "UNSUPPORTED")])
def test_attention_refused(lib, codes, kw, name):
    assert attend(lib, **kw) == codes["QVL_ERR_" + name], lib.qvl_last_error()


def sample(lib, **kw):
    a = dict(dtype=0, x=P, stride=1000, rows=3, vocab=1000, u=P, t=None, k=None, p=None, m=None, out=P, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.qvl_sample_tokens(None, a["dtype"], a["x"], a["stride"], a["rows"], a["vocab"], a["u"], a["t"], 1.0, a["k"], 0, a["p"], 1.0, a["m"],
                                 0.0, a["out"], a["ws"], a["bytes"])


@pytest.mark.parametrize("kw,name", [
    (dict(dtype=3), "UNSUPPORTED"), (dict(vocab=0), "INVALID_ARG"), (dict(vocab=(1 << 18) + 1), "UNSUPPORTED"), (dict(rows=-1), "INVALID_ARG"),
    (dict(stride=-1), "INVALID_ARG"), (dict(x=None), "INVALID_ARG"), (dict(u=None), "INVALID_ARG"), (dict(out=None), "INVALID_ARG"),
    (dict(x=P + 2), "MISALIGNED"), (dict(out=P + 4), "MISALIGNED"), (dict(u=P + 2), "MISALIGNED"), (dict(t=P + 1), "MISALIGNED"),
    (dict(ws=None), "WORKSPACE"), (dict(bytes=100), "WORKSPACE"), (dict(ws=P + 8), "MISALIGNED")])
def test_sample_refused(lib, codes, kw, name):
    assert sample(lib, **kw) == codes["QVL_ERR_" + name], lib.qvl_last_error()
    assert sample(lib, rows=0) == 0


# ---------------------------------------------------------------------------------------------
# the host layer, on host tensors, nothing launched
# ---------------------------------------------------------------------------------------------
@pytest.fixture()
def ops(pkg, monkeypatch):
    """decoder_cache with a library that accepts all and tells what it was called with."""
    ops, calls = pkg.decoder_cache, []
    fake = type("Lib", (), {"__getattr__": lambda self, name: lambda *a: calls.append((name, a)) or 0})()
    for m in (ops, pkg.decoder_sample):
        monkeypatch.setattr(m, "_elsewhere", lambda device: False)
        monkeypatch.setattr(m, "_stream", lambda device: 7)
    monkeypatch.setattr(ops, "_paged_bytes", lambda *a: 64)
    monkeypatch.setattr(pkg.decoder_sample, "_sample_bytes", lambda *a: 64)
    monkeypatch.setattr(pkg.capi, "load", lambda: fake)
    ops.calls = calls
    return ops


def cache_of(ops, pages=4, rows=16, heads=2, dim=64):
    c = ops.PagedCache.__new__(ops.PagedCache)
    c.n_pages, c.page_rows, c.num_kv_heads, c.head_dim, c.page_bytes = pages, rows, heads, dim, heads * rows // 16 * 1088
    c._data = torch.zeros(pages, c.page_bytes, dtype=torch.uint8)
    c._where, c._args = c._data.device, (c._data.data_ptr(), pages, rows)
    return c


def rotary_of(pkg, dim=64):
    rot = pkg.decoder_attn.TextRotary.__new__(pkg.decoder_attn.TextRotary)
    rot.head_dim, rot.table, rot._streams = dim, torch.zeros(dim // 2, 2, dtype=torch.int64), {7}
    return rot


def state(n=3, width=2):
    return torch.zeros(n, width, dtype=torch.int32), torch.ones(n, dtype=torch.int32)


def test_cache_needs_a_gpu(pkg):
    with pytest.raises(ValueError, match="GPU"):
        pkg.decoder_cache.PagedCache(2, 16, 2, 64, device="cpu")
    with pytest.raises(pkg.capi.QVLError, match="power of two"):
        pkg.decoder_cache.PagedCache(2, 20, 2, 64)


def test_calls_on_host_tensors_are_refused(pkg):
    ops = pkg.decoder_cache
    c, (table, lens) = cache_of(ops), state()
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    for call in (lambda: ops.paged_attention(q, c, table, lens, max_len=1), lambda: ops.append_paged(k, k.clone(), c, table, lens),
                 lambda: ops.unpack_paged(c, table, lens, torch.zeros(3, dtype=torch.int64), k, k.clone(), max_len=1),
                 lambda: pkg.decoder_sample.sample_tokens(torch.zeros(2, 9), torch.zeros(2))):
        with pytest.raises(ValueError, match="run on the GPU"):
            call()


def test_what_was_written_counts_as_changed(ops, pkg):
    c, (table, lens) = cache_of(ops), state()
    q, k, w = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.ones(64)
    v0 = c.data._version
    out = torch.zeros(3, 4, 64)
    ops.qk_norm_rotary_paged(q, k, k, w, w, torch.zeros(3, dtype=torch.int32), rotary_of(pkg), c, table, lens, q_out=out)
    assert c.data._version > v0 and out._version > 0
    v0 = c.data._version
    ops.append_paged(k, k, c, table, lens)
    assert c.data._version > v0
    a, b = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64)
    ops.unpack_paged(c, table, lens, torch.zeros(3, dtype=torch.int64), a, b, max_len=1)
    assert a._version > 0 and b._version > 0
    tokens = torch.zeros(2, dtype=torch.int64)
    pkg.decoder_sample.sample_tokens(torch.zeros(2, 9), torch.zeros(2), out=tokens)
    assert tokens._version > 0


def test_rotations_are_recorded_on_the_streams_that_read_them(ops, pkg, monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_read_on", lambda t, streams, stream: seen.append(stream) or streams.add(stream))
    c, (table, lens), rot = cache_of(ops), state(), rotary_of(pkg)
    rot._streams = {1}
    q, k, w = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.ones(64)
    for _ in range(2):
        ops.qk_norm_rotary_paged(q, k, k, w, w, torch.zeros(3, dtype=torch.int32), rot, c, table, lens)
    assert seen == [7]


def test_host_layer_refusals(ops, pkg):
    c, (table, lens), rot = cache_of(ops), state(), rotary_of(pkg)
    q, k, w, pos = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.ones(64), torch.zeros(3, dtype=torch.int32)
    start = torch.zeros(3, dtype=torch.int64)
    attend = lambda q=q, c=c, table=table, lens=lens, **kw: ops.paged_attention(q, c, table, lens, **{"max_len": 1, **kw})
    append = lambda q=q, k=k, v=k, qn=w, pos=pos, rot=rot, c=c, table=table, lens=lens, **kw: ops.qk_norm_rotary_paged(
        q, k, v, qn, w, pos, rot, c, table, lens, **kw)
    store = lambda k=k, v=k, **kw: ops.append_paged(k, v, c, table, lens, **kw)
    unpack = lambda k=k, v=k, lens=lens, start=start, **kw: ops.unpack_paged(c, table, lens, start, k, v, max_len=1, **kw)
    attend(), append(), store(), unpack(v=k.clone())
    grad = lambda t: t.clone().requires_grad_()
    for call, error in [
            (lambda: attend(q=torch.zeros(3, 256)), ValueError), (lambda: attend(q=q.to(torch.float16)), TypeError),
            (lambda: attend(q=torch.zeros(3, 4, 128)), ValueError), (lambda: attend(q=grad(q)), ValueError),
            (lambda: attend(table=table.long()), TypeError), (lambda: attend(table=table[0]), ValueError),
            (lambda: attend(table=table.t().contiguous().t()), ValueError), (lambda: attend(lens=lens.long()), TypeError),
            (lambda: attend(lens=lens[:2]), ValueError), (lambda: attend(q=q[:2]), ValueError),
            (lambda: attend(cu_q=torch.zeros(3, dtype=torch.int32)), ValueError), (lambda: attend(out=q[:2]), ValueError),
            (lambda: attend(out=torch.zeros(3, 1, 64).expand(3, 4, 64)), ValueError), (lambda: attend(out=grad(q)), ValueError),
            (lambda: append(k=k[:2]), ValueError), (lambda: append(k=torch.zeros(3, 1, 64), v=torch.zeros(3, 1, 64)), ValueError),
            (lambda: append(v=torch.zeros(3, 1, 64)), ValueError), (lambda: append(qn=w.double()), TypeError), (lambda: append(qn=grad(w)), ValueError),
            (lambda: append(pos=pos.long()), TypeError), (lambda: append(pos=pos[:2]), ValueError), (lambda: append(rot=rotary_of(pkg, 128)), ValueError),
            (lambda: append(c=cache_of(ops, dim=128)), ValueError), (lambda: append(q_out=q[:2]), ValueError), (lambda: append(k=grad(k)), ValueError),
            (lambda: append(v=k.bfloat16()), TypeError), (lambda: store(v=k[:1]), ValueError), (lambda: store(k=grad(k)), ValueError),
            (lambda: unpack(v=k[:1]), ValueError), (lambda: unpack(k=torch.zeros(1, 2, 64).expand(3, 2, 64), v=k.clone()), ValueError),
            (lambda: unpack(v=k.clone(), start=start.int()), TypeError), (lambda: unpack(v=k.clone(), first=start), TypeError),
            (lambda: unpack(k=grad(k), v=k.clone()), ValueError)]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        attend(q=grad(q))


def test_sample_host_refusals(ops, pkg):
    s = pkg.decoder_sample.sample_tokens
    x, u = torch.zeros(2, 9), torch.zeros(2)
    s(x, u, temperature=0.0, top_k=3, top_p=0.5, min_p=0.1)
    per = dict(temperature=torch.ones(2), top_k=torch.ones(2, dtype=torch.int32), top_p=torch.ones(2), min_p=torch.zeros(2))
    s(x, u, **per)
    name, args = ops.calls[-1]
    assert name == "qvl_sample_tokens" and args[7] == per["temperature"].data_ptr() and args[9] == per["top_k"].data_ptr()
    for call, error in [
            (lambda: s(x[0], u), ValueError), (lambda: s(x.double(), u), TypeError), (lambda: s(x.t(), torch.zeros(9)), ValueError),
            (lambda: s(x, u.double()), TypeError), (lambda: s(x, u[:1]), ValueError), (lambda: s(x.clone().requires_grad_(), u), ValueError),
            (lambda: s(x, u, temperature=-1.0), ValueError), (lambda: s(x, u, temperature=float("nan")), ValueError),
            (lambda: s(x, u, temperature=float("inf")), ValueError), (lambda: s(x, u, top_k=-1), ValueError), (lambda: s(x, u, top_k=1.5), ValueError),
            (lambda: s(x, u, top_p=1.1), ValueError), (lambda: s(x, u, min_p=-0.1), ValueError),
            (lambda: s(x, u, top_k=torch.ones(2)), TypeError), (lambda: s(x, u, top_p=torch.ones(3)), ValueError),
            (lambda: s(x, u, out=torch.zeros(2)), TypeError), (lambda: s(x, u, out=torch.zeros(3, dtype=torch.int64)), ValueError)]:
        with pytest.raises(error):
            call()


def test_copies_of_a_cache_have_pages_of_their_own(ops):
    """Deep copies, pickled ones and a cache whose data got other memory: every call takes the address that data has then."""
    import copy
    import pickle
    c, (table, lens) = cache_of(ops), state()
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    where = {"qvl_paged_append": 17, "qvl_paged_attention": 5, "qvl_paged_unpack": 2}    # the cache among the arguments

    def addresses(c):
        ops.calls.clear()
        ops.append_paged(k, k, c, table, lens)
        ops.paged_attention(q, c, table, lens, max_len=1)
        ops.unpack_paged(c, table, lens, torch.zeros(3, dtype=torch.int64), k.clone(), k.clone(), max_len=1)
        assert [name for name, _ in ops.calls] == list(where)
        return {a[where[name]] for name, a in ops.calls}

    others = [c, copy.deepcopy(c), pickle.loads(pickle.dumps(c))]
    for x in others:
        assert addresses(x) == {x.data.data_ptr()}
    assert len({x.data.data_ptr() for x in others}) == 3
    assert addresses(copy.copy(c)) == {c.data.data_ptr()}                # (a shallow copy is the same pages)
    c.data.data = c.data.clone()
    assert addresses(c) == {c.data.data_ptr()}


def test_data_that_is_not_the_caches_pages_is_refused(ops):
    table, lens = state()
    k = torch.zeros(3, 2, 64)
    for other in (lambda d: d[:3], lambda d: d.reshape(-1), lambda d: d.t().contiguous().t(), lambda d: d[:, :64].contiguous()):
        c = cache_of(ops)
        c.data.data = other(c.data)
        with pytest.raises(ValueError, match="pages"):
            ops.append_paged(k, k, c, table, lens)
