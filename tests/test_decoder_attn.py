"""CPU checks of the decoder operators: the rotation table, the causal work list and every refusal of the C entries and of
the Python layer that needs no GPU."""
import ctypes as C
import math
from fractions import Fraction

import numpy as np
import pytest

FAKE = 1 << 20   # never dereferenced: validation fails first


def table(pkg, head_dim, theta, section, interleaved):
    out = np.zeros((head_dim // 2, 2), np.uint64)
    sec = (C.c_int32 * 3)(*section)
    pkg.capi.check(pkg.capi.load().qvl_text_rotary_table(head_dim, theta, sec, interleaved, out.ctypes.data))
    return out


@pytest.mark.parametrize("head_dim,theta,section,interleaved", [
    (128, 5e6, (24, 20, 20), 1), (128, 5e6, (24, 20, 20), 0), (64, 1e4, (12, 10, 10), 1), (64, 1e4, (32, 0, 0), 0)])
def test_rotary_table(pkg, head_dim, theta, section, interleaved):
    t = table(pkg, head_dim, theta, section, interleaved)
    half = head_dim // 2
    for j in range(half):
        want = theta ** (-2.0 * j / head_dim) / (2 * math.pi)
        # the reference itself is a double: 2^-50 covers its power, division and pi; the entry is rounded to 2^-64
        # turns, off by up to half of that (one unit where the long double power ends near a tie)
        assert abs(float(Fraction(int(t[j, 0]), 2 ** 64)) - want) < 2.0 ** -50 * want + 2.0 ** -64
        if interleaved:
            axis = 1 if j % 3 == 1 and j < 3 * section[1] else 2 if j % 3 == 2 and j < 3 * section[2] else 0
        else:
            axis = 0 if j < section[0] else 1 if j < section[0] + section[1] else 2
        assert int(t[j, 1]) == axis


def test_rotary_table_refusals(pkg):
    f = pkg.capi.load().qvl_text_rotary_table
    out = np.zeros((128, 2), np.uint64)
    sec = lambda *s: (C.c_int32 * 3)(*s)
    for hd, theta, s in [(0, 1e4, sec(0, 0, 0)), (130, 1e4, sec(65, 0, 0)), (260, 1e4, sec(130, 0, 0)), (64, 1.0, sec(32, 0, 0)),
                         (64, float("inf"), sec(32, 0, 0)), (64, float("nan"), sec(32, 0, 0)), (64, 1e4, sec(12, 10, 9)),
                         (64, 1e4, sec(-1, 23, 10)), (64, 1e4, sec(33, 0, 0))]:
        assert f(hd, theta, s, 0, out.ctypes.data) == -1
    assert f(64, 1e4, None, 0, out.ctypes.data) == -1
    assert f(64, 1e4, sec(32, 0, 0), 0, None) == -1


def worklist(pkg, new, length, start, hq, hkv, hd=128, dtype=1, n_cus=256, tile_rows=0):
    lib = pkg.capi.load()
    a = [np.array(v, np.int64) for v in (new, length, start)]
    p = [v.ctypes.data_as(C.POINTER(C.c_int64)) for v in a]
    n, parts, joins, rows = C.c_int64(), C.c_int64(), C.c_int64(), C.c_int32(tile_rows)
    call = lambda items, cap: lib.qvl_causal_worklist(len(new), *p, hq, hkv, hd, dtype, n_cus, C.byref(rows), items, cap, C.byref(n),
                                                      C.byref(parts), C.byref(joins))
    pkg.capi.check(call(None, 0))
    items = np.zeros((n.value + joins.value, pkg.capi.QVL_CAUSAL_ITEM_WORDS), np.int32)
    ptr = items.ctypes.data_as(C.POINTER(C.c_int32))
    pkg.capi.check(call(ptr, len(items)))
    if len(items):
        assert call(ptr, len(items) - 1) == -1
    return items[:n.value].tolist(), items[n.value:].tolist(), parts.value, rows.value


@pytest.mark.parametrize("tile_rows", [0, 128, 256])
@pytest.mark.parametrize("new,old,hq,hkv,hd,dtype", [
    ([1], [0], 16, 8, 128, 1), ([300, 0, 1, 129], [0, 5, 77, 4000], 16, 8, 128, 1), ([2048], [0], 32, 8, 128, 1),
    ([40], [24000], 32, 8, 128, 1), ([1181, 317, 5], [0, 64, 0], 14, 2, 64, 0), ([7] * 40, [0] * 40, 4, 1, 64, 1),
    ([513], [1000], 6, 2, 128, 0)])
def test_worklist_covers_every_row_and_key_once(pkg, new, old, hq, hkv, hd, dtype, tile_rows):
    if tile_rows == 256 and dtype == 0:
        pytest.skip("bf16 only")
    length = [a + b for a, b in zip(new, old)]
    start = [(1 << 33) + 17 * i for i in range(len(new))]
    items, joins, n_parts, height = worklist(pkg, new, length, start, hq, hkv, hd, dtype, tile_rows=tile_rows)
    assert height in ((128, 256) if dtype == 1 else (128,)) and tile_rows in (0, height)
    group = hq // hkv
    q0 = np.concatenate([[0], np.cumsum(new)])
    seq_of = lambda first, n_new: [j for j in range(len(new)) if q0[j] == first and new[j] == n_new][0]
    tiles = {}
    for first, n_new, n_keys, row0, head, slot, lo, hi, t0, t1 in items:
        if n_new == 0:          # padding of a short queue
            continue
        i = seq_of(first, n_new)
        assert n_keys == length[i] and (hi << 32 | lo & 0xffffffff) == start[i]
        assert row0 % height == 0 and 0 <= row0 < n_new * group and -1 <= slot < n_parts
        tiles.setdefault((i, row0, head), []).append((t0, t1, slot))
    assert set(tiles) == {(i, r, h) for i in range(len(new)) for r in range(0, new[i] * group, height) for h in range(hkv)}
    cut = {}
    for (i, row0, head), got in tiles.items():
        got.sort()
        last = (min(row0 + height, new[i] * group) - 1) // group         # the tile's last token
        keys = max(min(old[i] + last + 1, length[i]), 0)
        assert got[0][0] == 0 and got[-1][1] == -(-keys // (64 if dtype == 1 else 32))
        assert all(a[1] == b[0] and a[1] > a[0] for a, b in zip(got, got[1:]))
        if len(got) > 1:                                                # consecutive slots, in the order of the keys
            assert [s for _, _, s in got] == list(range(got[0][2], got[0][2] + len(got)))
            cut[i, row0, head] = got[0][2], len(got)
        else:
            assert got[0][2] == -1
    assert sum(n for _, n in cut.values()) == n_parts
    slots = sorted(s for got in tiles.values() for _, _, s in got if s >= 0)
    assert slots == list(range(n_parts))
    assert {(seq_of(j[0], j[1]), j[3], j[4]): (j[5], j[9]) for j in joins} == cut and len(joins) == len(cut)


def test_worklist_cuts_all_tiles_of_a_sequence_at_the_same_keys(pkg):
    """Tiles of about 120 and 380 key steps on 256 slots: the long ones are cut, so that they end with the short ones."""
    items, joins, n_parts, height = worklist(pkg, [811, 300], [7824, 24301], [0, 7824], 32, 8, tile_rows=256)
    assert n_parts > 0 and joins
    steps = sorted((it[9] - it[8] for it in items if it[1]), reverse=True)
    slots = [0] * 256
    for s in steps:                                                     # as the dispatcher does: next job to the first slot free
        slots[slots.index(min(slots))] += s
    assert max(slots) <= 1.25 * sum(steps) / 256
    for i in (0, 811):
        ends = [{it[9] for it in items if it[1] and it[0] == i and it[3] == r and it[5] >= 0} for r in {it[3] for it in items if it[0] == i}]
        common = min(ends, key=len)
        assert all(len(common - e) <= 1 for e in ends)                  # but for the last, where the tile's keys end


def test_worklist_refusals(pkg):
    f = pkg.capi.load().qvl_causal_worklist
    n, w, g, rows = C.c_int64(), C.c_int64(), C.c_int64(), C.c_int32()
    one = lambda v: (C.c_int64 * 1)(v)
    ok = dict(new=4, length=9, start=0, hq=8, hkv=2, hd=128, dt=1, cus=256, rows=0)

    def rc(**k):
        a = dict(ok, **k)
        return f(1, one(a["new"]), one(a["length"]), one(a["start"]), a["hq"], a["hkv"], a["hd"], a["dt"], a["cus"],
                 C.byref(C.c_int32(a["rows"])), None, 0, C.byref(n), C.byref(w), C.byref(g))

    assert rc() == 0
    for bad in (dict(new=-1), dict(length=-1), dict(start=-1), dict(hq=7), dict(hq=0), dict(hkv=0), dict(cus=0), dict(start=1 << 57), dict(rows=64), dict(cus=1 << 17)):
        assert rc(**bad) == -1, bad
    for bad in (dict(hd=96), dict(dt=2), dict(hq=8192, hkv=8192), dict(length=1 << 30), dict(new=1 << 29),
                dict(rows=256, dt=0), dict(new=1 << 26, hq=64, hkv=64)):
        assert rc(**bad) == -2, bad
    assert f(1, None, one(1), one(0), 8, 2, 128, 1, 256, C.byref(rows), None, 0, C.byref(n), C.byref(w), C.byref(g)) == -1
    assert f(1, one(1), one(1), one(0), 8, 2, 128, 1, 256, C.byref(rows), None, 0, None, C.byref(w), C.byref(g)) == -1
    assert f(1, one(1), one(1), one(0), 8, 2, 128, 1, 256, C.byref(rows), None, 0, C.byref(n), None, C.byref(g)) == -1
    assert f(1, one(1), one(1), one(0), 8, 2, 128, 1, 256, C.byref(rows), None, 0, C.byref(n), C.byref(w), None) == -1
    assert f(1, one(1), one(1), one(0), 8, 2, 128, 1, 256, None, None, 0, C.byref(n), C.byref(w), C.byref(g)) == -1


def rotary_args(**change):
    a = dict(stream=None, dtype=1, q=FAKE, q_row=2048, q_head=128, k=FAKE, k_row=2048, k_head=128, v=FAKE, v_row=2048,
             v_head=128, qw=FAKE, kw=FAKE, eps=1e-6, pos=FAKE, pos_stride=4, table=FAKE, rows=FAKE, out_rows=9, qo=FAKE,
             qo_row=2048, qo_head=128, ko=FAKE, ko_row=2048, ko_head=128, vo=FAKE, vo_row=2048, vo_head=128, n=4, hq=16,
             hkv=8, hd=128)
    assert not set(change) - set(a)
    a.update(change)
    return list(a.values())


def test_qk_norm_rotary_refusals(pkg):
    f = pkg.capi.load().qvl_qk_norm_rotary
    for want, bad in [(-2, dict(dtype=2)), (-2, dict(hd=96)), (-1, dict(n=-1)), (-1, dict(hq=0)), (-1, dict(hkv=0)),
                      (-1, dict(eps=-1.0)), (-1, dict(eps=float("nan"))), (-1, dict(rows=None, out_rows=3)), (-1, dict(v=None)),
                      (-1, dict(vo=None)), (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(qw=None)), (-1, dict(kw=None)),
                      (-1, dict(pos=None)), (-1, dict(table=None)), (-1, dict(qo=None)), (-1, dict(ko=None)),
                      (-1, dict(q_row=-8)), (-1, dict(k_head=1 << 31)), (-3, dict(q=FAKE + 8)), (-3, dict(v_row=2044)),
                      (-3, dict(ko_head=132)), (-3, dict(rows=FAKE + 4)), (-3, dict(kw=FAKE + 4)), (-1, dict(pos_stride=-1)),
                      (-2, dict(hq=4097)), (-2, dict(n=1 << 30)), (-1, dict(out_rows=-1))]:
        assert f(*rotary_args(**bad)) == want, bad
    assert f(*rotary_args(n=0, q=None)) == 0      # nothing to do


def attn_common(**change):
    a = dict(stream=None, dtype=1, q=FAKE, q_row=2048, q_head=128, k=FAKE, k_row=1024, k_head=128, v=FAKE, v_row=1024,
             v_head=128, kv_rows=100)
    a.update({k: v for k, v in change.items() if k in a})
    return list(a.values())


def attn_tail(**change):
    a = dict(scale=0.1, out=FAKE, out_row=2048, out_head=128, n=4, hq=16, hkv=8, hd=128, ws=FAKE, ws_bytes=1 << 40)
    a.update({k: v for k, v in change.items() if k in a})
    return list(a.values())


ATTN_BAD = [(-2, dict(dtype=3)), (-2, dict(hd=80)), (-1, dict(hq=12)), (-1, dict(hkv=0)), (-1, dict(n=-1)), (-1, dict(kv_rows=-1)),
            (-1, dict(scale=0.0)), (-1, dict(scale=-1.0)), (-1, dict(scale=float("inf"))), (-1, dict(scale=float("nan"))),
            (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(out=None)), (-1, dict(q_head=-128)),
            (-1, dict(k_row=1 << 31)), (-3, dict(q=FAKE + 2)), (-3, dict(k_row=1020)), (-3, dict(out_head=4)),
            (-2, dict(hq=8192, hkv=8192)), (-2, dict(n=1 << 30))]


def test_causal_attention_refusals(pkg):
    f = pkg.capi.load().qvl_causal_attention

    def rc(items=FAKE, n_items=3, n_parts=0, n_joins=0, rows=128, **k):
        return f(*attn_common(**k), rows, items, n_items, n_parts, n_joins, *attn_tail(**k))

    for want, bad in ATTN_BAD + [(-1, dict(items=None)), (-3, dict(items=FAKE + 4)), (-1, dict(n_parts=4, n_joins=1)),
                                 (-1, dict(n_parts=-1)), (-1, dict(n_items=1 << 31)), (-1, dict(n_items=-1)), (-1, dict(rows=64)),
                                 (-1, dict(n_parts=2)), (-1, dict(n_joins=1)), (-1, dict(n_parts=2, n_joins=2)),
                                 (-1, dict(n_parts=2, n_joins=-1)), (-2, dict(rows=256, dtype=0)),
                                 (-4, dict(n_parts=2, n_joins=1, ws=None)), (-4, dict(n_parts=2, n_joins=1, ws_bytes=2 * 128 * 130 * 4 - 1)),
                                 (-3, dict(n_parts=2, n_joins=1, ws=FAKE + 8))]:
        assert rc(**bad) == want, bad
    assert rc(n=0, q=None) == 0 and rc(items=None, n_items=0) == 0
    nb = C.c_size_t()
    size = pkg.capi.load().qvl_causal_workspace_size
    assert size(128, 128, 0, C.byref(nb)) == 0 and nb.value == 0
    assert size(128, 256, 3, C.byref(nb)) == 0 and nb.value == 3 * 256 * 130 * 4
    assert size(96, 128, 4, C.byref(nb)) == -2 and size(128, 128, -1, C.byref(nb)) == -1
    assert size(128, 128, 4, None) == -1 and size(128, 64, 4, C.byref(nb)) == -1


def test_decode_attention_refusals(pkg):
    f = pkg.capi.load().qvl_decode_attention

    def rc(cu_q=None, n_seqs=4, ks=FAKE, kl=FAKE, max_len=100, cg=None, groups=0, ps=None, pl=None, max_prefix=0, **k):
        return f(*attn_common(**k), cu_q, n_seqs, ks, kl, max_len, cg, groups, ps, pl, max_prefix, *attn_tail(**k))

    for want, bad in ATTN_BAD[:-1] + [
            (-1, dict(n_seqs=-1)), (-1, dict(n_seqs=5)), (-1, dict(ks=None)), (-1, dict(kl=None)), (-1, dict(max_len=-1)),
            (-1, dict(groups=1)), (-1, dict(groups=1, cg=FAKE, ps=FAKE)), (-1, dict(groups=-1)), (-1, dict(max_prefix=-1)),
            (-3, dict(ks=FAKE + 4)), (-3, dict(kl=FAKE + 2)), (-3, dict(cu_q=FAKE + 1)),
            (-3, dict(groups=1, cg=FAKE, ps=FAKE + 4, pl=FAKE)), (-2, dict(n=70000, n_seqs=70000))]:
        assert rc(**bad) == want, bad
    assert rc(n=0, n_seqs=0, q=None) == 0


# ---------------------------------------------------------------------------------------------
# the Python layer's own checks (tensors on the CPU: every call ends before a launch)
# ---------------------------------------------------------------------------------------------
def test_python_refusals_on_the_cpu(pkg):
    torch = pytest.importorskip("torch")
    ops = pkg.decoder_attn
    q, k = torch.zeros(3, 8, 64), torch.zeros(9, 2, 64)
    ks, kl = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    dec = lambda **a: ops.decode_attention(a.get("q", q), a.get("k", k), a.get("v", k), a.get("ks", ks), a.get("kl", kl),
                                           max_len=9, **{n: a[n] for n in ("cu_q", "out") if n in a})
    with pytest.raises(ValueError, match="run on the GPU"):
        dec()
    with pytest.raises(ValueError, match="run on the GPU"):
        ops.TextRotary(64, 1e4, (32, 0, 0), False, device="cpu")
    with pytest.raises(ValueError, match="rows, heads, head_dim"):
        dec(q=q[0])
    with pytest.raises(ValueError, match="head_dim 32"):
        dec(k=k[..., :32], v=k[..., :32])
    with pytest.raises(ValueError, match="last axis"):
        dec(k=k[..., ::2], v=k[..., ::2])
    with pytest.raises(TypeError, match="bfloat16"):
        dec(k=k.bfloat16())
    with pytest.raises(ValueError, match="rows"):
        dec(v=k[:8])
    with pytest.raises(ValueError, match="heads"):
        dec(v=torch.zeros(9, 4, 64))
    with pytest.raises(TypeError, match="k_len"):
        dec(kl=kl.long())
    with pytest.raises(ValueError, match="k_len"):
        dec(kl=kl[:2])
    with pytest.raises(ValueError, match="cu_q"):
        dec(cu_q=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="out"):
        dec(out=torch.zeros(2, 8, 64))
    with pytest.raises(ValueError, match="over one another"):
        dec(out=torch.zeros(1, 8, 64).expand(3, 8, 64))
    with pytest.raises(ValueError, match="gradient"):
        dec(q=q.clone().requires_grad_())
    spec = pkg.spec_from_config({"text_config": {"hidden_size": 2048, "num_attention_heads": 16, "num_hidden_layers": 28,
                                                 "num_key_value_heads": 8, "head_dim": 128, "intermediate_size": 6144,
                                                 "rms_norm_eps": 1e-6, "vocab_size": 151936, "rope_theta": 5e6,
                                                 "rope_scaling": {"mrope_section": [24, 20, 20], "mrope_interleaved": True,
                                                                  "factor": 2.0}}})
    with pytest.raises(ValueError, match="factor"):
        ops.TextRotary.from_spec(spec.text, device="cpu")


def rotary_call(pkg, torch, **a):
    """qk_norm_rotary on CPU tensors: past its own checks it ends at the refusal of the device."""
    ops = pkg.decoder_attn
    rot = ops.TextRotary.__new__(ops.TextRotary)
    rot.head_dim, rot.table = 64, torch.zeros(32, 2, dtype=torch.int64)
    z = lambda *shape: torch.zeros(*shape)
    t = dict(q=z(3, 8, 64), k=z(3, 2, 64), v=z(3, 2, 64), q_norm=z(64), k_norm=z(64), k_cache=z(9, 2, 64), v_cache=z(9, 2, 64))
    t.update(a)
    return ops.qk_norm_rotary(t["q"], t["k"], t["v"], t["q_norm"], t["k_norm"], torch.zeros(3, dtype=torch.int32), rot,
                              k_cache=t["k_cache"], v_cache=t["v_cache"], rows=torch.arange(3), q_out=t.get("q_out"))


@pytest.mark.parametrize("name,shape", [("q", (3, 8, 64)), ("k", (3, 2, 64)), ("v", (3, 2, 64)), ("q_norm", (64,)), ("k_norm", (64,)),
                                        ("k_cache", (9, 2, 64)), ("v_cache", (9, 2, 64)), ("q_out", (3, 8, 64))])
def test_gradients_of_every_input_are_refused(pkg, name, shape):
    """The norms' weights above all: they are a model's parameters, and would get no gradient without a word."""
    torch = pytest.importorskip("torch")
    learned = torch.nn.Parameter(torch.zeros(shape))
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        rotary_call(pkg, torch, **{name: learned})
    with torch.no_grad(), pytest.raises(ValueError, match="run on the GPU"):
        rotary_call(pkg, torch, **{name: learned})
    with pytest.raises(ValueError, match="run on the GPU"):
        rotary_call(pkg, torch, **{name: learned.detach()})


@pytest.mark.parametrize("name,shape", [("q", (3, 8, 64)), ("v", (3, 2, 64)), ("k_norm", (64,)), ("k_cache", (9, 2, 64))])
def test_forward_gradients_are_refused(pkg, name, shape):
    """A tangent of forward-mode differentiation would be dropped; its tensor does not say that it requires a gradient."""
    torch = pytest.importorskip("torch")
    import torch.autograd.forward_ad as fa
    with fa.dual_level():
        dual = fa.make_dual(torch.zeros(shape), torch.ones(shape))
        with pytest.raises(ValueError, match=f"{name} carries a tangent"):
            rotary_call(pkg, torch, **{name: dual})
        with pytest.raises(ValueError, match="run on the GPU"):                  # others beside it are no matter
            rotary_call(pkg, torch, **{name: fa.unpack_dual(dual).primal})
    with pytest.raises(ValueError, match="run on the GPU"):
        rotary_call(pkg, torch)


class Recorded:
    """Stands for a device tensor that an object of the package owns."""
    def __init__(self, device):
        self.device, self.streams = device, []

    def data_ptr(self):
        return FAKE

    def record_stream(self, stream):
        self.streams.append(stream)


def test_lists_and_tables_outlive_the_streams_they_are_used_on(pkg, monkeypatch):
    """The memory of a plan's list and of a rotation's table belongs to the stream that they were made on: torch's allocator has
    to hear of every other stream that reads them, or hands it out again while a kernel there still waits. (Nothing is launched.)"""
    torch = pytest.importorskip("torch")
    ops = pkg.decoder_attn
    now, cpu = [7], torch.device("cpu")
    monkeypatch.setattr(ops, "_elsewhere", lambda device: False)
    monkeypatch.setattr(ops, "_stream", lambda device: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream", now[0]))
    monkeypatch.setattr(pkg.capi, "load", lambda: type("Lib", (), {"__getattr__": lambda self, name: lambda *a: 0})())
    plan = ops.CausalPlan.__new__(ops.CausalPlan)
    plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.dtype, plan.device = 8, 2, 64, torch.float32, cpu
    plan.n_tokens, plan.kv_rows, plan.tile_rows, plan.n_items, plan.n_parts, plan.n_joins = 3, 3, 128, 2, 0, 0
    plan.workspace_bytes, plan.items = 0, Recorded(cpu)
    plan._streams = {7}
    rot = ops.TextRotary.__new__(ops.TextRotary)
    rot.head_dim, rot.table, rot._streams = 64, Recorded(cpu), {7}
    q, k, w = torch.zeros(3, 8, 64), torch.zeros(3, 2, 64), torch.zeros(64)
    for step, want in [(7, []), (9, [9]), (7, [9]), (9, [9]), (11, [9, 11])]:
        now[0] = step
        ops.causal_attention(q, k, k, plan)
        ops.qk_norm_rotary(q, k, None, w, w, torch.zeros(3, dtype=torch.int32), rot)
        assert plan.items.streams == rot.table.streams == [("stream", s) for s in want], step


def test_written_tensors_count_as_changed(pkg, monkeypatch):
    """Autograd keeps what another operation saved for its backward pass, and looks at the version of it: a cache that a decoder
    operator wrote to in between must not pass as unchanged. (Nothing is launched.)"""
    torch = pytest.importorskip("torch")
    ops = pkg.decoder_attn
    monkeypatch.setattr(ops, "_elsewhere", lambda device: False)
    monkeypatch.setattr(ops, "_stream", lambda device: 7)
    monkeypatch.setattr(pkg.capi, "load", lambda: type("Lib", (), {"__getattr__": lambda self, name: lambda *a: 0})())
    rot = ops.TextRotary.__new__(ops.TextRotary)
    rot.head_dim, rot.table, rot._streams = 64, Recorded(torch.device("cpu")), {7}
    plan = ops.CausalPlan.__new__(ops.CausalPlan)
    plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.dtype, plan.device = 8, 2, 64, torch.float32, torch.device("cpu")
    plan.n_tokens, plan.kv_rows, plan.tile_rows, plan.n_items, plan.n_parts, plan.n_joins = 3, 3, 128, 2, 0, 0
    plan.workspace_bytes, plan.items, plan._streams = 0, Recorded(torch.device("cpu")), {7}
    q, k, v, w = torch.zeros(3, 8, 64), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(64)
    kc, vc, out = torch.zeros(9, 2, 64), torch.zeros(9, 2, 64), torch.zeros(3, 8, 64)
    pos, start, n = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)

    learned = torch.zeros(9, 2, 64, requires_grad=True)
    loss = (learned * kc).sum()                                      # saves kc
    ops.qk_norm_rotary(q, k, v, w, w, pos, rot, k_cache=kc, v_cache=vc, rows=start, q_out=out)
    assert (kc._version, vc._version, out._version) == (1, 1, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    ops.qk_norm_rotary(q, k, None, w, w, pos, rot, q_out=q)
    assert (q._version, k._version) == (1, 0)
    ops.causal_attention(q, k, v, plan, out=out)
    assert out._version == 2
    ops.decode_attention(q, kc, vc, start, n, max_len=9, out=out)
    assert out._version == 3
    ops.prefix_attention(q, kc, vc, start, n, start[:1], n[:1], n[:2], max_len=9, max_prefix=9, out=out)
    assert out._version == 4
    assert (k._version, v._version, kc._version, vc._version, w._version) == (0, 0, 1, 1, 0)
    with torch.inference_mode():                                     # tensors without a version
        made = torch.zeros(3, 8, 64)
        ops.decode_attention(q, kc, vc, start, n, max_len=9, out=made)
