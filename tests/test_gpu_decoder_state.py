"""GPU tests of what lies around the decoder operators' kernels: the streams and memory of the objects they read, their
workspaces, and autograd's book of what was written."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_attn


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def test_plan_dropped_before_its_kernel_has_run(ops):
    """A plan and a rotation made on one stream, used on another that is still busy, and dropped: what the first stream
    allocates then is other memory."""
    q, k, w = rand((70, 8, 64), BF, 1), rand((70, 2, 64), BF, 2), torch.ones(64, device=DEV)
    pos = torch.arange(70, dtype=torch.int32, device=DEV)
    make = lambda: (ops.CausalPlan([70], num_heads=8, num_kv_heads=2, head_dim=64, dtype=BF, device=DEV),
                    ops.TextRotary(64, 1e4, (12, 10, 10), True, DEV))
    call = lambda plan, rot: (ops.causal_attention(q, k, k, plan), *ops.qk_norm_rotary(q, k, None, w, w, pos, rot)[:2])
    want = call(*make())
    torch.cuda.synchronize()
    plan, rot = make()
    sizes = plan.items.shape, rot.table.shape
    at = plan.items.data_ptr(), rot.table.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                            # some 50 ms
        got = call(plan, rot)
    del plan, rot
    taken = [torch.zeros(sizes[0], dtype=torch.int32, device=DEV) for _ in range(8)]
    taken += [torch.zeros(sizes[1], dtype=torch.int64, device=DEV) for _ in range(8)]
    assert not {t.data_ptr() for t in taken} & set(at)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def short_rows(name, rows, hkv, D, dtype):
    """Caches whose rows lie closer than a row is long, with a value that only seen rows hold: (k, v)."""
    inf = float("inf")
    if name == "one row":
        k, v = rand((1, hkv, D), dtype, 1), rand((1, hkv, D), dtype, 2)
        v[0, :, 3], v[0, :, D - 1] = inf, -inf
        return k, v
    if name == "expanded":
        k, v = short_rows("one row", 1, hkv, D, dtype)
        return k.expand(rows, hkv, D), v.expand(rows, hkv, D)
    flat = rand((2, hkv, rows * 16 + D), dtype, 3)
    k, v = (x.as_strided((rows, hkv, D), (16, rows * 16 + D, 1), x.storage_offset()) for x in flat)
    return k, v


def assert_sees_all(got, q, k, v):
    """Tokens that see every key, against float64: infinite where a value is, else within the bound of the attention tests (scores
    of D products off by (D + 8) 2^-24 sum|q_i k_i| scale + 4 2^-24 max|s|, sums of n terms by n 2^-24, bf16 weights and the
    output by half a step)."""
    D, g, u = q.shape[-1], q.shape[1] // k.shape[1], 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    for h in range(q.shape[1]):
        qh, kh, vh = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        s, mass = qh @ kh.t() * D ** -0.5, qh.abs() @ kh.abs().t() * D ** -0.5
        w, bad = torch.softmax(s, 1), ~vh.isfinite().all(0)
        vh = torch.where(bad[None], 0.0, vh)
        ds = (D + 8) * 2.0 ** -24 * mass.amax(1, keepdim=True) + 4 * 2.0 ** -24 * s.abs().amax(1, keepdim=True)
        A, want = w @ vh.abs(), w @ vh
        tol = (2 * ds + 2 * k.shape[0] * 2.0 ** -24 + (2 * u if got.dtype == BF else 0.0)) * A + u * want.abs()
        assert ((got[:, h].double() - want).abs() <= tol)[:, ~bad].all() and got[:, h][:, bad].isinf().all()


@pytest.mark.parametrize("dtype,hq", [(BF, 8), (BF, 80), (F32, 8), (F32, 80)])     # fp32: tiles of 16 rows, and of 32
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", ["one row", "expanded", "overlapping"])
@pytest.mark.parametrize("n", [1, 40])                                          # 40: prefixes in tiles of 128 rows
def test_rows_closer_than_a_row_is_long(ops, dtype, hq, D, name, n):
    """What lies behind a sequence's last key is then a copy of keys before it, not outside: infinite values there must not
    meet the weight 0 of a key that is not seen. Against float64, and bit for bit against the same rows in a cache of their own
    but for prefixes, which take tiles of 32 rows here and may take 128 there."""
    length = 1 if name == "one row" else 70
    k, v = short_rows(name, 200, 2, D, dtype)
    if name == "overlapping":
        v[length - 1, :, D - 5] = float("inf")
    kc, vc = torch.zeros(400, 2, D, dtype=dtype, device=DEV), torch.zeros(400, 2, D, dtype=dtype, device=DEV)
    kc[:length], vc[:length] = k[:length], v[:length]
    q = rand((n, hq, D), dtype, 5)
    t = lambda x, dt: torch.tensor(x, dtype=dt, device=DEV)
    start, lens, none = t([0] * n, torch.int64), t([length] * n, torch.int32), t([0] * n, torch.int32)
    calls = {"decode": lambda k, v: ops.decode_attention(q, k, v, start, lens, max_len=length),
             "own": lambda k, v: ops.prefix_attention(q, k, v, start, lens, start[:1], none[:1], t([0, n], torch.int32), max_len=length,
                                                      max_prefix=0),
             "prefix": lambda k, v: ops.prefix_attention(q, k, v, start, none, start[:1], lens[:1], t([0, n], torch.int32), max_len=0,
                                                         max_prefix=length),
             "causal": lambda k, v: ops.causal_attention(q, k, v, ops.CausalPlan([n], [length], [0], num_heads=hq, num_kv_heads=2,
                                                                                 head_dim=D, dtype=dtype, device=DEV))}
    for what, call in calls.items():
        got, want = call(k, v), call(kc, vc)
        if what != "prefix":
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1e3), want.nan_to_num(1e3)), what
        last = got if what != "causal" else got[-1:]                 # (a prompt's last token sees every key)
        assert_sees_all(last, q[-last.shape[0]:], k[:length], v[:length])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_nothing_is_taken_from_what_a_workspace_held(ops, monkeypatch, dtype, D):
    """Workspaces full of NaN: what a join reads of them has to be written first, the parts of sequences without a prefix, without
    keys and of bad keys too."""
    hkv, hq = 2, 8
    t = lambda x, dt: torch.tensor(x, dtype=dt, device=DEV)
    lengths = [40, 3, 17, 900, 9, 0, 33]
    start = [3 + sum(lengths[:i]) for i in range(7)]
    k, v = rand((3000, hkv, D), dtype, 1), rand((3000, hkv, D), dtype, 2)
    one, few, many = rand((7, hq, D), dtype, 3), rand((21, hq, D), dtype, 4), rand((200, hq, D), dtype, 5)
    ks, kl = t(start, torch.int64), t(lengths, torch.int32)
    bad = t([-1] + start[1:], torch.int64)
    cu = t([0, 3, 6, 9, 12, 15, 18, 21], torch.int32)
    pre = (t([1100, 2000], torch.int64), t([700, 129], torch.int32))
    cut = ops.CausalPlan([200], [2900], [0], num_heads=hq, num_kv_heads=hkv, head_dim=D, dtype=dtype, device=DEV)
    assert cut.n_joins > 0
    prefix = lambda q, start, cu_g, **kw: ops.prefix_attention(q, k, v, start, kl, *pre, t(cu_g, torch.int32), max_len=900, max_prefix=700, **kw)
    calls = [lambda: ops.decode_attention(one, k, v, ks, kl, max_len=900), lambda: ops.decode_attention(few, k, v, ks, kl, max_len=900, cu_q=cu),
             lambda: ops.decode_attention(one, k, v, bad, kl, max_len=900), lambda: prefix(one, ks, [2, 4, 5]),
             lambda: prefix(one, bad, [0, 4, 4]), lambda: prefix(few, ks, [2, 4, 5], cu_q=cu), lambda: prefix(few, ks, [0, 0, 7], cu_q=cu),
             lambda: ops.causal_attention(many, k, v, cut)]
    want = [c() for c in calls]
    held = []

    def poisoned(nbytes, q):
        if nbytes:
            held.append(torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV))      # of every float: NaN
        return held[-1] if nbytes else None

    monkeypatch.setattr(ops, "_workspace", poisoned)
    for i, (c, w) in enumerate(zip(calls, want)):
        got = c()
        assert len(held) == i + 1 and torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(7.0), w.nan_to_num(7.0)), i
    for i, w in enumerate(want):
        assert w.isnan().any() == (i in (2, 4)), i


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_values_go_to_the_cache_bit_for_bit(ops, dtype, D):
    """Every bf16 there is (for fp32: with further bits behind), signalling NaN among them."""
    n, hkv = 65536 // D // 2, 2
    b = torch.arange(65536, dtype=torch.int32)
    b = (b - (b >= 32768).int() * 65536).to(torch.int16) if dtype == BF else ((b << 16) + 0x4321 * (b % 3 > 0)).to(torch.int32)
    v = b.view(n, hkv, D).view(dtype).to(DEV)
    vc, kc = torch.zeros_like(v), torch.zeros_like(v)
    rows = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(DEV)
    ops.qk_norm_rotary(rand((n, 4, D), dtype, 1), rand((n, hkv, D), dtype, 2), v, torch.ones(D, device=DEV), torch.ones(D, device=DEV),
                       torch.arange(n, dtype=torch.int32, device=DEV), ops.TextRotary(D, 1e4, (D // 2, 0, 0), False, DEV), k_cache=kc,
                       v_cache=vc, rows=rows)
    word = torch.int16 if dtype == BF else torch.int32
    assert torch.equal(vc[rows].view(word), v.view(word))
