"""GPU tests of the decoder operators against plain float64 computations.

Tolerances (u = half a step of the dtype: 2^-24 fp32, 2^-8 bf16):
rotary     a head's sum of squares adds 16 products in a lane and crosses 3 exchanges: 20 roundings, halved by the root; the
           root, division, scaling by the norm, sine, cosine and rotation add 10 more at most. So |error| <= 20 * 2^-24
           (|a| + |b|) for the rotated pair (a, b), and u |value| for the output's rounding.
attention  with w the softmax weights and A = sum w |v|: a score of D products, its scaling and the power of two are off
           by at most (D + 8) 2^-24 (sum |q_i k_i| scale) + 4 * 2^-24 max|s| absolutely, which moves a weight by that relative
           amount, numerator and denominator alike; the fp32 sums over n keys add n 2^-24 each (they are split into
           shorter runs, which only helps). bf16 kernels round the weights (u each, numerator and denominator), and the
           output is rounded (u): |error| <= (2 (score error) + 2 n 2^-24 [+ 2 u bf16]) A + u |value|.
           These bounds are for the worst alignment of all roundings; independent ones leave their root mean square, so
           the error of all outputs together, relative to theirs, is also held below one u in bf16 (rounded outputs are
           2^-9.3 off, the weights' rounding adds as much again) and below 2^-18 in fp32 (scores up to 2^5 with 2^-24).
"""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_attn


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


# ---------------------------------------------------------------------------------------------
# qk_norm_rotary
# ---------------------------------------------------------------------------------------------
def rotary_ref(x, w, pos, theta, section, interleaved, eps):
    """(float64 result, |a| + |b| of each rotated pair)."""
    D = x.shape[-1]
    half = D // 2
    if interleaved:
        axes = [j % 3 if j < 3 * section[j % 3] else 0 for j in range(half)]
    else:
        axes = [0] * section[0] + [1] * section[1] + [2] * section[2]
    angle = pos.double()[axes].t() * theta ** (-2.0 * torch.arange(half, dtype=torch.float64, device=x.device) / D)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    y = x.double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    a, b = y[..., :half], y[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([a.abs() + b.abs()] * 2, -1)


def assert_rotary(got, x, w, pos, rotary, eps=1e-6):
    want, size = rotary_ref(x, w, pos, rotary.theta, rotary.section, rotary.interleaved, eps)
    tol = 20 * 2.0 ** -24 * size + HALF_STEP[got.dtype] * want.abs()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq,hkv,D,section,interleaved", [
    (16, 8, 128, (24, 20, 20), True), (32, 8, 128, (24, 20, 20), False), (14, 2, 64, (12, 10, 10), True),
    (1, 1, 64, (32, 0, 0), False), (3, 3, 128, (24, 20, 20), True)])
@pytest.mark.parametrize("n", [1, 5, 130])
def test_rotary_into_cache(ops, dtype, hq, hkv, D, section, interleaved, n):
    rot = ops.TextRotary(D, 5e6, section, interleaved, DEV)
    qkv = rand((n, (hq + 2 * hkv) * D), dtype, n + hq)
    q = qkv[:, :hq * D].unflatten(1, (hq, D))
    k = qkv[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D))
    v = qkv[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
    qw, kw = 1 + 0.2 * rand((D,), F32, 1), 1 + 0.2 * rand((D,), F32, 2)
    pos = torch.randint(0, 40000, (3, n), generator=torch.Generator().manual_seed(n), dtype=torch.int32).to(DEV)
    R = 2 * n + 3
    rows = torch.randperm(R, generator=torch.Generator().manual_seed(n))[:n].to(DEV)
    kc, vc = rand((R, hkv, D), dtype, 7), rand((R, hkv, D), dtype, 8)
    kc0, vc0, qkv0 = kc.clone(), vc.clone(), qkv.clone()
    qo, ko, vo = ops.qk_norm_rotary(q, k, v, qw, kw, pos, rot, k_cache=kc, v_cache=vc, rows=rows)
    assert ko is kc and vo is vc
    assert_rotary(qo, q, qw, pos, rot)
    assert_rotary(kc[rows], k, kw, pos, rot)
    assert torch.equal(vc[rows], v)
    rest = torch.ones(R, dtype=torch.bool, device=DEV)
    rest[rows] = False
    assert torch.equal(kc[rest], kc0[rest]) and torch.equal(vc[rest], vc0[rest])    # every other row as it was
    assert torch.equal(qkv, qkv0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_far_and_negative_positions(ops, dtype):
    pos = torch.tensor([0, 1, 65537, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -1, -(2 ** 31)], dtype=torch.int32, device=DEV)
    rot = ops.TextRotary(128, 1e6, (64, 0, 0), False, DEV)
    q, k = rand((8, 4, 128), dtype, 1), rand((8, 2, 128), dtype, 2)
    w = torch.ones(128, device=DEV)
    qo, ko, v = ops.qk_norm_rotary(q, k, None, w, w, pos, rot)
    assert v is None
    # the float64 reference's own angle at 2^31 is off by 2^31 * 2^-53: far below the tolerance
    assert_rotary(qo, q, w, pos[None].repeat(3, 1), rot)
    assert_rotary(ko, k, w, pos[None].repeat(3, 1), rot)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_two_tokens_of_one_row(ops, dtype):
    """The row holds values of the one or the other, and no other row changes."""
    n, hq, hkv, D = 64, 4, 2, 64
    rot = ops.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    w = 1 + 0.1 * rand((D,), F32, 3)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    q, k, v = rand((n, hq, D), dtype, 1), rand((n, hkv, D), dtype, 2), rand((n, hkv, D), dtype, 4)
    _, alone, _ = ops.qk_norm_rotary(q, k, v, w, w, pos, rot)
    kc, vc = rand((40, hkv, D), dtype, 5), rand((40, hkv, D), dtype, 6)
    kc0, vc0 = kc.clone(), vc.clone()
    rows = (torch.arange(n, device=DEV) // 2) + 4                            # tokens 2 i and 2 i + 1 both to row i + 4
    ops.qk_norm_rotary(q, k, v, w, w, pos, rot, k_cache=kc, v_cache=vc, rows=rows)
    for got, a in ((kc, alone), (vc, v)):
        assert ((got[4:36] == a[0::2]) | (got[4:36] == a[1::2])).all()
    assert torch.equal(kc[36:], kc0[36:]) and torch.equal(vc[:4], vc0[:4]) and torch.equal(kc[:4], kc0[:4])


def test_rotary_strides_in_place_and_dropped_rows(ops):
    n, hq, hkv, D = 70, 6, 2, 64
    rot = ops.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    w = 1 + 0.1 * rand((D,), F32, 3)
    pos = torch.arange(3 * n, dtype=torch.int32, device=DEV).view(3, n)
    q, k, v = rand((hq, n, D), BF, 1).transpose(0, 1), rand((n, hkv, D + 8), BF, 2)[..., :D], rand((n, hkv, D), BF, 3)
    q0, k0 = q.clone(), k.clone()
    R = 50
    kc, vc = rand((hkv, R, D), BF, 4).transpose(0, 1), rand((hkv, R, D), BF, 5).transpose(0, 1)   # head-major caches
    kc0, vc0 = kc.clone(), vc.clone()
    rows = torch.full((n,), -1, dtype=torch.int64, device=DEV)
    rows[3], rows[4], rows[69], rows[10], rows[11] = 0, 49, 7, 50, 1 << 40
    qo, _, _ = ops.qk_norm_rotary(q, k, v, w, w, pos, rot, k_cache=kc, v_cache=vc, rows=rows, q_out=q)   # q in place
    assert qo is q
    assert_rotary(q, q0, w, pos, rot)
    keep = torch.tensor([3, 4, 69], device=DEV)
    assert_rotary(kc[rows[keep]], k0[keep], w, pos[:, keep], rot)
    assert torch.equal(vc[rows[keep]], v[keep])
    rest = torch.ones(R, dtype=torch.bool, device=DEV)
    rest[rows[keep]] = False
    assert torch.equal(kc[rest], kc0[rest]) and torch.equal(vc[rest], vc0[rest])
    assert ops.qk_norm_rotary(q[:0], k[:0], None, w, w, pos[:, :0].contiguous(), rot)[0].shape == (0, hq, D)


def test_rotary_row_of_zeros_and_infinities(ops):
    """A head of zeros stays zero (eps > 0), and a head that holds infinities or NaN touches no other head."""
    rot = ops.TextRotary(128, 1e6, (64, 0, 0), False, DEV)
    q, k = rand((4, 8, 128), F32, 1), rand((4, 8, 128), F32, 2)
    q[1, 2] = 0
    q[2, 3, 5] = float("inf")
    k[3, 4, 6] = float("nan")
    w = torch.ones(128, device=DEV)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    qo, ko, _ = ops.qk_norm_rotary(q, k, None, w, w, pos, rot)
    assert (qo[1, 2] == 0).all()
    fq, fk = qo.isfinite().all(-1), ko.isfinite().all(-1)
    assert not fq[2, 3] and not fk[3, 4] and int(fq.sum()) == 31 and int(fk.sum()) == 31


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def attention_ref(q, keys, values, visible, scale):
    """One sequence in float64: q [n, Hq, D], keys / values [L, Hkv, D], visible [n]: how many of the keys each token sees
    (the first `prefix` + ... in order). Returns (out, A = sum w|v|, score error bound)."""
    n, hq, D = q.shape
    g = hq // keys.shape[1]
    out = torch.zeros(n, hq, D, dtype=torch.float64, device=q.device)
    A, ds = torch.zeros_like(out), torch.zeros(n, hq, 1, dtype=torch.float64, device=q.device)
    mask = torch.arange(keys.shape[0], device=q.device)[None] < visible[:, None]
    for h in range(hq):
        kh, vh, qh = keys[:, h // g].double(), values[:, h // g].double(), q[:, h].double()
        # keys that no token sees may hold anything
        kh, vh = torch.where(mask.any(0)[:, None], kh, 0), torch.where(mask.any(0)[:, None], vh, 0)
        s = (qh @ kh.t()) * scale
        mass = (qh.abs() @ kh.abs().t()) * scale
        s = torch.where(mask, s, -math.inf)
        m = s.amax(1, keepdim=True).clamp_min(-1e300) if keys.shape[0] else torch.zeros(n, 1, device=q.device)
        w = torch.exp(s - m)
        w = torch.where(mask, w, 0)
        l = w.sum(1, keepdim=True)
        w = torch.where(l > 0, w / l.clamp_min(1e-300), 0)
        out[:, h], A[:, h] = w @ vh, w @ vh.abs()
        if keys.shape[0]:
            big = torch.where(mask, s.abs(), 0).amax(1, keepdim=True)
            ds[:, h] = (D + 8) * 2.0 ** -24 * torch.where(mask, mass, 0).amax(1, keepdim=True) + 4 * 2.0 ** -24 * big
    return out, A, ds


def assert_attention(got, ref, n_keys):
    want, A, ds = ref
    u = HALF_STEP[got.dtype]
    tol = (2 * ds + 2 * n_keys * 2.0 ** -24 + (2 * u if got.dtype == BF else 0)) * A + u * want.abs()
    err = (got.double() - want).abs()
    assert err.isfinite().all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    norm = float(want.norm())
    if norm > 0:
        rel = float(err.norm()) / norm
        assert rel <= (2.0 ** -8 if got.dtype == BF else 2.0 ** -18), rel


def causal_case(hq, hkv, D, dtype, new, old, seed=0, kv=None):
    """q, k, v of a packed prefill and, by sequence, (first token, new, first row, keys)."""
    rows, seqs, q0 = 3, [], 0
    for a, b in zip(new, old):
        length = max(a + b, 0)
        seqs.append((q0, a, rows, length))
        q0, rows = q0 + a, rows + length + 2
    q = rand((q0 + 2, hq, D), dtype, seed, 1.4)
    k, v = (rand((rows, hkv, D), dtype, seed + 1, 1.4), rand((rows, hkv, D), dtype, seed + 2)) if kv is None else kv(rows)
    return q, k, v, seqs


def plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows=0):
    return ops.CausalPlan([s[1] for s in seqs], [s[3] for s in seqs], [s[2] for s in seqs], num_heads=hq, num_kv_heads=hkv,
                          head_dim=D, dtype=dtype, device=DEV, tile_rows=tile_rows)


# both tile heights of bf16, and fp32's
KERNELS = [(BF, 128), (BF, 256), (F32, 128)]


def check_causal(out, q, k, v, seqs, scale):
    for q0, n, row, length in seqs:
        if n == 0:
            continue
        visible = (torch.arange(n, device=DEV) + length - n + 1).clamp_min(0)
        ref = attention_ref(q[q0:q0 + n], k[row:row + length], v[row:row + length], visible, scale)
        assert_attention(out[q0:q0 + n], ref, length)


CAUSAL = [  # new tokens, keys before them (negative: fewer keys than new tokens)
    ([1], [0]), ([64], [0]), ([65, 1, 130], [0, 0, 0]), ([0, 3, 0], [4, 0, 0]), ([33], [1000]), ([1, 2, 3], [63, 64, 65]),
    ([300], [-40]), ([5], [-5]), ([257, 31], [129, 2049]), ([700], [0])]


@pytest.mark.parametrize("dtype,tile_rows", KERNELS)
@pytest.mark.parametrize("hq,hkv,D", [(16, 8, 128), (32, 8, 128), (14, 2, 64), (4, 4, 64), (6, 2, 128), (5, 1, 128)])
@pytest.mark.parametrize("new,old", CAUSAL)
def test_causal(ops, dtype, tile_rows, hq, hkv, D, new, old):
    q, k, v, seqs = causal_case(hq, hkv, D, dtype, new, old, seed=sum(new) + hq)
    plan = plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows)
    out = torch.full_like(q, 7.0)
    assert ops.causal_attention(q, k, v, plan, out=out) is out
    check_causal(out, q, k, v, seqs, D ** -0.5)
    assert (out[sum(new):] == 7.0).all()            # rows behind the last sequence


@pytest.mark.parametrize("dtype,tile_rows", KERNELS)
def test_causal_long_and_peaked(ops, dtype, tile_rows):
    """Scores whose maximum moves up along the keys, by far more than one power of two a tile, and a scale of its own."""
    hq, hkv, D = 4, 2, 128
    q, k, v, seqs = causal_case(hq, hkv, D, dtype, [900], [1500], seed=5)
    k = (k.float() * torch.linspace(0.1, 3.0, k.shape[0], device=DEV)[:, None, None]).to(dtype)
    out = ops.causal_attention(q, k, v, plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows), scale=0.2)
    check_causal(out, q, k, v, seqs, 0.2)


@pytest.mark.parametrize("dtype,tile_rows", KERNELS)
def test_causal_large_scores(ops, dtype, tile_rows):
    """Scores of hundreds, of both signs: the weights under- and overflow without the running maximum."""
    hq, hkv, D = 4, 2, 64
    q, k, v, seqs = causal_case(hq, hkv, D, dtype, [200], [77], seed=6)
    q = (q.float() * 40).to(dtype)
    out = ops.causal_attention(q, k, v, plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows))
    for q0, n, row, length in seqs:
        visible = torch.arange(n, device=DEV) + length - n + 1
        want, A, ds = attention_ref(q[q0:q0 + n], k[row:row + length], v[row:row + length], visible, D ** -0.5)
        # the weights of near ties move by the score error, which is no small number here: only the worst-case bound
        u = HALF_STEP[dtype]
        tol = (torch.expm1(2 * ds) + 2 * length * 2.0 ** -24 + (2 * u if dtype == BF else 0)) * A + u * want.abs()
        # a key whose weight is tiny in float64 may take part in the error with |v| up to the largest
        tol = tol + torch.expm1(2 * ds) * float(v.double().abs().max()) * 2.0 ** -4
        assert ((out[q0:q0 + n].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("D", [64, 128])
def test_causal_scores_far_above_the_first_tile(ops, D):
    """Some rows' scores from key 64 on exceed the first 64 by 2^400 in the weight, others stay far below: sums held against
    the first tile's maximum overflow, and those rows alone are formed again. Every row is exact to the usual bound."""
    hq, hkv, n, old = 4, 2, 130, 200
    q, k, v, seqs = causal_case(hq, hkv, D, BF, [n], [old], seed=31)
    row = seqs[0][2]
    u = rand((D,), F32, 32)
    u = u / u.norm()
    away = lambda x: x.float() - (x.float() @ u)[..., None] * u           # nothing of direction u in it
    kf, qf = away(k), away(q)
    kf[row + 64:row + old + n] += 20.0 * u                                  # keys 64 and later
    side = torch.where(torch.arange(n, device=DEV) % 3 == 0, 1.0, -1.0)     # every third token looks there, the others away
    qf[:n] += (side * 14.0 * math.sqrt(D))[:, None, None] * u               # +-280 of a score, +-404 in powers of two
    q, k = qf.to(BF), kf.to(BF)
    for rows in (128, 256):
        check_causal(ops.causal_attention(q, k, v, plan_of(ops, seqs, hq, hkv, D, BF, rows)), q, k, v, seqs, D ** -0.5)


def test_captured_causal_attention(ops):
    """A captured prefill of cut and joined tiles, replayed with other inputs in the same buffers and eager work between."""
    hq, hkv, D = 32, 8, 128
    q, k, v, seqs = causal_case(hq, hkv, D, BF, [300, 20], [3000, 5], seed=33)
    plan = plan_of(ops, seqs, hq, hkv, D, BF)
    assert plan.n_joins > 0
    n = sum(s[1] for s in seqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.causal_attention(q, k, v, plan)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.causal_attention(q, k, v, plan)
    for i in range(4):
        q.copy_(rand(tuple(q.shape), BF, 70 + i))
        v.copy_(rand(tuple(v.shape), BF, 80 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(got[:n]), bits(ops.causal_attention(q, k, v, plan)[:n])), i


def test_nothing_to_do(ops):
    """Plans without sequences or without tokens, caches without rows, decode steps without sequences."""
    q, k = rand((3, 8, 64), BF, 1), rand((5, 2, 64), BF, 2)
    for new, keys in ([], []), ([0, 0], [0, 4]):
        plan = ops.CausalPlan(new, keys, [0] * len(new), num_heads=8, num_kv_heads=2, head_dim=64, dtype=BF, device=DEV)
        out = torch.full_like(q, 7.0)
        assert (ops.causal_attention(q, k, k, plan, out=out) == 7.0).all()
        assert ops.causal_attention(q[:0], k, k, plan).shape == (0, 8, 64)
    plan = ops.CausalPlan([3], [0], [0], num_heads=8, num_kv_heads=2, head_dim=64, dtype=BF, device=DEV)
    assert (ops.causal_attention(q, k[:0], k[:0], plan) == 0).all()          # no keys at all: zeros
    none = lambda dt: torch.zeros(0, dtype=dt, device=DEV)
    assert ops.decode_attention(q[:0], k, k, none(torch.int64), none(torch.int32), max_len=9).shape == (0, 8, 64)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert (ops.decode_attention(q, k[:0], k[:0], zero.long(), zero, max_len=0) == 0).all()


@pytest.mark.parametrize("dtype,tile_rows", KERNELS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_causal_masked_keys_hold_anything(ops, dtype, tile_rows, bad):
    """Rows of the caches outside the sequences, and a token's later keys, hold NaN or infinities; the tokens that do
    see a bad key may be anything, the others are exact."""
    hq, hkv, D, n, old = 8, 2, 128, 150, 70
    q, k, v, seqs = causal_case(hq, hkv, D, dtype, [n, 64], [old, 0], seed=8)
    clean_k, clean_v = k.clone(), v.clone()
    used = torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
    for _, _, row, length in seqs:
        used[row:row + length] = True
    k[~used], v[~used] = bad, bad
    at = seqs[0][2] + old + 100                     # key of new token 100 of the first sequence
    k[at], v[at + 1] = bad, bad                     # and the value of token 101
    v[at + 20, :, ::3] = bad
    out = ops.causal_attention(q, k, v, plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows))
    plan = plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows)
    want = ops.causal_attention(q, clean_k, clean_v, plan)
    assert torch.equal(bits(out[:100]), bits(want[:100])) and torch.equal(bits(out[n:n + 64]), bits(want[n:n + 64]))
    # token 101's value is seen by tokens 101 on, in every dim
    assert not out[101:n].isfinite().all(-1).any()


@pytest.mark.parametrize("dtype,tile_rows", KERNELS)
def test_causal_strided_views(ops, dtype, tile_rows):
    hq, hkv, D = 12, 4, 64
    q, k, v, seqs = causal_case(hq, hkv, D, dtype, [90, 45], [30, 0], seed=9)
    plan = plan_of(ops, seqs, hq, hkv, D, dtype, tile_rows)
    want = ops.causal_attention(q, k, v, plan)
    headmajor = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    padded = lambda t: torch.cat([t, t, t], 2)[..., D:2 * D]
    out = padded(torch.zeros_like(q))
    for qq, kk, vv, oo in [(headmajor(q), headmajor(k), padded(v), None), (padded(q), padded(k), headmajor(v), out)]:
        got = ops.causal_attention(qq, kk, vv, plan, out=oo)
        assert torch.equal(bits(got[:135]), bits(want[:135]))


def test_causal_offsets_past_32_bits(ops):
    """Keys that begin more than 4 GiB into the cache, and a head stride that alone passes it."""
    D, n = 64, 100
    rows = (1 << 31) // D + 5000                    # 4 GiB of bf16 rows of one head, and some
    k, v = torch.empty((rows, 1, D), dtype=BF, device=DEV), torch.empty((rows, 1, D), dtype=BF, device=DEV)
    first = rows - 1000
    k[first:], v[first:] = rand((1000, 1, D), BF, 1), rand((1000, 1, D), BF, 2)
    q = rand((n, 2, D), BF, 3)
    seqs = [(0, n, first + 300, 650)]
    out = ops.causal_attention(q, k, v, plan_of(ops, seqs, 2, 1, D, BF))
    check_causal(out, q, k, v, seqs, D ** -0.5)
    ks, kl = torch.tensor([first + 300], device=DEV), torch.tensor([650], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    check_causal(ops.decode_attention(q, k, v, ks, kl, max_len=650, cu_q=cu), q, k, v, seqs, D ** -0.5)
    del k, v
    half = (1 << 30) + 8 * D                        # elements between the two heads: over 2 GiB
    flat = torch.empty((2 * half,), dtype=BF, device=DEV)
    k = flat.as_strided((700, 2, D), (D, half, 1))
    k.copy_(rand((700, 2, D), BF, 4))
    seqs = [(0, n, 20, 680)]
    check_causal(ops.causal_attention(q, k, k, plan_of(ops, seqs, 2, 2, D, BF)), q, k, k, seqs, D ** -0.5)


def decode_state(lengths, prefixes=(), groups=(), new=None):
    rows, starts, pstarts = 4, [], []
    for p in prefixes:
        pstarts.append(rows)
        rows += p + 1
    for length in lengths:
        starts.append(rows)
        rows += length + 3
    t = lambda v, dt: torch.tensor(v, dtype=dt, device=DEV)
    st = dict(rows=rows, starts=starts, pstarts=pstarts, k_start=t(starts, torch.int64), k_len=t(list(lengths), torch.int32),
              prefix_start=t(pstarts, torch.int64), prefix_len=t(list(prefixes), torch.int32),
              cu_groups=t(np.concatenate([[0], np.cumsum(groups)]).tolist(), torch.int32))
    st["new"] = new or [1] * len(lengths)
    st["cu_q"] = None if new is None else t(np.concatenate([[0], np.cumsum(new)]).tolist(), torch.int32)
    return st


def decode_call(ops, st, q, k, v, lengths, prefixes, **kw):
    if len(prefixes):
        return ops.prefix_attention(q, k, v, st["k_start"], st["k_len"], st["prefix_start"], st["prefix_len"],
                                    st["cu_groups"], max_len=max(lengths), max_prefix=max(prefixes), cu_q=st["cu_q"], **kw)
    return ops.decode_attention(q, k, v, st["k_start"], st["k_len"], max_len=max(lengths), cu_q=st["cu_q"], **kw)


def check_decode(out, st, q, k, v, lengths, prefixes, groups, scale):
    group = [g for g, n in enumerate(groups) for _ in range(n)] or [None] * len(lengths)
    at = 0
    for i, (n, length) in enumerate(zip(st["new"], lengths)):
        p = prefixes[group[i]] if group[i] is not None else 0
        ps = st["pstarts"][group[i]] if group[i] is not None else 0
        kk = torch.cat([k[ps:ps + p], k[st["starts"][i]:st["starts"][i] + length]])
        vv = torch.cat([v[ps:ps + p], v[st["starts"][i]:st["starts"][i] + length]])
        visible = p + (torch.arange(n, device=DEV) + length - n + 1).clamp_min(0)
        if n:
            assert_attention(out[at:at + n], attention_ref(q[at:at + n], kk, vv, visible, scale), p + length)
        at += n


DECODE = [  # lengths, new tokens (None: one each), prefixes, sequences of each group
    ([1], None, [], []), ([9001], None, [], []), ([0, 1, 2, 63, 64, 65, 1000, 0], None, [], []),
    ([5, 40, 200, 3], [3, 1, 0, 5], [], []), ([300, 2], [40, 9], [], []), ([17] * 70, None, [], []),
    ([1, 5, 33], None, [1000], [3]), ([1], None, [64], [1]), ([0, 1, 70, 9, 4], None, [129, 0, 513], [2, 2, 1]),
    ([3, 50, 9, 1], [2, 3, 1, 4], [700, 33], [1, 3]), ([1 + i % 7 for i in range(80)], None, [2000], [80]),
    ([2, 2, 2], None, [65, 64, 63], [0, 3, 0]), ([5] * 37, [3] * 37, [300, 190], [36, 1])]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq,hkv,D", [(16, 8, 128), (32, 8, 128), (14, 2, 64), (4, 4, 64), (40, 1, 128)])
@pytest.mark.parametrize("lengths,new,prefixes,groups", DECODE)
def test_decode_and_prefix(ops, dtype, hq, hkv, D, lengths, new, prefixes, groups):
    st = decode_state(lengths, prefixes, groups, new)
    n = sum(st["new"])
    k, v = rand((st["rows"], hkv, D), dtype, 1, 1.4), rand((st["rows"], hkv, D), dtype, 2)
    q = rand((n + (2 if new else 0), hq, D), dtype, 3, 1.4)
    out = torch.full_like(q, 7.0)
    assert decode_call(ops, st, q, k, v, lengths, prefixes, out=out) is out
    check_decode(out, st, q, k, v, lengths, prefixes, groups, D ** -0.5)
    assert (out[n:] == 7.0).all()


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 64)])
@pytest.mark.parametrize("n", [65, 256, 257, 300, 1100])
def test_decode_of_many_sequences(ops, dtype, D, n):
    """More sequences than a wave's lanes, and than a workgroup's threads; some empty, one much longer than the rest."""
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 90, (n,), generator=g).tolist()
    lengths[n // 3], lengths[n - 1] = 5000, 0
    new = None if n % 2 else torch.randint(0, 3, (n,), generator=g).tolist()
    st = decode_state(lengths, new=new)
    m = sum(st["new"])
    k, v, q = rand((st["rows"], 2, D), dtype, 1, 1.4), rand((st["rows"], 2, D), dtype, 2), rand((m, 8, D), dtype, 3, 1.4)
    out = decode_call(ops, st, q, k, v, lengths, [])
    check_decode(out, st, q, k, v, lengths, [], [], D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sequences_of_no_group_have_no_prefix(ops, dtype):
    """cu_groups that covers sequences 2 to 4 of 7: the others (a padded batch's tail, say) see their own keys alone."""
    lengths, prefixes, groups = [40, 3, 17, 60, 9, 0, 33], [700, 129], [2, 1]
    st = decode_state(lengths, prefixes, groups)
    k, v, q = rand((st["rows"], 2, 64), dtype, 1), rand((st["rows"], 2, 64), dtype, 2), rand((7, 8, 64), dtype, 3)
    st["cu_groups"] = torch.tensor([2, 4, 5], dtype=torch.int32, device=DEV)
    want = torch.empty_like(q)
    for i, g in enumerate([None, None, 0, 0, 1, None, None]):
        one = decode_state(lengths, prefixes, groups)
        pick = lambda t: t[i:i + 1].contiguous()
        if g is None:
            want[i] = ops.decode_attention(q[i:i + 1], k, v, pick(one["k_start"]), pick(one["k_len"]), max_len=lengths[i])[0]
        else:
            want[i] = ops.prefix_attention(q[i:i + 1], k, v, pick(one["k_start"]), pick(one["k_len"]), one["prefix_start"][g:g + 1],
                                           one["prefix_len"][g:g + 1], torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                                           max_len=lengths[i], max_prefix=prefixes[g])[0]
    for _ in range(3):                                                      # with whatever an earlier call left in the workspace
        junk = torch.full((1 << 22,), float("nan"), device=DEV)
        del junk
        out = decode_call(ops, st, q, k, v, lengths, prefixes)
        check_rows = [attention_ref(q[i:i + 1], k[s:s + n], v[s:s + n], torch.tensor([n], device=DEV), 64 ** -0.5)
                      for i, (s, n) in enumerate(zip(st["starts"], lengths))]
        for i in (0, 1, 5, 6):
            assert_attention(out[i:i + 1], check_rows[i], max(lengths[i], 1))
        # the two orders of joining differ by their fp32 sums and each output's rounding
        err = (out.double() - want.double()).abs()
        assert (err <= (2 * HALF_STEP[dtype] + 8192 * 2.0 ** -24 + (4 * 2.0 ** -8 if dtype == BF else 0)) * float(v.double().abs().max())).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hint", [1, 64, 100000])
def test_decode_lengths_other_than_the_hints(ops, dtype, hint):
    """max_len and max_prefix only lay the launch out: sequences longer or shorter than them are right too."""
    lengths, prefixes, groups = [700, 3, 1300], [900, 40], [2, 1]
    st = decode_state(lengths, prefixes, groups)
    k, v, q = rand((st["rows"], 2, 128), dtype, 1), rand((st["rows"], 2, 128), dtype, 2), rand((3, 8, 128), dtype, 3)
    out = ops.prefix_attention(q, k, v, st["k_start"], st["k_len"], st["prefix_start"], st["prefix_len"], st["cu_groups"],
                               max_len=hint, max_prefix=hint)
    check_decode(out, st, q, k, v, lengths, prefixes, groups, 128 ** -0.5)
    st = decode_state(lengths)
    out = ops.decode_attention(q, k, v, st["k_start"], st["k_len"], max_len=hint)
    check_decode(out, st, q, k, v, lengths, [], [], 128 ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decode_bad_state_comes_out_nan(ops, dtype):
    """Keys or prefixes that leave the cache: the sequence's tokens are NaN, the others are right, nothing outside is read."""
    lengths, prefixes, groups = [40, 50, 60, 70, 80, 9, 10], [100, 30], [6, 1]
    st = decode_state(lengths, prefixes, groups)
    R = st["rows"]
    k, v, q = rand((R, 2, 64), dtype, 1), rand((R, 2, 64), dtype, 2), rand((7, 4, 64), dtype, 3)
    st["k_start"][1], st["k_start"][2], st["k_len"][3], st["k_start"][4] = -1, R - 59, -2, 1 << 60
    st["prefix_len"][1] = R
    for p in ([], prefixes):
        out = decode_call(ops, st, q, k, v, lengths, p)
        bad = [1, 2, 3, 4] + ([6] if p else [])
        assert out[bad].isnan().all()
        ok = [i for i in range(7) if i not in bad]
        assert out[ok].isfinite().all()
        want = decode_call(ops, decode_state(lengths, prefixes, groups), q, k, v, lengths, p)
        assert torch.equal(bits(out[ok]), bits(want[ok]))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_decode_unseen_rows_hold_anything(ops, dtype, bad):
    lengths, new, prefixes, groups = [33, 70, 5, 128], [1, 4, 2, 3], [65], [4]
    st = decode_state(lengths, prefixes, groups, new)
    k, v, q = rand((st["rows"], 2, 128), dtype, 1), rand((st["rows"], 2, 128), dtype, 2), rand((10, 8, 128), dtype, 3)
    want = decode_call(ops, st, q, k, v, lengths, prefixes)
    used = torch.zeros(st["rows"], dtype=torch.bool, device=DEV)
    for s, n in zip(st["starts"] + st["pstarts"], lengths + prefixes):
        used[s:s + n] = True
    k[~used], v[~used] = bad, bad
    last = st["starts"][1] + 69                     # the last key of the second sequence: only its last token sees it
    k[last], v[last] = bad, bad
    out = decode_call(ops, st, q, k, v, lengths, prefixes)
    keep = [i for i in range(10) if i != 4]
    assert torch.equal(bits(out[keep]), bits(want[keep]))
    assert not out[4].isfinite().any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_steps_follow_the_lengths(ops, dtype):
    """A captured decode step: rotary into the cache, then attention, replayed as the device's lengths grow; eager work
    runs between the replays, and each is compared with the eager calls bit for bit."""
    hq, hkv, D, n, slot = 16, 8, 128, 5, 64
    rot = ops.TextRotary(D, 5e6, (24, 20, 20), True, DEV)
    w = 1 + 0.1 * rand((D,), F32, 1)
    base = n * slot
    k, v = rand((base + 300, hkv, D), dtype, 2), rand((base + 300, hkv, D), dtype, 3)
    x = rand((n, (hq + 2 * hkv) * D), dtype, 4)
    q, kn, vn = x[:, :hq * D].view(n, hq, D), x[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D)), x[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
    starts = torch.arange(n, device=DEV) * slot
    lens = torch.tensor([1, 7, 30, 31, 2], dtype=torch.int32, device=DEV)
    pos, rows = (lens - 1).clone(), starts + lens - 1
    pre = [torch.tensor(a, dtype=d, device=DEV) for a, d in (([base], torch.int64), ([290], torch.int32), ([0, n], torch.int32))]

    def step(kc, vc):
        qr, _, _ = ops.qk_norm_rotary(q, kn, vn, w, w, pos, rot, k_cache=kc, v_cache=vc, rows=rows)
        return (ops.decode_attention(qr, kc, vc, starts, lens, max_len=slot),
                ops.prefix_attention(qr, kc, vc, starts, lens, *pre, max_len=slot, max_prefix=290))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k.clone(), v.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    kg, vg = k.clone(), v.clone()
    with torch.cuda.graph(graph):
        got = step(kg, vg)
    ke, ve = k.clone(), v.clone()
    for i in range(4):
        want = step(ke, ve)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got + (kg, vg), want + (ke, ve)):
            assert torch.equal(bits(a), bits(b)), i
        x.copy_(rand(tuple(x.shape), dtype, 50 + i))
        lens += 1
        pos += 1
        rows += 1


def test_called_from_another_device(ops, monkeypatch):
    """The path that makes the tensors' device current first (taken here by saying so once a call)."""
    hq, hkv, D = 8, 2, 64
    q, k, v, seqs = causal_case(hq, hkv, D, BF, [70], [30], seed=41)
    plan, rot = plan_of(ops, seqs, hq, hkv, D, BF), ops.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    w, pos, rows = torch.ones(D, device=DEV), torch.arange(100, dtype=torch.int32, device=DEV), torch.arange(100, device=DEV)
    start, lens = torch.tensor([seqs[0][2]], device=DEV), torch.tensor([100], dtype=torch.int32, device=DEV)

    def calls():
        kc, vc = torch.zeros(100, hkv, D, dtype=BF, device=DEV), torch.zeros(100, hkv, D, dtype=BF, device=DEV)
        n, alone = q.shape[0], ops.qk_norm_rotary(q, k[:q.shape[0]], None, w, w, pos[:q.shape[0]], rot)
        cached = ops.qk_norm_rotary(q, k[:n], v[:n], w, w, pos[:n], rot, k_cache=kc, v_cache=vc, rows=rows[:n])
        return [alone[0], alone[1], *cached, ops.causal_attention(q, k, v, plan)[:70],
                ops.decode_attention(q[:1], k, v, start, lens, max_len=100)]

    want = calls()
    real, said = ops._elsewhere, []
    monkeypatch.setattr(ops, "_elsewhere", lambda device: (said.append(1), len(said) % 2 == 1 or real(device))[1])
    got = calls()
    assert len(said) == 8
    for a, b in zip(got, want):
        assert torch.equal(bits(a), bits(b))


def test_two_streams_at_once(ops):
    """The same plan and caches used from two streams that overlap: each call's workspace is its own."""
    hq, hkv, D = 32, 8, 128
    q, k, v, seqs = causal_case(hq, hkv, D, BF, [500, 60], [1500, 9], seed=4)
    plan = plan_of(ops, seqs, hq, hkv, D, BF)
    lens = torch.tensor([1999], dtype=torch.int32, device=DEV)
    start = torch.tensor([seqs[0][2]], device=DEV)
    qs = [rand(tuple(q.shape), BF, 60 + i, 1.4) for i in range(4)]
    want = [(ops.causal_attention(x, k, v, plan), ops.decode_attention(x[:1], k, v, start, lens, max_len=1999)) for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(3):
        for i, x in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, ops.causal_attention(x, k, v, plan), ops.decode_attention(x[:1], k, v, start, lens, max_len=1999)))
    torch.cuda.synchronize()
    n = sum(s[1] for s in seqs)
    for i, a, b in got:
        assert torch.equal(bits(a[:n]), bits(want[i][0][:n])) and torch.equal(bits(b), bits(want[i][1]))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_then_tokens(ops, pkg, dtype):
    """A layer's work as a chat does it: inject the image rows, prefill two prompts, then decode, then ask twice about the
    first prompt as a shared prefix; against one float64 pass over everything."""
    hq, hkv, D, n_img = 8, 2, 64, 12
    rot = ops.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    qw, kw = 1 + 0.2 * rand((D,), F32, 1), 1 + 0.2 * rand((D,), F32, 2)
    lens = [50, 21]
    hidden = rand((1, sum(lens), (hq + 2 * hkv) * D), dtype, 3)       # stands for the qkv Dense's rows
    tokens = torch.zeros((1, sum(lens)), dtype=torch.int32, device=DEV)
    tokens[0, 5:5 + n_img] = 9
    hidden, mask, _ = pkg.decoder_io.inject_vision(hidden, tokens, rand((n_img, (hq + 2 * hkv) * D), dtype, 4), 9)
    x = hidden[0]
    split = lambda x: (x[:, :hq * D].unflatten(1, (hq, D)), x[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D)),
                       x[:, (hq + hkv) * D:].unflatten(1, (hkv, D)))
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).repeat(3, 1).to(DEV)
    starts = [0, 80]
    R = 160
    kc, vc = torch.full((R, hkv, D), float("nan"), dtype=dtype, device=DEV), torch.full((R, hkv, D), float("nan"), dtype=dtype, device=DEV)
    rows = torch.cat([torch.arange(n) + s for n, s in zip(lens, starts)]).to(DEV)
    q, k, v = split(x)
    qr, _, _ = ops.qk_norm_rotary(q, k, v, qw, kw, pos, rot, k_cache=kc, v_cache=vc, rows=rows)
    plan = ops.CausalPlan(lens, lens, starts, num_heads=hq, num_kv_heads=hkv, head_dim=D, dtype=dtype, device=DEV)
    out = ops.causal_attention(qr, kc, vc, plan)
    seqs = [(0, 50, 0, 50), (50, 21, 80, 21)]
    check_causal(out, qr, kc, vc, seqs, D ** -0.5)
    for step in range(3):                                             # three tokens of both chats
        now = [n + step + 1 for n in lens]
        x = rand((2, (hq + 2 * hkv) * D), dtype, 10 + step)
        q, k, v = split(x)
        p = torch.tensor([a - 1 for a in now], dtype=torch.int32, device=DEV)
        qr, _, _ = ops.qk_norm_rotary(q, k, v, qw, kw, p, rot, k_cache=kc, v_cache=vc,
                                      rows=torch.tensor([s + a - 1 for s, a in zip(starts, now)], device=DEV))
        out = ops.decode_attention(qr, kc, vc, torch.tensor(starts, device=DEV), torch.tensor(now, dtype=torch.int32, device=DEV),
                                   max_len=64)
        check_causal(out, qr, kc, vc, [(i, 1, s, a) for i, (s, a) in enumerate(zip(starts, now))], D ** -0.5)
        assert_rotary(qr, q, qw, p[None].repeat(3, 1), rot)
    # two questions of 2 and 3 tokens that share the first chat's 53 rows; their own rows begin at 110 and 120
    new = [2, 3]
    x = rand((5, (hq + 2 * hkv) * D), dtype, 30)
    q, k, v = split(x)
    p = torch.tensor([53, 54, 53, 54, 55], dtype=torch.int32, device=DEV)
    qr, _, _ = ops.qk_norm_rotary(q, k, v, qw, kw, p, rot, k_cache=kc, v_cache=vc,
                                  rows=torch.tensor([110, 111, 120, 121, 122], device=DEV))
    t = lambda v, d: torch.tensor(v, dtype=d, device=DEV)
    out = ops.prefix_attention(qr, kc, vc, t([110, 120], torch.int64), t(new, torch.int32), t([0], torch.int64), t([53], torch.int32),
                               t([0, 2], torch.int32), max_len=3, max_prefix=53, cu_q=t([0, 2, 5], torch.int32))
    at = 0
    for n, s in zip(new, (110, 120)):
        kk, vv = torch.cat([kc[:53], kc[s:s + n]]), torch.cat([vc[:53], vc[s:s + n]])
        ref = attention_ref(qr[at:at + n], kk, vv, 54 + torch.arange(n, device=DEV), D ** -0.5)
        assert_attention(out[at:at + n], ref, 53 + n)
        at += n
