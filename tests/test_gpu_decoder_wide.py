"""GPU tests of the causal attention in tiles of 256 rows (bf16) where a row's scores run far from those of its first 64 keys,
by which its weights are shifted.

Scores here are powers of two: the scale is ln 2, so that q . k counts octaves (the kernels' softmax runs on powers of two).
Direction 0 holds the level of a key, q is 1 there; the other directions are small. The tolerance is that of the other
attention tests (u = 2^-8, half a step of bf16): a score of D products is off by at most (D + 8) 2^-24 sum|q_i k_i| scale +
4 2^-24 max|s|, a weight relatively by that, numerator and denominator alike; sums over n keys add n 2^-24 each; the weights and
the output are rounded (u each): |error| <= (2 (score error) + 2 n 2^-24 + 2 u) sum w|v| + u |value|.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV, BF = "cuda:0", torch.bfloat16
U = 2.0 ** -8
HQ, HKV = 4, 2


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_attn


def inputs(n, length, D, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((n, HQ, D), generator=g) * 0.25
    k, v = torch.randn((length, HKV, D), generator=g) * 0.25, torch.randn((length, HKV, D), generator=g)
    q[..., 0], k[..., 0] = 1.0, 0.0
    return q, k, v


def check(ops, q, k, v, n, length, tile_rows, joins=None, skip=0):
    """One sequence of `length` keys, the last n of them new; against float64. The first `skip` keys weigh nothing."""
    q, k, v = (x.to(BF).to(DEV) for x in (q, k, v))
    D = q.shape[-1]
    plan = ops.CausalPlan([n], [length], [0], num_heads=HQ, num_kv_heads=HKV, head_dim=D, dtype=BF, device=DEV, tile_rows=tile_rows)
    assert joins is None or (plan.n_joins > 0) == joins
    out = ops.causal_attention(q, k, v, plan, scale=math.log(2.0)).double()
    visible = torch.arange(n, device=DEV)[:, None] + length - n + 1
    mask = torch.arange(skip, length, device=DEV)[None] < visible
    for h in range(HQ):
        qh, kh, vh = q[:, h].double(), k[skip:, h // (HQ // HKV)].double(), v[skip:, h // (HQ // HKV)].double()
        s = torch.where(mask, (qh @ kh.t()) * math.log(2.0), -math.inf)
        mass = torch.where(mask, (qh.abs() @ kh.abs().t()) * math.log(2.0), 0.0)
        w = torch.softmax(s, 1)
        want, A = w @ vh, w @ vh.abs()
        ds = (D + 8) * 2.0 ** -24 * mass.amax(1, keepdim=True) + 4 * 2.0 ** -24 * torch.where(mask, s.abs(), 0.0).amax(1, keepdim=True)
        tol = (2 * ds + 2 * length * 2.0 ** -24 + 2 * U) * A + U * want.abs()
        err = (out[:, h] - want).abs()
        assert (err <= tol).all(), (h, float((err / tol).max()))     # (NaN fails)


LEVELS = [float(j) for j in range(90, 141)] + [j + 0.5 for j in range(118, 128)]


@pytest.mark.parametrize("tile_rows", [128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_late_keys_far_above_the_first_tile(ops, D, tile_rows):
    """Two late keys of one level, in different lanes of their rows: their weights together may be more than a float holds."""
    n, length = 130, 330
    for level in LEVELS:
        q, k, v = inputs(n, length, D, 1)
        k[100, :, 0] = k[100 + 4, :, 0] = level
        k[100, :, 1:], k[104, :, 1:] = 0.0, 0.0                   # exactly alike
        v[100], v[104] = 0.3, 0.4
        check(ops, q, k, v, n, length, tile_rows, joins=False)


def cut_of(ops, n, length, D, tile_rows):
    """The first key tile of each part of the plan's cut tiles."""
    plan = ops.CausalPlan([n], [length], [0], num_heads=HQ, num_kv_heads=HKV, head_dim=D, dtype=BF, device=DEV, tile_rows=tile_rows)
    items = plan.items.cpu()[:plan.n_items]
    assert plan.n_joins > 0
    return sorted({int(it[8]) for it in items if int(it[5]) >= 0})


@pytest.mark.parametrize("tile_rows", [128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_parts_whose_first_tiles_differ(ops, D, tile_rows):
    """A tile cut along its keys: the first part begins low and has a late key of the level that the second part begins with.
    Both have half of each row's weight."""
    n, length = 130, 1630
    first = cut_of(ops, n, length, D, tile_rows)
    for level in LEVELS + [float(j) for j in range(141, 151)]:
        q, k, v = inputs(n, length, D, 2)
        a, b = 64 * first[1] - 9, 64 * first[1] + 3
        k[a, :, 0] = k[b, :, 0] = level
        k[a, :, 1:], k[b, :, 1:] = 0.0, 0.0
        v[a], v[b] = 1.0, -0.75
        check(ops, q, k, v, n, length, tile_rows, joins=True)


@pytest.mark.parametrize("tile_rows", [128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_parts_whose_sums_are_large_together(ops, D, tile_rows):
    """Every part begins low and has a late key of the level: each part's sum is a float, all together may not be."""
    n, length = 130, 1630
    first = cut_of(ops, n, length, D, tile_rows)
    for level in LEVELS:
        q, k, v = inputs(n, length, D, 3)
        for p, t in enumerate(first):
            at = 64 * t + 64 + 5                                   # in the part's second key tile
            k[at, :, 0], k[at, :, 1:] = level, 0.0
            v[at] = 0.25 + 0.125 * p
        check(ops, q, k, v, n, length, tile_rows, joins=True)


@pytest.mark.parametrize("tile_rows", [128, 256])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("level", [0.0, 100.0, -100.0, -126.0, -200.0])
def test_first_tile_of_scores_of_minus_infinity(ops, D, tile_rows, cut, level):
    """The first 64 keys hold -inf (a way to take keys out): their scores are -inf, and the later keys lie at any level."""
    n, length = 130, 1630 if cut else 330
    q, k, v = inputs(n, length, D, 4)
    k[:, :, 0] = level
    k[:64, :, 0] = -math.inf
    check(ops, q, k, v, n, length, tile_rows, joins=cut, skip=64)
    # a row that sees keys of score -inf alone has no answer, and touches no other row
    k[:, :, 0], k[:200, :, 0] = 0.0, -math.inf
    q, k, v = (x.to(BF).to(DEV) for x in (q, k, v))
    plan = ops.CausalPlan([n], [230], [0], num_heads=HQ, num_kv_heads=HKV, head_dim=D, dtype=BF, device=DEV, tile_rows=tile_rows)
    out = ops.causal_attention(q, k, v, plan, scale=math.log(2.0))
    assert out[:100].isnan().all() and out[100:].isfinite().all()
