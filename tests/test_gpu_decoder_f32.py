"""GPU tests of how near the fp32 decode and prefix attention come to float64.

A score is a sum of D products, each addition rounded: relative to its partial sum by 0.41 2^-24 in the root mean square (a
rounding is even over half a step, which is 2^-24 of a value at the lower end of its power of two and half of that at the upper).
Products of independent values grow a partial sum like the root of their number i, so that a chain of n leaves
0.41 2^-24 sqrt(sum_i i) = 0.41 2^-24 n / sqrt 2 of a product's size. For D = 128 in two chains (the fewest these kernels take): sqrt 2 times 64 / sqrt 2, and
11 for their sum, 65; of a score's 11.3, with the factor, 2.4 2^-24. Values of deviation 1.4 make scores of deviation
1.96 sqrt(128 / D) sqrt(D / 128) = 1.96 nats, and a softmax weighs the larger ones, around 1.96^2 = 3.8: a weight is off by
2.4 2^-24 sqrt(1.96^2 + 3.8^2) = 10.3 2^-24, independently for each key, and an output, relative to its size, by as much. Scaling
and shift round by 0.41 2^-24 of up to 8 powers of two, 2.3 2^-24; the power of two, the sums and the output stay below 2^-24
each. Together sqrt(10.3^2 + 2.3^2 + 3) = 10.7 2^-24, 6.4e-7. The limit is 2^-20 = 16 2^-24.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_attn


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq,lengths,prefixes,groups", [
    (16, [2310], [], []), (16, [1000, 1, 3000, 500], [], []),                     # tiles of 16 rows
    (64, [2310, 700], [], []),                                                     # tiles of 32
    (16, [1, 2, 63, 64, 65, 130, 7, 300], [2310, 777], [5, 3]),                   # 16
    (64, [40, 9, 200], [2310], [3]),                                               # 32
    (16, [1 + 5 * i for i in range(40)], [4000], [40])])                           # 128
def test_error_of_fp32_outputs(ops, D, hq, lengths, prefixes, groups):
    hkv, g = 8 if D == 128 else 2, torch.Generator().manual_seed(D + hq)
    hq = hq * hkv // 8
    rand = lambda shape, std: (torch.randn(shape, generator=g) * std).to(DEV)
    rows = sum(lengths) + sum(prefixes)
    q, k, v = rand((len(lengths), hq, D), 1.4), rand((rows, hkv, D), 1.4), rand((rows, hkv, D), 1.0)
    at = [0]
    for n in prefixes + lengths:
        at.append(at[-1] + n)
    pstart, start = at[:len(prefixes)], at[len(prefixes):-1]
    t = lambda x, dt: torch.tensor(x, dtype=dt, device=DEV)
    args = (q, k, v, t(start, torch.int64), t(lengths, torch.int32))
    if prefixes:
        cu = [sum(groups[:i]) for i in range(len(groups) + 1)]
        out = ops.prefix_attention(*args, t(pstart, torch.int64), t(prefixes, torch.int32), t(cu, torch.int32), max_len=max(lengths),
                                   max_prefix=max(prefixes))
    else:
        out = ops.decode_attention(*args, max_len=max(lengths))
    group = [i for i, n in enumerate(groups) for _ in range(n)]
    want = torch.empty(out.shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(lengths):
        pick = torch.arange(start[i], start[i] + n, device=DEV)
        if prefixes:
            p = group[i]
            pick = torch.cat([torch.arange(pstart[p], pstart[p] + prefixes[p], device=DEV), pick])
        for h in range(hq):
            kh, vh = k[pick, h * hkv // hq].double(), v[pick, h * hkv // hq].double()
            want[i, h] = torch.softmax(kh @ q[i, h].double() * D ** -0.5, 0) @ vh
    assert float((out.double() - want).norm() / want.norm()) <= 2.0 ** -20
