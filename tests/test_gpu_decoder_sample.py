"""GPU tests of sample_tokens against a plain form in float64 and whole numbers."""
from fractions import Fraction

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture()
def sample(pkg):
    return pkg.decoder_sample.sample_tokens


def chosen(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, settings rounded to float32 as the operator takes them."""
    x = np.asarray(x, np.float64)
    t, p, f, u = (np.float64(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
        return -1
    order = np.lexsort((np.arange(len(x)), -x))
    if not t > 0 or top_k == 1 or p <= 0 or f > 1:
        return int(order[0])
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        w = np.exp((x - x.max()) / t)
    w = np.rint(np.where(x == -np.inf, 0.0, w) * 2.0 ** 44).astype(np.int64)       # (-infinity / infinity)
    order = order[:top_k] if top_k > 0 else order
    sorted_w = w[order]
    before = np.cumsum(sorted_w) - sorted_w
    keep = (before.astype(np.float64) < p * np.float64(sorted_w.sum())) | (not p < 1)
    keep &= sorted_w.astype(np.float64) >= f * 2.0 ** 44
    kept = np.zeros_like(w)
    kept[order[keep]] = sorted_w[keep]
    upto = np.cumsum(kept)
    u = u if u >= 0 else 0.0
    target = min(u * np.float64(upto[-1]), np.float64(upto[-1] - 1))
    return int(np.argmax(upto.astype(np.float64) > target))


def check(sample, x, u, **settings):
    got = sample(x, u, **settings).cpu().numpy()
    rows = x.float().cpu().numpy()
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v
    for i in range(len(rows)):
        want = chosen(rows[i], u[i].item(), **{k: at(v, i) for k, v in settings.items()})
        assert got[i] == want, (i, got[i], want, {k: at(v, i) for k, v in settings.items()})


def logits(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype).to(DEV), torch.rand(rows, generator=g).to(DEV)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.0), dict(top_k=1),
            dict(top_p=0.0), dict(min_p=1.0), dict(temperature=1.5, top_k=200, top_p=0.8, min_p=0.01), dict(top_k=10 ** 9, top_p=0.5),
            dict(temperature=30.0, top_p=0.7), dict(temperature=0.05, top_p=0.99, top_k=3000)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 1023, 1024, 1025, 4099, 32768])
@pytest.mark.parametrize("settings", SETTINGS)
def test_sizes(sample, dtype, vocab, settings):
    x, u = logits(17, vocab, dtype, vocab)
    check(sample, x, u, **settings)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 2, 40, 300])
@pytest.mark.parametrize("vocab", [151936, 151935, 262144])
def test_whole_vocabularies_and_settings_of_each_row(sample, dtype, rows, vocab):
    """Every mixture of settings in one call; 300 rows: more than a row for each compute unit."""
    x, u = logits(rows, vocab, dtype, rows)
    x = x * torch.linspace(0.2, 2.5, rows, device=DEV)[:, None].to(dtype)
    g = torch.Generator().manual_seed(rows + 1)
    pick = lambda values, dt: torch.tensor(values, dtype=dt)[torch.randint(0, len(values), (rows,), generator=g)].to(DEV)
    keep = torch.randperm(rows, generator=g)[:40].to(DEV)                # (the reference sorts on the host)
    settings = dict(temperature=pick([0.0, 0.3, 0.8, 1.0, 2.0], F32), top_k=pick([0, 0, 1, 20, 50, 1000, 5000, 100000], torch.int32),
                    top_p=pick([0.2, 0.9, 0.95, 1.0], F32), min_p=pick([0.0, 0.0, 0.02, 0.5], F32))
    got = sample(x, u, **settings)
    few = {k: v[keep].contiguous() for k, v in settings.items()}
    assert torch.equal(sample(x[keep], u[keep].contiguous(), **few), got[keep])
    check(sample, x[keep], u[keep].contiguous(), **few)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [3000, 151936])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=700), dict(top_p=0.37), dict(top_k=90001, top_p=0.25), dict(min_p=0.5, top_p=0.9)])
def test_equal_logits(sample, dtype, vocab, settings):
    """Ties go to the lowest index: rows of one value, of two, of whole numbers, of zeros of both signs."""
    g = torch.Generator().manual_seed(5)
    x = torch.stack([torch.full((vocab,), 2.5), torch.where(torch.rand(vocab, generator=g) < 0.4, 1.0, 1.5),
                     torch.randint(-3, 4, (vocab,), generator=g).float(), torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0),
                     torch.randint(-40, 1, (vocab,), generator=g).float()]).to(dtype).to(DEV)
    check(sample, x, torch.tensor([0.999, 0.31, 0.62, 0.5, 0.97], device=DEV), **settings)
    check(sample, x, torch.tensor([0.0, 0.0, 0.0, 1e-6, 0.0], device=DEV), **settings)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("vocab", [700, 20011])
def test_masked_tokens_and_rows_without_any(sample, dtype, settings, vocab):
    x, u = logits(9, vocab, dtype, 3)
    inf, nan = float("inf"), float("nan")
    x[0, ::2] = -inf
    x[1, :] = -inf
    x[2, :], x[2, 611] = -inf, -4.0
    x[3, vocab - 1] = nan
    x[4, 17] = inf
    x[5, :650] = -inf
    x[6, :], x[6, 5], x[6, vocab - 2] = -inf, nan, 1.0
    x[7, :] = torch.finfo(dtype).min                                     # a mask of the lowest value alone
    x[8, 3:] = torch.finfo(dtype).min
    check(sample, x, u, **settings)
    got = sample(x, u, **settings).cpu()
    assert got[1] == -1 and got[2] == 611 and got[3] == -1 and got[4] == -1 and got[6] == -1


@pytest.mark.parametrize("temperature", [1e-45, 1e-30, 1e30, 3e38, float("inf"), float("nan"), -1.0])
def test_far_temperatures(sample, temperature):
    """Given on the device, where nothing can refuse them: the smallest weigh the largest logit alone, the largest all the same."""
    x, u = logits(3, 5000, F32, 8)
    x[1, ::3] = -float("inf")
    x[2] = torch.linspace(-3e38, 3e38, 5000, dtype=torch.float64).float().to(DEV)
    t = torch.full((3,), temperature, device=DEV)
    for settings in (dict(), dict(top_p=0.6), dict(top_k=77)):
        check(sample, x, u, temperature=t, **settings)


def test_random_numbers_at_the_ends(sample):
    """0 takes the first kept token, what is not below 1 the last, what is below 0 or no number counts as 0."""
    x, _ = logits(7, 3001, F32, 4)
    x[:] = x[0]
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan"), 0.5], device=DEV)
    for settings in (dict(), dict(top_k=9), dict(top_p=0.7), dict(top_k=2000, top_p=0.9, min_p=0.001)):
        got = sample(x, u, **settings).tolist()
        assert got[4] == got[5] == got[0] == chosen(x[0].cpu().numpy(), 0.0, **settings)
        assert got[2] == got[3] == chosen(x[0].cpu().numpy(), 1.0, **settings)
        assert got[1] == chosen(x[0].cpu().numpy(), 1 - 2.0 ** -24, **settings)
        assert got[6] == chosen(x[0].cpu().numpy(), 0.5, **settings)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_rows_anywhere(sample, dtype, offset):
    """Rows of any stride and alignment, between values that must not be read as theirs."""
    rows, vocab = 5, 4099
    store = torch.full((rows, vocab + 37), 50.0, dtype=dtype, device=DEV)
    x, u = logits(rows, vocab, dtype, 6)
    view = store[:, offset:offset + vocab]
    view.copy_(x)
    for settings in (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.9), dict(temperature=0.0)):
        assert torch.equal(sample(view, u, **settings), sample(x, u, **settings))
        check(sample, view, u, **settings)
    one = x[:1].expand(3, vocab)                                         # one row three times
    assert sample(one, u[:1].expand(3).contiguous(), top_k=5).unique().numel() == 1


def test_frequencies(sample):
    """Evenly spaced random numbers give each kept token its share of them, to one."""
    n = 4096
    x = torch.randn(40, generator=torch.Generator().manual_seed(1)).to(DEV)
    u = (torch.arange(n, device=DEV) + 0.5) / n
    got = torch.bincount(sample(x.expand(n, 40), u, top_k=12, temperature=0.9), minlength=40).double().cpu()
    p = torch.softmax(x.double().cpu() / np.float64(np.float32(0.9)), 0)
    p[x.cpu().argsort(descending=True)[12:]] = 0
    assert ((got - p / p.sum() * n).abs() <= 1 + 1e-6).all()


def test_out_and_streams(sample):
    x, u = logits(64, 20000, BF, 2)
    want = sample(x, u, top_p=0.9)
    out = torch.zeros(64, dtype=torch.int64, device=DEV)
    assert sample(x, u, top_p=0.9, out=out) is out and torch.equal(out, want)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(sample(x, u, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert sample(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("settings", [dict(top_p=0.6), dict(top_p=0.999), dict(top_k=1500), dict(top_k=2700, top_p=0.7), dict(top_p=0.9, min_p=0.5)])
@pytest.mark.parametrize("unit", [1.0, 1e30, 1e-37])
def test_cuts_that_leave_some_of_each_segment(sample, dtype, settings, unit):
    """Segments of 1024 tokens of which from none to all reach the cut, also where logits and temperature are far from 1."""
    g = torch.Generator().manual_seed(8)
    x = torch.full((9 * 1024 + 37,), -12.0)
    for segment, left in enumerate((513, 0, 1, 64, 512, 65, 1024, 511, 63)):
        at = segment * 1024 + torch.randperm(1024, generator=g)[:left]
        x[at] = torch.rand(left, generator=g)
    x = (x * unit).to(dtype).to(DEV)[None].repeat(24, 1)
    check(sample, x, torch.rand(24, generator=g).to(DEV), temperature=unit, **settings)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [513, 600, 3001, 151936, 262144])
@pytest.mark.parametrize("spread", [0.0, 0.01])
def test_random_numbers_of_one_and_more_on_flat_rows(sample, dtype, vocab, spread):
    """What is not below 1 counts as just below it, and takes the kept token of the highest index, also where the weights' sum is far
    beyond 2^53 (512 equal tokens reach it) and one less than it is the same double."""
    x, _ = logits(1, vocab, dtype, vocab, spread)
    row = x[0].double().cpu().numpy()
    order = np.lexsort((np.arange(vocab), -row))
    w = [int(v) for v in np.rint(np.exp(row - row.max()) * 2.0 ** 44)]   # (Python's integers: sums up to 2^62)
    for settings in (dict(), dict(top_p=0.9), dict(top_k=511), dict(min_p=0.5), dict(top_k=vocab // 2 + 1, top_p=0.75), dict(top_p=0.5, min_p=0.25)):
        kept = order[:settings.get("top_k", vocab)].tolist()
        if "top_p" in settings:
            whole, upto, n = sum(w[i] for i in kept), 0, 0
            while n < len(kept) and upto < float(np.float32(settings["top_p"])) * whole:
                upto += w[kept[n]]
                n += 1
            kept = kept[:n]
        u = torch.tensor([1.0, 7.0, float("inf"), 0.0, -1.0, float("nan")], device=DEV)
        got = sample(x.expand(6, vocab), u, **settings).tolist()
        assert got == [max(kept)] * 3 + [min(kept)] * 3, settings


def on_borders(temperature, count, seed):
    """(top, x) of float32 whose distance in 32nds of a power of two, (top - x) 32 / (T ln 2), lies between two whole numbers: in the middle
    once the product is rounded, a little to one side of it before, and so that the two would come to different ones."""
    rng, found = np.random.default_rng(seed), []
    scale = np.float64(32 / 0.69314718055994530942) / np.float64(np.float32(temperature))
    while len(found) < count:
        half = int(rng.integers(1, 500)) + 0.5
        top = np.float32(half / scale)
        x = np.float32(np.float64(top) - half / scale)
        d = np.float64(top) - np.float64(x)
        side = Fraction(float(d)) * Fraction(float(scale)) - Fraction(half)
        if x != 0 and d * scale == half and side != 0 and np.rint(half) != half + (0.5 if side > 0 else -0.5):
            found.append((float(top), float(x)))
    return found


def border_rows(temperature, copies, seed):
    """Rows of one top, `copies` tokens at its border and lower ones, in any order, and a top-p that falls among the copies."""
    rng, rows, top_p = np.random.default_rng(seed), [], []
    for top, x in on_borders(temperature, 24, seed):
        row = np.concatenate([[top], np.full(copies, x), top - 16.5 * temperature - rng.random(40)])
        rows.append(row[rng.permutation(len(row))])
        w = np.exp((x - top) / temperature) * copies
        top_p.append((1 + w * 0.55) / (1 + w))
    return torch.tensor(np.array(rows), dtype=F32, device=DEV), torch.tensor(top_p, dtype=F32, device=DEV)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("copies", [1, 3, 200, 5000])
def test_no_token_outside_the_vocabulary(sample, temperature, copies):
    x, top_p = border_rows(temperature, copies, 3)
    for u in (0.0, 0.5, 0.99, 1.0):
        for settings in (dict(top_p=top_p), dict(top_k=1 + (copies + 1) // 2), dict(top_k=2 + copies, top_p=top_p)):
            got = sample(x, torch.full((len(x),), u, device=DEV), temperature=temperature, **settings)
            assert int(got.min()) >= 0 and int(got.max()) < x.shape[1]


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("copies", [1, 3, 200, 5000])
def test_logits_on_the_border_of_two_bins(sample, temperature, copies):
    """Every pass over a row has to come to the same bin, or tokens at the cut are lost or counted twice."""
    x, top_p = border_rows(temperature, copies, 3)
    for u in (0.02, 0.47, 0.73, 0.9, 0.97):
        us = torch.full((len(x),), u, device=DEV)
        for settings in (dict(top_p=top_p), dict(top_k=1 + (copies + 1) // 2), dict(top_k=2 + copies, top_p=top_p), dict(top_p=0.999, min_p=1e-5)):
            check(sample, x, us, temperature=temperature, **settings)
    pair = torch.tensor([[1.7003766, -4.748171e-08]], device=DEV)        # 78 and a half, 5e-15 more
    check(sample, pair, torch.tensor([0.97], device=DEV), top_p=0.9)
