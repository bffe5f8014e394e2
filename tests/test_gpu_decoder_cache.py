"""GPU tests of the paged 4-bit cache: what its pages stand for, against float64; attention over it; its pages' borders, strides, streams,
graphs and devices; and a decoder layer's run over it."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from .test_gpu_decoder_attn import assert_attention, assert_rotary, attention_ref, bits, rand  # noqa: E402

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HEADS = [(16, 8, 128), (32, 8, 128), (14, 2, 64), (4, 4, 64), (5, 1, 128)]
# the numbers, even codes first: the first of equal distances is the even code
NUMBERS = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64)


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_cache


def word(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def packed(x):
    """(what x [..., D] in float64 stands for in 4 bits, how far its nearest border between two codes is, in scales)."""
    g = x.double().unflatten(-1, (-1, 64))
    top = g.abs().amax(-1, keepdim=True)
    s = (top / 6).float().bfloat16()
    s = torch.where(top.isfinite() & s.isfinite(), s, float("nan")).double()
    numbers = NUMBERS.to(x.device)
    best = (g.abs()[..., None] - numbers * s[..., None]).abs().argmin(-1)
    y = torch.copysign(numbers[best] * s, g)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    margin = ((g.abs() / s)[..., None] - borders).abs().amin(-1)
    return y.flatten(-2), margin.flatten(-2)


class Chats:
    """Sequences whose pages lie anywhere in a cache full of NaN, the table's other entries outside the cache."""

    def __init__(self, ops, lengths, page_rows, hkv, D, new=None, seed=0, spare=2):
        self.lengths, self.page_rows = list(lengths), page_rows
        self.new = [1] * len(lengths) if new is None else list(new)
        need = [-(-v // page_rows) for v in lengths]
        total = sum(need) + spare
        order = np.random.default_rng(seed).permutation(total)
        table = np.full((len(lengths), max(need + [1]) + 1), 1 << 30, np.int32)
        table[:, ::2] = -1
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.cache = ops.PagedCache(total, page_rows, hkv, D, device=DEV)
        self.cache.data.fill_(0xff)                                      # codes -6, scales NaN
        self.table, self.k_len = torch.from_numpy(table).to(DEV), word(self.lengths)
        self.cu_q = None if new is None else word([0] + np.cumsum(self.new).tolist())
        self.ops = ops

    def fill(self, k, v):
        """Every token of every sequence, in order."""
        self.ops.append_paged(k, v, self.cache, self.table, self.k_len, cu_q=word([0] + np.cumsum(self.lengths).tolist()))

    def rows(self, dtype=F32, first=None):
        begin = [0] * len(self.lengths) if first is None else first
        n = [b - a for a, b in zip(begin, self.lengths)]
        start = word([0] + np.cumsum(n)[:-1].tolist(), torch.int64)
        k = torch.full((sum(n), self.cache.num_kv_heads, self.cache.head_dim), 77.0, dtype=dtype, device=DEV)
        v = torch.full_like(k, 77.0)
        return self.ops.unpack_paged(self.cache, self.table, self.k_len, start, k, v, max_len=max(n + [0]),
                                     first=None if first is None else word(begin))


# ---------------------------------------------------------------------------------------------
# what pages stand for
# ---------------------------------------------------------------------------------------------
LENGTHS = [([1], 16), ([5, 16, 17, 33], 16), ([300, 1, 64], 64), ([4097], 4096), ([130, 0, 31], 32)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hkv,D", [(8, 128), (3, 64), (11, 128), (1, 64)])
@pytest.mark.parametrize("lengths,page_rows", LENGTHS)
def test_appended_as_they_are(ops, dtype, hkv, D, lengths, page_rows):
    """Exactly the nearest numbers; read back in float32 exactly, in bfloat16 rounded once; and what was read back, appended again,
    gives the same bytes."""
    chats = Chats(ops, lengths, page_rows, hkv, D)
    n = sum(lengths)
    k, v = rand((n, hkv, D), dtype, 1, 3.0), rand((n, hkv, D), dtype, 2, 0.01)
    chats.fill(k, v)
    got = chats.rows()
    for x, y in zip((k, v), got):
        assert torch.equal(y.double(), packed(x)[0])
    for x, y in zip(got, chats.rows(BF)):
        assert torch.equal(x.to(BF), y)
    before = chats.cache.data.clone()
    chats.fill(*got)
    assert torch.equal(chats.cache.data, before)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_ties_and_borders(ops, dtype, D):
    """Values on the borders between two codes go to the even one, their neighbours to their own side."""
    s = 0.4375                                                           # bf16; max = 6 s
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64) * s
    ulp = 2.0 ** -8 if dtype == BF else 2.0 ** -23
    x = torch.cat([edge, edge * (1 - ulp), edge * (1 + ulp), torch.tensor([6 * s, 0.0, -0.0, 1e-30], dtype=torch.float64)])
    x = torch.cat([x, -x, torch.zeros(14, dtype=torch.float64)])
    row = x.to(dtype).to(DEV).repeat(D // 64).expand(3, 2, D).contiguous()
    chats = Chats(ops, [3], 16, 2, D)
    chats.fill(row, -row)
    k, v = chats.rows()
    assert torch.equal(k.double(), packed(row)[0]) and torch.equal(v, -k)
    want = torch.tensor([0, 1, 1, 2, 2, 4, 4], dtype=torch.float64) * s
    if dtype == F32:
        assert torch.equal(k[0, 0, :7].double().cpu(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_not_finite_or_far(ops, dtype, D):
    """A group with a NaN or an infinity stands for NaN, the others of its head and token are untouched; zeros, the smallest and the
    largest values."""
    x = rand((20, 2, D), dtype, 3)
    x[1, 0, 5], x[2, 1, D - 1], x[3, 0, 0] = float("nan"), float("inf"), float("-inf")
    x[4, 0], x[5, 1], x[6, 0] = 0.0, 3.0e38, 1e-36
    x[7, 0, :64] = 2.0 ** -120
    chats = Chats(ops, [20], 32, 2, D)
    chats.fill(x, x.flip(0))
    k, v = chats.rows()
    for y, z in ((k, x), (v, x.flip(0))):
        want = packed(z)[0]
        assert torch.equal(y.double().isnan(), want.isnan()) and torch.equal(y.double().nan_to_num(7.0), want.nan_to_num(7.0))
    assert k[1, 0, :64].isnan().all() and k[2, 1, D - 64:].isnan().all() and int(k.isnan().sum()) == 3 * 64


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("lengths,new,page_rows", [([7, 1, 300, 64], None, 64), ([5, 90, 20], [3, 81, 0], 16), ([1500], [1500], 128),
                                                   ([64] * 70, None, 32)])
def test_norm_rotary_into_pages(ops, pkg, dtype, hq, hkv, D, lengths, new, page_rows):
    """q within qk_norm_rotary's bound; keys as the float64 formula's nearest numbers (where that is 1e-10 of a scale from a
    border, hundreds of times the error of fp64 angles of positions up to 2^20, either side), values exactly."""
    chats = Chats(ops, lengths, page_rows, hkv, D, new)
    n = sum(chats.new)
    q, k, v = rand((n, hq, D), dtype, 1, 1.7), rand((n, hkv, D), dtype, 2, 1.7), rand((n, hkv, D), dtype, 3)
    qw, kw = 1 + 0.2 * rand((D,), F32, 4), 1 + 0.2 * rand((D,), F32, 5)
    section = (24, 20, 20) if D == 128 else (12, 10, 10)
    rot = pkg.decoder_attn.TextRotary(D, 5e6, section, True, DEV)
    pos = torch.randint(0, 1 << 20, (3, n), generator=torch.Generator().manual_seed(6)).to(torch.int32).to(DEV)
    got = ops.qk_norm_rotary_paged(q, k, v, qw, kw, pos, rot, chats.cache, chats.table, chats.k_len, cu_q=chats.cu_q)
    # (not bit for bit qk_norm_rotary's: each kernel's products and sums are joined as its compiler sees fit; the bound is that one's)
    assert_rotary(got, q, qw, pos, rot)
    first = [a - b for a, b in zip(chats.lengths, chats.new)]
    gk, gv = chats.rows(first=first)
    assert torch.equal(gv.double(), packed(v)[0])
    half = D // 2
    j = torch.arange(half, device=DEV)
    axis = torch.where(j < 3 * word(section)[j % 3], j % 3, 0)
    angle = pos.double()[axis].t() * (5e6 ** (-2.0 * j.double() / D))
    x = k.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * kw.double()
    a, b, c, s = x[..., :half], x[..., half:], angle.cos()[:, None], angle.sin()[:, None]
    y, margin = packed(torch.cat([a * c - b * s, b * c + a * s], -1))
    clear = margin > 1e-10
    assert (~clear).float().mean() < 1e-6
    assert torch.equal(gk.double()[clear], y[clear])
    if dtype == BF:                                                      # rows and heads of any stride, q in place
        other = Chats(ops, lengths, page_rows, hkv, D, new)
        qkv = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
        qs = qkv[:, :hq * D].unflatten(1, (hq, D))
        ks, vs = qkv[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D)), qkv[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
        back = ops.qk_norm_rotary_paged(qs, ks, vs, qw, kw, pos, rot, other.cache, other.table, other.k_len, cu_q=other.cu_q, q_out=qs)
        assert back.data_ptr() == qkv.data_ptr() and torch.equal(bits(qs.contiguous()), bits(got))
        assert torch.equal(other.cache.data, chats.cache.data)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_tokens_that_have_no_place(ops, pkg, dtype, D):
    """Tokens in pages outside the cache, before a sequence's start, beyond its line of the table or of no sequence are dropped; their
    rows of q_out are written, but for those of no sequence; nothing else changes."""
    hkv, hq, R = 2, 4, 16
    table = word([[0, 7], [-1, 1], [2, 2 ** 31 - 1], [3, 4]])
    cache = ops.PagedCache(6, R, hkv, D, device=DEV)
    k_len, cu = word([40, 20, 17, 1]), word([2, 12, 18, 20, 23])         # new: 10, 6, 2, 3
    n = 26
    q, k, v = rand((n, hq, D), dtype, 1), rand((n, hkv, D), dtype, 2), rand((n, hkv, D), dtype, 3)
    w, pos = torch.ones(D, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    rot = pkg.decoder_attn.TextRotary(D, 1e4, (D // 2, 0, 0), False, DEV)
    out = torch.full_like(q, 9.0)
    ops.qk_norm_rotary_paged(q, k, v, w, w, pos, rot, cache, table, k_len, cu_q=cu, q_out=out)
    assert_rotary(out[2:23], q[2:23], w, pos[2:23].repeat(3, 1), rot)
    assert bool((out[:2] == 9).all()) and bool((out[23:] == 9).all())
    ops.append_paged(k, v, cache, table, k_len, cu_q=cu)
    # written: sequence 1's tokens 16..19 (page 1), sequence 2's token 15 (page 2) and not 16, sequence 3's token 0 (page 3) and not -2, -1;
    # sequence 0's 30, 31 lie in page 7, 32..39 beyond the table
    out = [torch.full((64, hkv, D), 5.0, device=DEV) for _ in range(2)]
    ops.unpack_paged(cache, word([[0], [1], [2], [3]]), word([16] * 4), word([0, 16, 32, 48], torch.int64), *out, max_len=16)
    used = torch.zeros(64, dtype=torch.bool, device=DEV)
    used[16:20] = used[47] = used[48] = True
    for x, src in zip(out, (k, v)):
        assert bool((x[~used] == 0).all())
        assert torch.equal(x[used].double(), packed(torch.cat([src[14:18], src[18:19], src[22:23]]))[0])
    assert bool((cache.data[[0, 4, 5]] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_unpack_rows_and_ranges(ops, dtype):
    """Ranges that begin and end inside pages, rows of other strides, rows outside, pages of none, lengths other than the hint."""
    hkv, D = 3, 128
    chats = Chats(ops, [100, 37, 64, 0, 5], 32, hkv, D, seed=3)
    n = sum(chats.lengths)
    k, v = rand((n, hkv, D), F32, 1), rand((n, hkv, D), F32, 2)
    chats.fill(k, v)
    want = [packed(x)[0].float().to(dtype) for x in (k, v)]
    first, start = [17, 0, 63, 0, 9], [3, 90, 125, 40, 50]
    table = chats.table.clone()
    table[1, 1] = -5                                                     # tokens 32..36
    for hint in (0, 1, 100, 5000):
        store = torch.full((2, hkv, 130, D), 5.0, dtype=dtype, device=DEV)   # [heads, rows, dim] views
        x, y = (s.transpose(0, 1) for s in store)
        ops.unpack_paged(chats.cache, table, chats.k_len, word(start, torch.int64), x, y, max_len=hint, first=word(first))
        for got, w in zip((x, y), want):
            ref = torch.full((130, hkv, D), 5.0, dtype=dtype, device=DEV)
            ref[3:86] = w[17:100]
            ref[90:122] = w[100:132]
            ref[122:127] = float("nan")
            ref[125] = w[137 + 63]
            same = (got == ref) | (got.isnan() & ref.isnan())
            same[125:127] = True                                         # (two sequences' rows)
            assert bool(same.all())
    x, y = (torch.full((10, hkv, D), 5.0, dtype=dtype, device=DEV) for _ in range(2))
    ops.unpack_paged(chats.cache, chats.table, chats.k_len, word([-95, 8, 2 ** 40, -2 ** 62, 10], torch.int64), x, y, max_len=100)
    for got, w in zip((x, y), want):
        assert torch.equal(got[:5], w[95:100]) and torch.equal(got[8:], w[100:102]) and bool((got[5:8] == 5).all())


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def check_attention(out, chats, q, k, v, scale):
    at = row = 0
    for n, length in zip(chats.new, chats.lengths):
        if n:
            visible = (torch.arange(n, device=DEV) + length - n + 1).clamp_min(0)
            ref = attention_ref(q[at:at + n], k[row:row + length], v[row:row + length], visible, scale)
            # Values in 4 bits are often exactly 0, so that an output may be a sum of the smallest weights alone, which the bound below takes
            # for relative ones. A weight under 2^-126 of a part's running maximum may be lost (fp32 and bf16 hold no less): the maximum
            # lies at most 2^8 under the largest score, sums of weights are 1 at least, and a part joined with a factor under
            # 2^-126 loses at most 2^8 length times it; so at most length 2^-126 2^8 2^8 (max|v| + 6) in all, codes up to 6.
            lost = length * 2.0 ** -110 * (v.abs().max().item() + 6) if length else 0.0
            gone = (out[at:at + n].double() - ref[0]).abs() <= lost
            assert_attention(torch.where(gone, 0.0, out[at:at + n]), (torch.where(gone, 0.0, ref[0]), *ref[1:]), length)
        at, row = at + n, row + length


def filled(ops, lengths, page_rows, hkv, D, new=None, seed=0, **kw):
    chats = Chats(ops, lengths, page_rows, hkv, D, new, seed, **kw)
    n = sum(lengths)
    chats.fill(rand((n, hkv, D), F32, seed + 1, 1.4), rand((n, hkv, D), F32, seed + 2))
    return chats, *chats.rows()


ATTEND = [  # lengths, new tokens (None: one each), rows a page
    ([1], None, 16), ([9001], None, 64), ([0, 1, 2, 15, 16, 17, 31, 32, 33, 1000, 0], None, 16), ([5, 40, 200, 3], [3, 1, 0, 5], 32),
    ([300, 2], [40, 9], 128), ([17] * 70, None, 64), ([130] * 300, None, 16), ([700, 64, 129], [5, 2, 16], 4096)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq,hkv,D", HEADS + [(40, 1, 128)])
@pytest.mark.parametrize("lengths,new,page_rows", ATTEND)
def test_attention(ops, dtype, hq, hkv, D, lengths, new, page_rows):
    chats, k, v = filled(ops, lengths, page_rows, hkv, D, new)
    q = rand((sum(chats.new), hq, D), dtype, 9, 1.4)
    for scale in (None, 0.3):
        out = ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=max(lengths), cu_q=chats.cu_q, scale=scale)
        check_attention(out, chats, q, k, v, scale or D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hint", [1, 64, 100000])
def test_lengths_other_than_the_hint(ops, dtype, hint):
    chats, k, v = filled(ops, [2000, 3, 700], 64, 2, 64, seed=4)
    q = rand((3, 8, 64), dtype, 9, 1.4)
    check_attention(ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=hint), chats, q, k, v, 0.125)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences(ops, dtype, D):
    lengths = [1 + (37 * i) % 90 for i in range(1100)]
    chats, k, v = filled(ops, lengths, 32, 2, D, seed=5)
    q = rand((1100, 4, D), dtype, 9, 1.4)
    check_attention(ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=90), chats, q, k, v, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_far_apart(ops, dtype, D):
    """Maxima that rise along the keys by far more than an exponent's range, and scores in the thousands."""
    hkv, n = 2, 700
    chats = Chats(ops, [n], 64, hkv, D)
    k = rand((n, hkv, D), F32, 1) * torch.linspace(0.1, 60, n, device=DEV)[:, None, None]
    chats.fill(k, rand((n, hkv, D), F32, 2))
    k, v = chats.rows()
    q = rand((1, 4, D), dtype, 3, 3.0)
    check_attention(ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=n), chats, q, k, v, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_state_that_is_wrong_comes_out_nan(ops, dtype, D):
    """Lengths below none or beyond the table, and pages outside the cache: NaN for the tokens that see them, the others as before."""
    hkv, hq = 2, 6
    lengths, new = [70, 33, 20, 90, 500], [1, 2, 1, 3, 1]
    chats, k, v = filled(ops, lengths, 16, hkv, D, new, seed=6)
    q = rand((8, hq, D), dtype, 9, 1.4)
    call = lambda table, lens: ops.paged_attention(q, chats.cache, table, lens, max_len=500, cu_q=chats.cu_q)
    good = call(chats.table, chats.k_len)
    lens = chats.k_len.clone()
    lens[0], lens[2] = -1, 16 * chats.table.shape[1] + 1
    got = call(chats.table, lens)
    assert got[0].isnan().all() and got[3].isnan().all()
    # (other lengths cut the line of keys elsewhere, and sums are joined elsewhere: float64 tells, not the bits)
    check_attention(torch.where(torch.tensor([1, 0, 0, 1, 0, 0, 0, 0], device=DEV).bool()[:, None, None], good, got), chats, q, k, v, D ** -0.5)
    table = chats.table.clone()
    table[0, 2], table[1, 2], table[4, 0] = -1, chats.cache.n_pages, -(1 << 31)
    table[3, 5] = 1 << 30                                                # its tokens 80..89, of which the first new one, 87, is one
    got = call(table, chats.k_len)
    assert got[0].isnan().all() and got[4:].isnan().all() and got[3].equal(good[3])
    assert got[2].isnan().all() and torch.equal(bits(got[1]), bits(good[1]))   # sequence 1's key 32 is seen by its last token alone


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_cache_without_pages(ops, dtype):
    cache = ops.PagedCache(0, 16, 2, 64, device=DEV)
    table, q = word([[0], [0]]), rand((2, 4, 64), dtype, 1)
    out = ops.paged_attention(q, cache, table, word([0, 3]), max_len=3)
    assert bool((out[0] == 0).all()) and out[1].isnan().all()
    ops.append_paged(rand((2, 2, 64), dtype, 2), rand((2, 2, 64), dtype, 3), cache, table, word([1, 3]))
    k, v = (torch.zeros(3, 2, 64, dtype=dtype, device=DEV) for _ in range(2))
    ops.unpack_paged(cache, table, word([0, 3]), word([0, 0], torch.int64), k, v, max_len=3)
    assert k.isnan().all() and v.isnan().all()


def test_nothing_to_do(ops, pkg):
    cache = ops.PagedCache(2, 16, 2, 64, device=DEV)
    none, table = word([]), torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    empty = torch.empty(0, 2, 64, device=DEV)
    assert ops.paged_attention(empty, cache, table, none, max_len=0).shape == (0, 2, 64)
    ops.append_paged(empty, empty, cache, table, none)
    ops.unpack_paged(cache, table, none, none.long(), empty, empty, max_len=0)
    # sequences without new tokens: rows of q behind them are left alone
    out = torch.full((3, 4, 64), 3.0, device=DEV)
    ops.paged_attention(rand((3, 4, 64), F32, 1), cache, word([[0], [1]]), word([5, 0]), max_len=5, cu_q=word([1, 1, 2]), out=out)
    assert bool((out[[0, 2]] == 3).all()) and bool((out[1] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_strides_and_wide_tables(ops, dtype):
    chats, k, v = filled(ops, [70, 300, 9], 32, 4, 128, seed=7)
    q = rand((3, 12, 128), dtype, 9, 1.4)
    want = ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=300)
    wide = torch.full((6, chats.table.shape[1] + 5), 1 << 29, dtype=torch.int32, device=DEV)
    wide[::2, 3:3 + chats.table.shape[1]] = chats.table
    store = torch.full((12, 5, 136), 4.0, dtype=dtype, device=DEV)
    out = store.transpose(0, 1)[1:4, :, :128]
    qs = torch.cat([q, q], 2)[:, :, :128]
    got = ops.paged_attention(qs, chats.cache, wide[::2, 3:3 + chats.table.shape[1]], chats.k_len, max_len=300, out=out)
    assert torch.equal(bits(got.contiguous()), bits(want))
    out.fill_(4.0)
    assert bool((store == 4).all())


def test_offsets_past_32_bits(ops):
    """A cache of more than 4 GiB: pages at its end, written, read back and attended to."""
    hkv, D, R = 8, 128, 256
    n_pages = (5 << 30) // (hkv * 16 * 2176) + 1
    cache = ops.PagedCache(n_pages, R, hkv, D, device=DEV)
    assert cache.data.numel() > 5 << 30
    table = word([[n_pages - 1, n_pages - 2, 0]])
    k, v = rand((600, hkv, D), BF, 1), rand((600, hkv, D), BF, 2)
    ops.append_paged(k, v, cache, table, word([600]), cu_q=word([0, 600]))
    gk, gv = (torch.empty(600, hkv, D, device=DEV) for _ in range(2))
    ops.unpack_paged(cache, table, word([600]), word([0], torch.int64), gk, gv, max_len=600)
    assert torch.equal(gk.double(), packed(k)[0]) and torch.equal(gv.double(), packed(v)[0])
    q = rand((1, 32, D), BF, 3, 1.4)
    out = ops.paged_attention(q, cache, table, word([600]), max_len=600)
    assert_attention(out, attention_ref(q, gk, gv, word([600]), D ** -0.5), 600)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_nothing_is_taken_from_what_a_workspace_held(ops, monkeypatch, dtype, D):
    chats, k, v = filled(ops, [700, 0, 33, 2], 16, 2, D, [5, 1, 2, 1], seed=8)
    q = rand((9, 8, D), dtype, 9, 1.4)
    call = lambda: ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=700, cu_q=chats.cu_q)
    want = call()
    monkeypatch.setattr(ops, "_workspace", lambda n, q: torch.full((n,), 0xff, dtype=torch.uint8, device=q.device))
    assert torch.equal(bits(call()), bits(want))


# ---------------------------------------------------------------------------------------------
# graphs, streams, devices
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_steps_follow_the_lengths(ops, pkg, dtype):
    """A captured step (append, attention, read back, the next token), replayed as lengths grow into new pages and settings change;
    each replay is compared with the eager calls bit for bit."""
    hq, hkv, D, n = 16, 8, 128, 5
    rot = pkg.decoder_attn.TextRotary(D, 5e6, (24, 20, 20), True, DEV)
    w = 1 + 0.1 * rand((D,), F32, 1)
    x = rand((n, (hq + 2 * hkv) * D), dtype, 4)
    q, k, v = x[:, :hq * D].view(n, hq, D), x[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D)), x[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
    table = torch.arange(n * 4, dtype=torch.int32, device=DEV).view(n, 4).clone()
    lens = word([1, 15, 16, 31, 2])
    pos, start, u = (lens - 1).clone(), torch.arange(n, device=DEV) * 64, torch.rand(n, device=DEV)
    head = rand((hq * D, 500), dtype, 6, 0.05)
    top_p, top_k = torch.full((n,), 0.9, device=DEV), torch.full((n,), 40, dtype=torch.int32, device=DEV)

    def step(cache):
        qr = ops.qk_norm_rotary_paged(q, k, v, w, w, pos, rot, cache, table, lens)
        out = ops.paged_attention(qr, cache, table, lens, max_len=64)
        rows = [torch.zeros(n * 64, hkv, D, dtype=dtype, device=DEV) for _ in range(2)]
        ops.unpack_paged(cache, table, lens, start, *rows, max_len=64)
        return (qr, out, *rows, pkg.decoder_sample.sample_tokens(out.flatten(1).matmul(head), u, top_p=top_p, top_k=top_k))

    caches = [ops.PagedCache(n * 4 + 3, 16, hkv, D, device=DEV) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[2])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for i in range(4):
        want = step(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got + (caches[0].data,), want + (caches[1].data,)):
            assert torch.equal(bits(a) if a.is_floating_point() else a, bits(b) if b.is_floating_point() else b), i
        x.copy_(rand(tuple(x.shape), dtype, 50 + i))
        u.copy_(torch.rand(n, device=DEV))
        table[3] = word([20, 21, 22, 3])                                 # a sequence moves to other pages
        lens += 1
        pos += 1
        top_p -= 0.1
        top_k += 7


def test_two_streams_at_once(ops):
    """The same cache read from two streams that overlap: each call's workspace is its own."""
    chats, k, v = filled(ops, [3000, 40], 64, 8, 128, seed=4)
    qs = [rand((2, 32, 128), BF, 60 + i, 1.4) for i in range(4)]
    call = lambda q: ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=3000)
    want = [call(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, call(q)))
    torch.cuda.synchronize()
    for i, a in got:
        assert torch.equal(bits(a), bits(want[i]))


def test_called_from_another_device(ops, pkg, monkeypatch):
    """The path that makes the tensors' device current first (taken here by saying so once a call)."""
    hq, hkv, D = 8, 2, 64
    sample = pkg.decoder_sample
    q, k, v = rand((2, hq, D), BF, 1), rand((2, hkv, D), BF, 2), rand((2, hkv, D), BF, 3)
    w, pos = torch.ones(D, device=DEV), word([4, 9])
    rot = pkg.decoder_attn.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    logits, u = rand((2, 100), F32, 5), torch.rand(2, device=DEV)

    def calls(u=u):
        chats = Chats(ops, [5, 10], 16, hkv, D)
        chats.fill(rand((15, hkv, D), BF, 6), rand((15, hkv, D), BF, 7))
        qr = ops.qk_norm_rotary_paged(q, k, v, w, w, pos, rot, chats.cache, chats.table, chats.k_len)
        return [qr, ops.paged_attention(qr, chats.cache, chats.table, chats.k_len, max_len=10), *chats.rows(),
                sample.sample_tokens(logits, u, top_k=5)]

    want = calls()
    real, said = ops._elsewhere, []
    for module in (ops, sample):
        monkeypatch.setattr(module, "_elsewhere", lambda device: (said.append(1), len(said) % 2 == 1 or real(device))[1])
    got = calls()
    assert len(said) == 10
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompts_then_tokens(ops, pkg, dtype):
    """A layer's work as a server does it: two prompts into pages and through causal_attention on the rows that the pages stand for, then
    tokens step by step with their choice, then a second prompt onto one history; each against float64."""
    attn, sample = pkg.decoder_attn, pkg.decoder_sample
    hq, hkv, D, R, vocab = 8, 2, 64, 16, 300
    rot = attn.TextRotary(D, 1e4, (12, 10, 10), True, DEV)
    qw, kw = 1 + 0.2 * rand((D,), F32, 1), 1 + 0.2 * rand((D,), F32, 2)
    cache = ops.PagedCache(12, R, hkv, D, device=DEV)
    table = word([[3, 9, 1, 7, 11], [0, 5, 2, 8, 10]])
    embed, head = rand((vocab, (hq + 2 * hkv) * D), dtype, 3), rand((hq * D, vocab), dtype, 4, 0.2)
    split = lambda x: (x[:, :hq * D].unflatten(1, (hq, D)), x[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D)),
                       x[:, (hq + hkv) * D:].unflatten(1, (hkv, D)))

    def rows(lens):
        k, v = (torch.full((sum(lens), hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        start = word([0] + np.cumsum(lens)[:-1].tolist(), torch.int64)
        return ops.unpack_paged(cache, table, word(lens), start, k, v, max_len=max(lens))

    def prompt(lens, new, tokens):
        pos = torch.cat([torch.arange(a - b, a) for a, b in zip(lens, new)]).to(torch.int32).to(DEV)
        q, k, v = split(embed[tokens])
        cu = word([0] + np.cumsum(new).tolist())
        qr = ops.qk_norm_rotary_paged(q, k, v, qw, kw, pos, rot, cache, table, word(lens), cu_q=cu)
        k, v = rows(lens)
        plan = attn.CausalPlan(new, lens, num_heads=hq, num_kv_heads=hkv, head_dim=D, dtype=dtype, device=DEV)
        out = attn.causal_attention(qr, k, v, plan)
        paged = ops.paged_attention(qr, cache, table, word(lens), max_len=max(lens), cu_q=cu)
        at = row = 0
        k32, v32 = rows32(lens)
        for n, length in zip(new, lens):
            visible = torch.arange(n, device=DEV) + length - n + 1
            assert_attention(out[at:at + n], attention_ref(qr[at:at + n], k[row:row + length], v[row:row + length], visible, D ** -0.5), length)
            assert_attention(paged[at:at + n], attention_ref(qr[at:at + n], k32[row:row + length], v32[row:row + length], visible, D ** -0.5),
                             length)
            at, row = at + n, row + length
        return out[word(np.cumsum(new).tolist(), torch.int64) - 1]

    def rows32(lens):
        k, v = (torch.empty(sum(lens), hkv, D, device=DEV) for _ in range(2))
        return ops.unpack_paged(cache, table, word(lens), word([0] + np.cumsum(lens)[:-1].tolist(), torch.int64), k, v, max_len=max(lens))

    def choose(out, seed):
        logits = out.flatten(1).matmul(head)
        u = torch.rand(2, generator=torch.Generator().manual_seed(seed)).to(DEV)
        token = sample.sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.9)
        x = logits.double().cpu().numpy()
        for i in range(2):
            order = np.lexsort((np.arange(vocab), -x[i]))[:50]
            p = np.exp((x[i][order] - x[i].max()) / np.float64(np.float32(0.8)))
            kept = order[np.cumsum(p) - p < np.float64(np.float32(0.9)) * p.sum()]
            assert int(token[i]) in kept.tolist()
        return token

    lens = [50, 21]
    token = choose(prompt(lens, lens, torch.arange(71, device=DEV) % vocab), 0)
    for step in range(4):
        lens = [n + 1 for n in lens]
        q, k, v = split(embed[token])
        pos = word([n - 1 for n in lens])
        qr = ops.qk_norm_rotary_paged(q, k, v, qw, kw, pos, rot, cache, table, word(lens))
        out = ops.paged_attention(qr, cache, table, word(lens), max_len=80)
        k32, v32 = rows32(lens)
        for i, (a, b) in enumerate(((0, lens[0]), (lens[0], sum(lens)))):
            assert_attention(out[i:i + 1], attention_ref(qr[i:i + 1], k32[a:b], v32[a:b], word([lens[i]]), D ** -0.5), lens[i])
        token = choose(out, 1 + step)
    choose(prompt([lens[0] + 1, lens[1] + 30], [1, 30], torch.cat([token[:1], torch.arange(30, device=DEV)])), 9)


def test_a_copied_cache_is_written_and_read_alone(ops):
    import copy
    chats, k, v = filled(ops, [40, 7], 16, 2, 64, seed=11)
    q = rand((2, 4, 64), BF, 9, 1.4)
    attend = lambda cache: ops.paged_attention(q, cache, chats.table, chats.k_len, max_len=40)
    before, out = chats.cache.data.clone(), attend(chats.cache)
    other = copy.deepcopy(chats.cache)
    assert torch.equal(bits(attend(other)), bits(out))
    ops.append_paged(rand((47, 2, 64), BF, 3), rand((47, 2, 64), BF, 4), other, chats.table, chats.k_len, cu_q=word([0, 40, 47]))
    assert torch.equal(chats.cache.data, before) and not torch.equal(other.data, before)
    assert torch.equal(bits(attend(chats.cache)), bits(out)) and not torch.equal(bits(attend(other)), bits(out))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_unpack_from_before_a_sequence(ops, dtype):
    """A negative first counts rows as any other does: token t's row is k_start + t - first, and tokens before 0 are none."""
    hkv, D, lengths = 2, 64, [20, 33, 5, 40]
    chats = Chats(ops, lengths, 16, hkv, D, seed=12)
    chats.fill(rand((98, hkv, D), F32, 1), rand((98, hkv, D), F32, 2))
    want = chats.rows(dtype)
    first, start, R = [-3, -17, -(2 ** 31), 2], [0, 10, -(2 ** 31) + 70, 80], 110
    for hint in (1, 40):
        got = [torch.full((R, hkv, D), 5.0, dtype=dtype, device=DEV) for _ in range(2)]
        ops.unpack_paged(chats.cache, chats.table, chats.k_len, word(start, torch.int64), *got, max_len=hint, first=word(first))
        for x, w in zip(got, want):
            ref = torch.full((R, hkv, D), 5.0, dtype=dtype, device=DEV)
            ref[3:23] = w[:20]
            ref[27:60] = w[20:53]
            ref[70:75] = w[53:58]
            ref[80:110] = w[58 + 2:58 + 32]
            assert torch.equal(bits(x), bits(ref))
    far = [torch.full((R, hkv, D), 5.0, dtype=dtype, device=DEV) for _ in range(2)]   # rows all before 0, or all behind the last
    ops.unpack_paged(chats.cache, chats.table, chats.k_len, word([-60, -2 ** 62, 2 ** 62, R - 2], torch.int64), *far, max_len=40,
                     first=word([-3, -(2 ** 31), -(2 ** 31), -3]))
    assert all(bool((x == 5).all()) for x in far)


@pytest.mark.parametrize("D", [64, 128])
def test_what_was_read_back_comes_back_at_the_ends_of_the_range(ops, D):
    """Float32 values that pages stand for, appended again, come back from the smallest normal scale to the last whose sixfold is
    a float32; zeros and NaN too. Beyond, groups stand for what the formula says, and the header promises no more."""
    low, high = 2.0 ** -126, torch.tensor(0x7e2a, dtype=torch.int16).view(BF).double().item()   # the next bf16 above: 6 s > 2^128
    assert 6 * high < torch.finfo(F32).max < 6 * high * (1 + 2.0 ** -7)
    tops = [6 * low, 6 * low * (1 - 2.0 ** -10), 6 * low * 1.5, 6 * low * (1 + 2.0 ** -7), 6 * high, 6 * high * (1 - 2.0 ** -10), 3 * high, 0.0,
            float("nan")]
    x = rand((len(tops), 2, D), F32, 13).double().clamp(-1, 1)
    x[:, :, ::64] = 1.0
    x = (x * torch.tensor(tops, dtype=torch.float64, device=DEV)[:, None, None]).float()
    chats = Chats(ops, [len(tops)], 16, 2, D)
    chats.fill(x, -x)
    k, v = chats.rows()
    want = packed(x)[0]
    assert torch.equal(k.double().nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(k.isnan(), want.isnan())
    assert torch.equal(bits(v[:-1]), bits(-k[:-1])) and bool(k[:-1].isfinite().all())
    chats.fill(k, v)
    for again, x in zip(chats.rows(), (k, v)):
        assert torch.equal(bits(again[:-1]), bits(x[:-1])) and bool(again[-1].isnan().all())
    # the ends beyond: 3e-40 has a scale of the smallest subnormal, half of which is a tie; 3.4e38 rounds up to a scale whose sixfold is none
    y = torch.tensor([3e-40, 3.4e38], device=DEV)[:, None, None].expand(2, 2, D).contiguous()
    far = Chats(ops, [2], 16, 2, D)
    far.fill(y, y)
    k, v = far.rows()
    assert torch.equal(k[0].double(), packed(y[:1])[0][0]) and bool((k[1] == float("inf")).all())
    far.fill(k, v)
    k, v = far.rows()
    assert bool((k[0] == 0).all()) and bool(k[1].isnan().all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq,hkv,D,new", [(8, 2, 128, 1), (8, 2, 64, 3)])
@pytest.mark.parametrize("n,at", [(65, 64), (257, 100), (1100, 0)])
def test_many_sequences_of_which_one_is_long(ops, dtype, hq, hkv, D, new, n, at):
    """More sequences than lanes, than threads, than either: jobs that stay whole beside one that is cut over many runs."""
    lengths = [new + (29 * i) % 150 for i in range(n)]
    lengths[at] = 5000
    chats, k, v = filled(ops, lengths, 32, hkv, D, [new] * n, seed=14)
    q = rand((n * new, hq, D), dtype, 9, 1.4)
    out = ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=5000, cu_q=chats.cu_q)
    check_attention(out, chats, q, k, v, D ** -0.5)
    assert torch.equal(bits(ops.paged_attention(q, chats.cache, chats.table, chats.k_len, max_len=5000, cu_q=chats.cu_q)), bits(out))
