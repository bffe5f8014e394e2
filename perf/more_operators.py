"""The paged 4-bit cache of the text decoder and the choice of the next token: their time on the GPU beside their plain forms.

The cache holds a head's keys and values in groups of 64: a bf16 scale s and a 4-bit number (0, .5, 1, 1.5, 2, 3, 4 or 6, and a
sign) for each value. Sequences own pages of it, named by a page table. A case is a dict of plain values:
  append   keys and values of new tokens into their pages, with per-head norm and (t, h, w) rotation on the way or as they are;
           the new rows are read back, as the prompt's own attention does
  unpack   sequences read back from their pages into rows
  attend   attention of new tokens over the pages
  sample   the next token of each row of logits: temperature, top-k, top-p and min-p, from given random numbers
`run` computes the plain form, or calls the package where `own` is set; `exact` computes each operator in float64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
THETA = 5000000.0
GROUP = 64
UNIT = float(2 ** 44)
# query heads, key/value heads, head_dim, (t, h, w) section of the rotation frequencies
HEADS = {"2b": (16, 8, 128, (24, 20, 20)), "8b": (32, 8, 128, (24, 20, 20)), "narrow": (14, 2, 64, (12, 10, 10))}
VOCAB = 151936


def listed():
    return [
        # One decode step of 64 chats: a token each goes to the chat's last page.
        {"name": "append_step_64_bf16", "kind": "append", "heads": "8b", "dtype": "bfloat16", "page": 64,
         "old": ",".join(str((137 * i) % 1500) for i in range(64)), "new": ",".join(["1"] * 64), "rotate": True},
        # One image's prompt in the model's default dtype, into small pages.
        {"name": "append_prompt_1181_f32", "kind": "append", "heads": "2b", "dtype": "float32", "page": 16, "old": "0", "new": "1181",
         "rotate": True},
        # A long document and a chat's turn in one prefill.
        {"name": "append_document_bf16", "kind": "append", "heads": "8b", "dtype": "bfloat16", "page": 128, "old": "0,1311",
         "new": "17200,811", "rotate": True},
        # A prefill's rotated keys and values, moved into pages afterwards.
        {"name": "append_rows_24001_bf16", "kind": "append", "heads": "8b", "dtype": "bfloat16", "page": 64, "old": "0", "new": "24001",
         "rotate": False},
        # Three short histories as rows, for a prompt in the default dtype.
        {"name": "unpack_short_f32", "kind": "unpack", "heads": "narrow", "dtype": "float32", "page": 32, "lengths": "300,64,1181"},
        # Two long histories as rows, for the prompts that go on from them.
        {"name": "unpack_history_bf16", "kind": "unpack", "heads": "8b", "dtype": "bfloat16", "page": 64, "lengths": "24001,7013"},
        # The next token of one chat: where latency counts.
        {"name": "attend_1_bf16", "kind": "attend", "heads": "8b", "dtype": "bfloat16", "page": 64, "lengths": "9001", "new": 1},
        # The next token of 96 chats whose histories run from one token to 8000.
        {"name": "attend_96_bf16", "kind": "attend", "heads": "8b", "dtype": "bfloat16", "page": 64,
         "lengths": ",".join(str(1 + 83 * i + (i * i) % 61) for i in range(96)), "new": 1},
        # Three drafted tokens a chat in the default dtype, narrow heads, small pages.
        {"name": "attend_draft_f32", "kind": "attend", "heads": "narrow", "dtype": "float32", "page": 16,
         "lengths": ",".join(str(5 + 131 * i) for i in range(24)), "new": 3},
        # One chat's next token: the 20 likeliest, of them the nucleus.
        {"name": "sample_1_f32", "kind": "sample", "dtype": "float32", "rows": 1, "vocab": VOCAB, "spread": 2.5, "how": "all"},
        # 64 chats, each with settings of its own.
        {"name": "sample_64_bf16", "kind": "sample", "dtype": "bfloat16", "rows": 64, "vocab": VOCAB, "spread": 2.5, "how": "mixed"},
        # 256 samples of answers by their nucleus alone, flat distributions among them.
        {"name": "sample_256_f32", "kind": "sample", "dtype": "float32", "rows": 256, "vocab": VOCAB, "spread": 2.5, "how": "nucleus"},
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    text = lambda values: ",".join(str(v) for v in values)
    case = {"kind": rng.choice(["append", "unpack", "attend", "attend", "sample", "sample"]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    if case["kind"] == "sample":
        case.update(rows=log(1, 256 if case["dtype"] == "float32" else 400), vocab=rng.choice([VOCAB, VOCAB, log(1000, VOCAB)]),
                    spread=rng.choice([0.5, 2.5, 2.5, 5.0]), how=rng.choice(["all", "mixed", "nucleus", "top", "floor", "plain"]))
        return case
    case.update(heads=rng.choice(list(HEADS)), page=rng.choice([16, 32, 64, 64, 128, 256]))
    half = case["dtype"] == "bfloat16"
    if case["kind"] == "append":
        left = log(1, 18011 if half else 6000)
        new, old = [], []
        for _ in range(rng.choice([1, 1, 2, 8, 100])):
            if left > 0:
                new.append(log(1, left))
                old.append(rng.choice([0, log(1, 3000)]))
                left -= new[-1]
        case.update(new=text(new), old=text(old), rotate=rng.random() < 0.7)
    elif case["kind"] == "unpack":
        case.update(lengths=text(log(1, 16000 if half else 6000) for _ in range(rng.choice([1, 1, 2]))))
    else:
        n = log(1, 96)
        top = log(2, 8000 if n > 8 else 48000)
        case.update(lengths=text(rng.randint(1, top) for _ in range(n)), new=rng.choice([1, 1, 1, 2, 5]))
    return case


# -------------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# -------------------------------------------------------------------------------------------------------------------
def _ints(text):
    return [int(v) for v in text.split(",")]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32


def _normal(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _word(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(lengths, page, gen):
    """(number of pages, page table [sequences, width]) with the sequences' pages anywhere; -1 where there is none."""
    need = [-(-v // page) for v in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device=DEV).cpu().tolist()
    table = np.full((len(lengths), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return total, torch.from_numpy(table).to(DEV)


def _where(lengths, firsts, page, table):
    """The slot (page * page_rows + row) of every token first <= t < length, one sequence after the other."""
    seq = np.repeat(np.arange(len(lengths)), [b - a for a, b in zip(firsts, lengths)])
    t = np.concatenate([np.arange(a, b) for a, b in zip(firsts, lengths)])
    seq, t = torch.from_numpy(seq).to(DEV), torch.from_numpy(t).to(DEV)
    return table[seq, t // page].long() * page + t % page


def _empty_cache(total, page, hkv, d):
    return {"k_codes": torch.zeros(total * page, hkv, d // 2, dtype=torch.uint8, device=DEV),
            "v_codes": torch.zeros(total * page, hkv, d // 2, dtype=torch.uint8, device=DEV),
            "k_scales": torch.zeros(total * page, hkv, d // GROUP, dtype=torch.bfloat16, device=DEV),
            "v_scales": torch.zeros(total * page, hkv, d // GROUP, dtype=torch.bfloat16, device=DEV)}


def _prepare_sample(case, gen, st):
    b, v = case["rows"], case["vocab"]
    x = torch.randn((b, v), generator=gen, device=DEV) * case["spread"]
    likely = torch.randint(0, v, (b, 12), generator=gen, device=DEV)           # a few tokens a model thinks likely
    x.scatter_add_(1, likely, torch.rand((b, 12), generator=gen, device=DEV) * 4 * case["spread"])
    st["logits"] = x.to(_dtype(case))
    st["u"] = torch.rand(b, generator=gen, device=DEV)
    how = case["how"]
    settings = {"temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if how in ("all", "top"):
        settings["top_k"] = 20
    if how in ("all", "nucleus"):
        settings["top_p"] = 0.95
    if how in ("all", "floor"):
        settings["min_p"] = 0.02
    if how == "mixed":                                                          # every row its own
        pick = lambda values, dtype: torch.tensor(values, dtype=dtype, device=DEV)[
            torch.randint(0, len(values), (b,), generator=gen, device=DEV)]
        settings = {"temperature": pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32), "top_k": pick([0, 1, 20, 50, 1000], torch.int32),
                    "top_p": pick([0.5, 0.9, 0.95, 1.0], torch.float32), "min_p": pick([0.0, 0.0, 0.05], torch.float32)}
    st["settings"] = settings


def _prepare_cache(case, gen, st):
    hq, hkv, d, section = HEADS[case["heads"]]
    dt, page = _dtype(case), case["page"]
    if case["kind"] == "append":
        new, old = _ints(case["new"]), _ints(case["old"])
        lengths = [a + b for a, b in zip(new, old)]
    else:
        lengths = _ints(case["lengths"])
        new = [min(case.get("new", 0), v) for v in lengths]
        old = [0] * len(lengths)
    total, table = _pages(lengths, page, gen)
    st.update(lengths=lengths, new=new, page=page, table=table, k_len=_word(lengths), slots=_where(lengths, old, page, table))
    n, rows = sum(new), len(st["slots"])
    st["cu_q"] = None if all(v == 1 for v in new) else _word([0] + np.cumsum(new).tolist())
    st["first"] = _word(old)
    st["k_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum([b - a for a, b in zip(old, lengths)])[:-1]])).to(DEV)
    st["cache"] = _empty_cache(total, page, hkv, d)
    if case["kind"] == "append":
        qkv = _normal(gen, (n, (hq + 2 * hkv) * d), 1.7, dt)                   # what the qkv Dense leaves, one row a token
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        st["q_norm"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        st["k_norm"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        at = np.concatenate([np.arange(a, b) for a, b in zip(old, lengths)])   # a video's tokens step through (t, h, w)
        st["positions"] = torch.from_numpy(np.stack([at, at + at % 7, at + at % 11]).astype(np.int32)).to(DEV)
        st["section"] = section
    else:
        k, v = _normal(gen, (rows, hkv, d), 1.4, torch.float32), _normal(gen, (rows, hkv, d), 1.0, torch.float32)
        for name, x in (("k", k), ("v", v)):
            codes, scales = _quantise(x.double())
            st["cache"][name + "_codes"][st["slots"]] = codes
            st["cache"][name + "_scales"][st["slots"]] = scales
        st["q"] = _normal(gen, (n, hq, d), 1.4, dt)
    return total, k if case["kind"] != "append" else None, v if case["kind"] != "append" else None


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "sample":
        _prepare_sample(case, gen, st)
    else:
        total, k, v = _prepare_cache(case, gen, st)
    if own:
        from __graft_entry__ import load_package
        pkg = load_package()
        st["pkg"] = pkg
        if case["kind"] != "sample":
            hq, hkv, d, section = HEADS[case["heads"]]
            ops = pkg.decoder_cache
            st["paged"] = ops.PagedCache(total, case["page"], hkv, d, device=DEV)
            st["rotary"] = pkg.decoder_attn.TextRotary(d, THETA, section, device=DEV)
            if k is not None:
                cu = _word([0] + np.cumsum(st["lengths"]).tolist())
                ops.append_paged(k, v, st["paged"], st["table"], st["k_len"], cu_q=cu)
    return st


# -------------------------------------------------------------------------------------------------------------------
# one pass
# -------------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """(codes, two a byte, scales) of x [..., D] in float64: the nearest numbers, ties to the even code."""
    g = x.unflatten(-1, (-1, GROUP))
    scale = (g.abs().amax(-1) / 6).float().bfloat16()
    t = g.abs() / scale.double()[..., None]
    code = ((t > 0.25).byte() + (t >= 0.75).byte() + (t > 1.25).byte() + (t >= 1.75).byte() + (t > 2.5).byte() + (t >= 3.5).byte()
            + (t > 5.0).byte() + 8 * (g < 0).byte()).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales):
    """What codes and scales stand for, in float32 (exact)."""
    number = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    number = torch.cat([number, -number])
    byte = torch.arange(256, device=DEV)
    pair = torch.stack([number[byte % 16], number[byte // 16]], -1)
    x = pair[codes.int()].flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _plain_append(st):
    cache, slots, k, v = st["cache"], st["slots"], st["k"].double(), st["v"].double()
    out = []
    if st["case"]["rotate"]:
        d = k.shape[-1]
        half = d // 2
        axis = torch.tensor([j % 3 if j < 3 * st["section"][j % 3] else 0 for j in range(half)], device=DEV)
        freq = THETA ** (-2.0 * torch.arange(half, dtype=torch.float64, device=DEV) / d)
        angle = st["positions"].double()[axis].t() * freq      # in 64 bits: positions run far
        cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

        def turn(x, weight, cos, sin):
            y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
            a, b = y[..., :half], y[..., half:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        out.append(turn(st["q"].float(), st["q_norm"], cos.float(), sin.float()).to(st["q"].dtype))
        k = turn(k, st["k_norm"].double(), cos, sin)           # in 64 bits: values next to a border between two codes
    for name, x in (("k", k), ("v", v)):
        codes, scales = _quantise(x)
        cache[name + "_codes"][slots] = codes
        cache[name + "_scales"][slots] = scales
    return out + _plain_unpack(st, st["k"].dtype)


def _plain_unpack(st, dtype):
    cache, slots = st["cache"], st["slots"]
    return [_values(cache[name + "_codes"][slots], cache[name + "_scales"][slots]).to(dtype) for name in ("k", "v")]


def _plain_attend(st):
    q, cache, page = st["q"], st["cache"], st["page"]
    hq, d = q.shape[1], q.shape[2]
    hkv = cache["k_codes"].shape[1]
    n, most = len(st["lengths"]), max(st["new"])
    width = st["table"].shape[1]
    slots = (st["table"].clamp(min=0).long()[:, :, None] * page + torch.arange(page, device=DEV)).flatten(1)
    k = _values(cache["k_codes"][slots], cache["k_scales"][slots])             # [sequences, keys, hkv, d], padded to the longest
    v = _values(cache["v_codes"][slots], cache["v_scales"][slots])
    keys = width * page
    new = torch.tensor(st["new"], device=DEV)
    first = torch.cumsum(new, 0) - new
    row = torch.arange(most, device=DEV)
    at = (first[:, None] + torch.minimum(row, new[:, None] - 1)).flatten()     # a sequence's last token where it has fewer
    rows = q[at].float().view(n, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(n * hkv, -1, d)
    s = torch.matmul(rows, k.permute(0, 2, 3, 1).reshape(n * hkv, d, keys).contiguous()) * d ** -0.5
    s = s.view(n, hkv, most, hq // hkv, keys)
    seen = st["k_len"][:, None].long() - new[:, None] + torch.minimum(row, new[:, None] - 1)
    s = s.masked_fill(torch.arange(keys, device=DEV) > seen[:, None, :, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n * hkv, -1, keys), v.permute(0, 2, 1, 3).reshape(n * hkv, keys, d).contiguous())
    o = (o.view(n, hkv, most, hq // hkv, d) / total).permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)
    return o[row < new[:, None]].to(q.dtype)


def _plain_sample(st):
    x, u = st["logits"].double(), st["u"].double()
    column = lambda name, dtype: torch.as_tensor(st["settings"][name], device=DEV).to(dtype).expand(x.shape[0])[:, None]
    temperature, top_k = column("temperature", torch.float32).double(), column("top_k", torch.int64)
    # settings are float32, as a user's tensors of them are
    top_p, min_p = column("top_p", torch.float32).double(), column("min_p", torch.float32).double()
    v = x.shape[1]
    z = (x - x.amax(1, keepdim=True)) / temperature
    w = torch.round(torch.exp(z.nan_to_num(nan=0.0)) * UNIT).to(torch.int64)   # whole numbers: a sum does not depend on its order
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    sorted_w = w.gather(1, order)
    rank = torch.arange(v, device=DEV)
    sorted_w = torch.where((top_k > 0) & (rank >= top_k), 0, sorted_w)
    before = torch.cumsum(sorted_w, 1) - sorted_w
    whole = sorted_w.sum(1, keepdim=True).double()
    keep = (before.double() < top_p * whole) | (rank == 0) | (top_p >= 1)
    keep &= (sorted_w.double() >= min_p * UNIT) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sorted_w, 0))
    upto = torch.cumsum(kept, 1)
    token = (upto.double() <= u[:, None] * upto[:, -1:].double()).sum(1)
    return torch.where(temperature[:, 0] > 0, token, order[:, 0])


def run(state):
    st = state
    kind = st["case"]["kind"]
    if not own:
        if kind == "append":
            return _plain_append(st)
        if kind == "unpack":
            return _plain_unpack(st, _dtype(st["case"]))
        return _plain_attend(st) if kind == "attend" else _plain_sample(st)
    pkg = st["pkg"]
    if kind == "sample":
        return pkg.decoder_sample.sample_tokens(st["logits"], st["u"], **st["settings"])
    ops, cache, table, k_len = pkg.decoder_cache, st["paged"], st["table"], st["k_len"]
    if kind == "attend":
        return ops.paged_attention(st["q"], cache, table, k_len, max_len=max(st["lengths"]), cu_q=st["cu_q"])
    out = []
    if kind == "append" and st["case"]["rotate"]:
        out.append(ops.qk_norm_rotary_paged(st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"], st["positions"], st["rotary"],
                                            cache, table, k_len, eps=EPS, cu_q=st["cu_q"]))
    elif kind == "append":
        ops.append_paged(st["k"], st["v"], cache, table, k_len, cu_q=st["cu_q"])
    rows, (_, hkv, d, _) = len(st["slots"]), HEADS[st["case"]["heads"]]
    k = torch.empty(rows, hkv, d, dtype=_dtype(st["case"]), device=DEV)
    v = torch.empty_like(k)
    ops.unpack_paged(cache, table, k_len, st["k_start"], k, v, max_len=max(st["new"] if kind == "append" else st["lengths"]),
                     first=st["first"])
    return out + [k, v]


# -------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# -------------------------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * size + case["rows"] * 28, "flops": 4 * values}
    hq, hkv, d, _ = HEADS[case["heads"]]
    packed = 2 * hkv * (d // 2 + d // GROUP * 2)               # bytes of a token's keys and values
    if case["kind"] == "append":
        n = sum(_ints(case["new"]))
        moved = n * (2 * hkv * d * size + packed)
        if case["rotate"]:
            moved += n * (2 * hq * d * size + 12) + 8 * d
        return {"bytes": moved + n * (packed + 2 * hkv * d * size), "flops": n * (hq * 8 + hkv * 40) * d}
    lengths = _ints(case["lengths"])
    if case["kind"] == "unpack":
        return {"bytes": sum(lengths) * (packed + 2 * hkv * d * size), "flops": sum(lengths) * 2 * hkv * d}
    new = [min(case["new"], v) for v in lengths]
    pairs = sum(n * (v - n) + n * (n + 1) // 2 for n, v in zip(new, lengths))
    return {"bytes": 2 * sum(new) * hq * d * size + sum(lengths) * packed, "flops": 4 * pairs * hq * d}


# -------------------------------------------------------------------------------------------------------------------
# the operators in float64
# -------------------------------------------------------------------------------------------------------------------
def _nearest(x):
    """What the 4-bit form of x [..., D] stands for, by the distance to each number."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    scale = (g.abs().max(-1, keepdim=True)[0] / 6).float().bfloat16().double()
    best, far = torch.zeros_like(g), g.abs().clone()
    for number, even in ((0.5, False), (1.0, True), (1.5, False), (2.0, True), (3.0, False), (4.0, True), (6.0, False)):
        now = (g.abs() - number * scale).abs()
        # in the order of the codes: an even one takes a tie from the odd one before it
        closer = (now <= far) if even else (now < far)
        best, far = torch.where(closer, number * scale, best), torch.where(closer, now, far)
    return torch.copysign(best, g).reshape(x.shape)


def _exact_rows(st):
    return [_values(st["cache"][n + "_codes"][st["slots"]].clone(), st["cache"][n + "_scales"][st["slots"]]).double() for n in ("k", "v")]


def _exact_append(st):
    k, v = st["k"].double(), st["v"].double()
    if not st["case"]["rotate"]:
        return [_nearest(k), _nearest(v)]
    half = k.shape[-1] // 2
    section, pos = st["section"], st["positions"].double()
    j = torch.arange(half, device=DEV)
    use_h, use_w = ((j % 3 == a) & (j < 3 * section[a]) for a in (1, 2))
    where = torch.where(use_w, pos[2][:, None], torch.where(use_h, pos[1][:, None], pos[0][:, None]))
    angle = where * torch.exp(-math.log(THETA) * j.double() / half)

    def turn(x, weight):
        x = x.double()
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / (2 * half) + EPS) * weight.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
        return torch.cat([z.real, z.imag], -1)

    return [turn(st["q"], st["q_norm"]), _nearest(turn(k, st["k_norm"])), _nearest(v)]


def _exact_attend(st):
    k, v = _exact_rows(st)
    q = st["q"].double()
    per, out, at, base = q.shape[1] // k.shape[1], torch.zeros_like(st["q"], dtype=torch.float64), 0, 0
    for n, length in zip(st["new"], st["lengths"]):
        ks, vs = k[base:base + length], v[base:base + length]
        for h in range(q.shape[1]):
            s = (ks[:, h // per].contiguous() @ q[at:at + n, h].t().contiguous()) / math.sqrt(q.shape[2])
            hidden = torch.arange(length, device=DEV)[:, None] > length - n + torch.arange(n, device=DEV)
            w = torch.softmax(torch.where(hidden, float("-inf"), s), 0)
            out[at:at + n, h] = w.t().contiguous() @ vs[:, h // per].contiguous()
        at, base = at + n, base + length
    return out


def exact(case, seed):
    if case["kind"] == "sample":
        return None
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    return _exact_rows(st) if case["kind"] == "unpack" else _exact_attend(st)
