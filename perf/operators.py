"""The decoder operators whose time on the GPU is watched, beside their plain forms.

Between the injection of the vision rows and the next token a text decoder layer needs its queries and keys normalised
and rotated, attention over the prompt, and attention of new tokens over the cache. A case is a dict of plain values:
  rotary   per-head RMSNorm of queries and keys and the (t, h, w) position rotation; keys and values go to cache rows
  causal   attention of packed prompts, each over the keys it already has and causally over its own
  decode   attention of a few new tokens of each sequence over that sequence's cache
  prefix   the same where groups of sequences share a prefix (an image's tokens, a system prompt), which lies once in
           the cache
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
# query heads, key/value heads, head_dim, (t, h, w) section of the rotation frequencies
HEADS = {"2b": (16, 8, 128, (24, 20, 20)), "8b": (32, 8, 128, (24, 20, 20)), "narrow": (14, 2, 64, (12, 10, 10))}


def listed():
    return [
        # One decode step of 64 chats: a token each, its key and value written to the chat's cache slot.
        {"name": "rotary_step_64_bf16", "kind": "rotary", "heads": "8b", "dtype": "bfloat16", "tokens": 64, "image": 0,
         "first": 9000, "rows": "slots", "interleaved": True},
        # One image's prompt in the model's default dtype; keys and values appended to one sequence's rows.
        {"name": "rotary_prompt_1181_f32", "kind": "rotary", "heads": "2b", "dtype": "float32", "tokens": 1181,
         "image": 34, "first": 0, "rows": "append", "interleaved": True},
        # A long document in one prefill.
        {"name": "rotary_document_18011_bf16", "kind": "rotary", "heads": "8b", "dtype": "bfloat16", "tokens": 18011,
         "image": 84, "first": 131, "rows": "append", "interleaved": True},
        # Prompts of unlike lengths packed into one prefill, from a single token to a few images.
        {"name": "causal_packed_bf16", "kind": "causal", "heads": "2b", "dtype": "bfloat16",
         "new": "1,37,577,1153,2309,4099", "old": "0,0,0,0,0,0"},
        # One long video prompt in a prefill.
        {"name": "causal_long_16411_bf16", "kind": "causal", "heads": "8b", "dtype": "bfloat16", "new": "16411", "old": "0"},
        # A chat turn with a picture onto long histories that lie in the cache already.
        {"name": "causal_turn_bf16", "kind": "causal", "heads": "8b", "dtype": "bfloat16", "new": "300,811",
         "old": "24001,7013"},
        # Three prompts in the default dtype, narrow heads.
        {"name": "causal_packed_f32", "kind": "causal", "heads": "narrow", "dtype": "float32", "new": "1181,317,5",
         "old": "0,64,0"},
        # The next token of one chat: where latency counts.
        {"name": "decode_1_bf16", "kind": "decode", "heads": "8b", "dtype": "bfloat16", "lengths": "9001", "new": 1},
        # The next token of 96 chats whose histories run from one token to 8000.
        {"name": "decode_96_bf16", "kind": "decode", "heads": "8b", "dtype": "bfloat16",
         "lengths": ",".join(str(1 + 83 * i + (i * i) % 61) for i in range(96)), "new": 1},
        # 48 questions about one video whose tokens lie in the cache once.
        {"name": "prefix_video_bf16", "kind": "prefix", "heads": "8b", "dtype": "bfloat16", "prefixes": "9216",
         "groups": "48", "lengths": ",".join(str(11 + (37 * i) % 400) for i in range(48)), "new": 1},
        # Samples of answers to two prompts in the default dtype.
        {"name": "prefix_samples_f32", "kind": "prefix", "heads": "2b", "dtype": "float32", "prefixes": "2310,777",
         "groups": "5,3", "lengths": "1,2,63,64,65,130,7,300", "new": 1},
        # 256 samples after one long prompt.
        {"name": "prefix_samples_256_bf16", "kind": "prefix", "heads": "8b", "dtype": "bfloat16", "prefixes": "24007",
         "groups": "256", "lengths": ",".join(str(1 + (53 * i) % 257) for i in range(256)), "new": 1},
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    text = lambda values: ",".join(str(v) for v in values)
    case = {"kind": rng.choice(["rotary", "causal", "causal", "decode", "prefix"]), "heads": rng.choice(list(HEADS)),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    half = case["dtype"] == "bfloat16"
    if case["kind"] == "rotary":
        tokens = log(1, 18011 if half else 6000)
        case.update(tokens=tokens, image=rng.choice([0, min(84, math.isqrt(tokens))]), first=rng.choice([0, log(1, 200000)]),
                    rows=rng.choice(["slots", "append", "none"] if tokens <= 256 else ["append", "none"]),
                    interleaved=rng.random() < 0.7)
    elif case["kind"] == "causal":
        left = log(1, 9000 if half else 3000)
        new, old = [], []
        while left > 0 and len(new) < 8:
            new.append(min(left, log(1, left)))
            old.append(rng.choice([0, 0, log(1, 12000 if half else 4000)]))
            left -= new[-1]
        case.update(new=text(new), old=text(old))
    elif case["kind"] == "decode":
        n = log(1, 96)
        top = log(2, 8000 if n > 8 else 32000)
        case.update(lengths=text(rng.randint(1, top) for _ in range(n)), new=rng.choice([1, 1, 1, 2, 5]))
    else:
        groups = [log(1, 64) for _ in range(rng.choice([1, 1, 2, 3]))]
        case.update(prefixes=text(log(16, 12000 if half else 4000) for _ in groups), groups=text(groups),
                    lengths=text(log(1, 400) for _ in range(sum(groups))), new=rng.choice([1, 1, 1, 3]))
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


def _starts(lengths, first=0):
    """Where each of the runs begins when they lie one after the other."""
    return [first + v for v in np.concatenate([[0], np.cumsum(lengths)[:-1]]).tolist()]


def _positions(tokens, image, first):
    """(t, h, w) of a prompt: text counts on, an image of image x image tokens keeps t and walks h and w."""
    pos = np.arange(first, first + tokens, dtype=np.int64)[None].repeat(3, 0)
    at = tokens // 8
    n = min(image * image, tokens - at)
    if image > 0 and n > 0:
        i = np.arange(n)
        pos[0, at:at + n] = first + at
        pos[1, at:at + n] = first + at + i // image
        pos[2, at:at + n] = first + at + i % image
        pos[:, at + n:] = first + at + image + np.arange(tokens - at - n)
    return torch.from_numpy(pos.astype(np.int32)).to(DEV)


def _prepare_rotary(case, gen, st):
    hq, hkv, d, section = HEADS[case["heads"]]
    n, dt = case["tokens"], _dtype(case)
    qkv = _normal(gen, (n, (hq + 2 * hkv) * d), 1.7, dt)       # what the qkv Dense leaves, one row a token
    st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
    st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
    st["q_norm"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
    st["k_norm"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
    st["section"] = section
    if case["rows"] == "slots":                                # every sequence has its own 96 rows
        st["positions"] = torch.randint(0, case["first"] + 1, (1, n), generator=gen, device=DEV).repeat(3, 1).to(torch.int32)
        within = torch.randint(0, 96, (n,), generator=gen, device=DEV)
        st["rows"], cache = torch.arange(n, device=DEV) * 96 + within, 96 * n
    else:
        st["positions"] = _positions(n, case["image"], case["first"])
        st["rows"], cache = torch.arange(n, device=DEV) + 5, n + 9
    if case["rows"] == "none":
        st["rows"] = st["k_cache"] = st["v_cache"] = None
    else:
        st["k_cache"] = _normal(gen, (cache, hkv, d), 1.0, dt)
        st["v_cache"] = _normal(gen, (cache, hkv, d), 1.0, dt)


def _prepare_attention(case, gen, st):
    hq, hkv, d, _ = HEADS[case["heads"]]
    dt = _dtype(case)
    if case["kind"] == "causal":
        new, old = _ints(case["new"]), _ints(case["old"])
        lengths = [a + b for a, b in zip(new, old)]
        prefixes, groups = [], []
    else:
        own_lengths = _ints(case["lengths"])
        new = [min(case["new"], v) for v in own_lengths]
        lengths = own_lengths
        prefixes = _ints(case["prefixes"]) if case["kind"] == "prefix" else []
        groups = _ints(case["groups"]) if case["kind"] == "prefix" else []
    starts = _starts(prefixes + lengths)
    rows = sum(prefixes) + sum(lengths)
    st["q"] = _normal(gen, (sum(new), hq, d), 1.4, dt)
    st["k"] = _normal(gen, (rows, hkv, d), 1.4, dt)
    st["v"] = _normal(gen, (rows, hkv, d), 1.0, dt)
    st["new"], st["lengths"], st["starts"] = new, lengths, starts[len(prefixes):]
    st["prefixes"], st["prefix_starts"], st["groups"] = prefixes, starts[:len(prefixes)], groups
    long = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    if case["kind"] != "causal":
        st["k_start"], st["k_len"] = long(st["starts"]), word(lengths)
        st["cu_q"] = None if max(new) == 1 else word([0] + np.cumsum(new).tolist())
        st["prefix_start"], st["prefix_len"] = long(st["prefix_starts"]), word(prefixes)
        st["cu_groups"] = word([0] + np.cumsum(groups).tolist())


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    (_prepare_rotary if case["kind"] == "rotary" else _prepare_attention)(case, gen, st)
    if own:
        from __graft_entry__ import load_package
        ops = st["ops"] = load_package().decoder_attn
        hq, hkv, d, section = HEADS[case["heads"]]
        if case["kind"] == "rotary":
            st["rotary"] = ops.TextRotary(d, THETA, section, interleaved=case["interleaved"], device=DEV)
        elif case["kind"] == "causal":
            st["plan"] = ops.CausalPlan(st["new"], st["lengths"], st["starts"], num_heads=hq, num_kv_heads=hkv,
                                        head_dim=d, dtype=_dtype(case), device=DEV)
    return st


# -------------------------------------------------------------------------------------------------------------------
# one pass
# -------------------------------------------------------------------------------------------------------------------
def _axes(section, interleaved, half):
    """Which of (t, h, w) each rotation frequency follows."""
    if not interleaved:
        return [0] * section[0] + [1] * section[1] + [2] * section[2]
    return [j % 3 if j < 3 * section[j % 3] else 0 for j in range(half)]


def _plain_rotary(st):
    case = st["case"]
    d = st["q"].shape[-1]
    half = d // 2
    axes = torch.tensor(_axes(st["section"], case["interleaved"], half), device=DEV)
    freq = THETA ** (-2.0 * torch.arange(half, dtype=torch.float64, device=DEV) / d)
    angle = st["positions"].double()[axes].t() * freq          # [tokens, half], in 64 bits: positions run far
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, weight):
        x32 = x.float()
        y = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS) * weight
        a, b = y[..., :half], y[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)

    q, k = turn(st["q"], st["q_norm"]), turn(st["k"], st["k_norm"])
    if st["rows"] is None:
        return q, k
    st["k_cache"][st["rows"]] = k
    st["v_cache"][st["rows"]] = st["v"]
    return q, st["k_cache"], st["v_cache"]


def _plain_attention(st):
    q, k, v = st["q"], st["k"], st["v"]
    hq, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    out = torch.empty_like(q)
    group = [g for g, n in enumerate(st["groups"]) for _ in range(n)]
    at = 0
    for i, (n, length, start) in enumerate(zip(st["new"], st["lengths"], st["starts"])):
        own_k, own_v, before = k[start:start + length], v[start:start + length], 0
        if group:
            p, before = st["prefix_starts"][group[i]], st["prefixes"][group[i]]
            own_k, own_v = torch.cat([k[p:p + before], own_k]), torch.cat([v[p:p + before], own_v])
        kt = own_k.float().permute(1, 2, 0).contiguous()       # [hkv, d, keys]
        vt = own_v.float().transpose(0, 1).contiguous()        # [hkv, keys, d]
        keys = before + length
        step = max(1, (1 << 28) // (hq * keys))                # rows of scores kept to 1 GiB
        for a in range(0, n, step):
            b = min(n, a + step)
            rows = q[at + a:at + b].float().unflatten(1, (hkv, hq // hkv)).permute(1, 0, 2, 3).reshape(hkv, -1, d)
            s = torch.matmul(rows, kt) * d ** -0.5
            if n > 1:
                last = torch.arange(keys - n + a, keys - n + b, device=DEV).repeat_interleave(hq // hkv)
                s = s.masked_fill(torch.arange(keys, device=DEV)[None] > last[:, None], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(p, vt) / p.sum(-1, keepdim=True)
            out[at + a:at + b] = o.unflatten(1, (b - a, hq // hkv)).permute(1, 0, 2, 3).reshape(b - a, hq, d).to(out.dtype)
        at += n
    return out


def run(state):
    st = state
    kind = st["case"]["kind"]
    if not own:
        return _plain_rotary(st) if kind == "rotary" else _plain_attention(st)
    ops = st["ops"]
    if kind == "rotary":
        q, k, v = ops.qk_norm_rotary(st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"], st["positions"], st["rotary"],
                                     eps=EPS, k_cache=st["k_cache"], v_cache=st["v_cache"], rows=st["rows"])
        return (q, k) if st["rows"] is None else (q, k, v)
    if kind == "causal":
        return ops.causal_attention(st["q"], st["k"], st["v"], st["plan"])
    if kind == "decode":
        return ops.decode_attention(st["q"], st["k"], st["v"], st["k_start"], st["k_len"], max_len=max(st["lengths"]),
                                    cu_q=st["cu_q"])
    return ops.prefix_attention(st["q"], st["k"], st["v"], st["k_start"], st["k_len"], st["prefix_start"],
                                st["prefix_len"], st["cu_groups"], max_len=max(st["lengths"]),
                                max_prefix=max(st["prefixes"]), cu_q=st["cu_q"])


# -------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# -------------------------------------------------------------------------------------------------------------------
def work(case):
    hq, hkv, d, _ = HEADS[case["heads"]]
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "rotary":
        n = case["tokens"]
        moved = 2 * n * (hq + hkv) * d * size + n * 12 + 2 * d * 4
        if case["rows"] != "none":
            moved += 2 * n * hkv * d * size + n * 8
        return {"bytes": moved, "flops": 8 * n * (hq + hkv) * d}
    if case["kind"] == "causal":
        new, old = _ints(case["new"]), _ints(case["old"])
        lengths = [a + b for a, b in zip(new, old)]
        before = [0] * len(new)
        keys = sum(lengths)
    else:
        lengths = _ints(case["lengths"])
        new = [min(case["new"], v) for v in lengths]
        prefixes = _ints(case["prefixes"]) if case["kind"] == "prefix" else [0]
        groups = _ints(case["groups"]) if case["kind"] == "prefix" else [len(lengths)]
        before = [p for p, n in zip(prefixes, groups) for _ in range(n)]
        keys = sum(lengths) + sum(prefixes)
    pairs = sum(n * (b + v - n) + n * (n + 1) // 2 for n, v, b in zip(new, lengths, before))
    return {"bytes": 2 * sum(new) * hq * d * size + 2 * keys * hkv * d * size, "flops": 4 * pairs * hq * d}


# -------------------------------------------------------------------------------------------------------------------
# the operators in float64
# -------------------------------------------------------------------------------------------------------------------
def _exact_rotary(st):
    half = st["q"].shape[-1] // 2
    section, pos = st["section"], st["positions"].double()
    j = torch.arange(half, device=DEV)
    if st["case"]["interleaved"]:
        pick = lambda axis: (j % 3 == axis) & (j < 3 * section[axis])
        use_h, use_w = pick(1), pick(2)
    else:
        use_h = (j >= section[0]) & (j < section[0] + section[1])
        use_w = j >= section[0] + section[1]
    where = torch.where(use_w, pos[2][:, None], torch.where(use_h, pos[1][:, None], pos[0][:, None]))
    angle = where / torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV), j.double() / half)
    phase = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turn(x, weight):
        x = x.double()
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / (2 * half) + EPS) * weight.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * phase
        return torch.cat([z.real, z.imag], -1)

    q, k = turn(st["q"], st["q_norm"]), turn(st["k"], st["k_norm"])
    if st["rows"] is None:
        return q, k
    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    k_cache.index_copy_(0, st["rows"], k)
    v_cache.index_copy_(0, st["rows"], st["v"].double())
    return q, k_cache, v_cache


def _exact_attention(st):
    q, k, v = st["q"], st["k"], st["v"]
    per = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    seq, at = 0, 0
    prefixes = [(p, b, n) for p, b, n in zip(st["prefix_starts"], st["prefixes"], st["groups"])] or [(0, 0, len(st["new"]))]
    for p, b, members in prefixes:
        for _ in range(members):
            n, length, start = st["new"][seq], st["lengths"][seq], st["starts"][seq]
            rows = list(range(p, p + b)) + list(range(start, start + length))
            rows = torch.tensor(rows, device=DEV)
            ks, vs = k[rows].double(), v[rows].double()
            for h in range(q.shape[1]):
                kh, vh = ks[:, h // per].contiguous(), vs[:, h // per].contiguous()
                for a in range(0, n, 4096):
                    t = torch.arange(a, min(n, a + 4096), device=DEV)
                    w = (kh @ q[at + t, h].double().t().contiguous()).t() / math.sqrt(q.shape[2])
                    hidden = torch.arange(len(rows), device=DEV)[None] - (len(rows) - n) > t[:, None]
                    w = torch.where(hidden, torch.zeros_like(w), torch.exp(w - torch.where(hidden, w - 1e300, w).max(1, keepdim=True)[0]))
                    out[at + t, h] = (w @ vh) / w.sum(1, keepdim=True)
            at += n
            seq += 1
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_rotary(st) if case["kind"] == "rotary" else _exact_attention(st)
