"""Rotary positions, a paged cache with its appended rows and the attention that
reads it, and a batch's decode step over it, as timed cases.

The shapes are the model's attention (32 query heads over 4 kv heads of 128) and
neighbours of it (other head counts and widths), at the batches and lengths a
serving loop meets. A case is a dict of plain values; its ``kind`` picks the
operator:

- ``rotate``: rows of heads rotated at the positions of their tokens;
- ``append``: rows of several sequences, K normed and rotated on the way where
  the case says so, written to the pages their positions fall in, and read back;
- ``attend``: one new token of each sequence over its pages;
- ``step``: a batch's whole step of a layer: q and k normed and rotated, k and v
  appended, attention over each sequence's rows; the new rows are read back.

A sequence's row at position p is row p % page of page table[sequence][p // page].
Pages hold f16, f32, or the Q8_0 blocks of 32 values: the block's scale is its
largest magnitude over 127 and a value's code its product with the scale's
reciprocal, rounded half away from zero, each step in 32 bits; the scale is
stored in f16. A stored value reads as the f16 nearest to scale times code.

Norm and rotation round as the framework's other prologues do: the mean of
squares, angles, cosines and sines in 64 bits, rounded to 32; x * inv * weight and
the rotation's products and sums in 32 bits, one rounding each.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
EPS = 1e-6


def listed():
    return [
        # A decode token's query and key heads.
        {"name": "rotate_1x36", "kind": "rotate", "rows": 1, "heads": 36, "dim": 128, "rot": 128, "layout": "half",
         "scaling": "none", "far": 4096, "spread": False},
        # A ragged chunk of heads that rotate only a part of themselves, neighbours paired.
        {"name": "rotate_1001x9_part", "kind": "rotate", "rows": 1001, "heads": 9, "dim": 80, "rot": 32,
         "layout": "interleaved", "scaling": "linear", "far": 16000, "spread": True},
        # A long prompt's chunk far beyond the trained context.
        {"name": "rotate_4096x36_yarn", "kind": "rotate", "rows": 4096, "heads": 36, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "yarn", "far": 131072, "spread": False},
        # One token's rows: launches count.
        {"name": "append_1", "kind": "append", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "far": 4096, "page": 64,
         "elem": "f16", "heads": 32, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half", "scaling": "none",
         "norm": True},
        # A token of each request of a batch, into 8-bit pages.
        {"name": "append_64_q8", "kind": "append", "seqs": 64, "rows_lo": 1, "rows_hi": 1, "far": 8000, "page": 32,
         "elem": "q8_0", "heads": 32, "kv_heads": 4, "dim": 128, "rot": 64, "layout": "interleaved",
         "scaling": "ntk", "norm": False},
        # Several prompts' chunks at once, of uneven lengths.
        {"name": "append_9_prompts", "kind": "append", "seqs": 9, "rows_lo": 100, "rows_hi": 1200, "far": 30000,
         "page": 64, "elem": "f16", "heads": 32, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half",
         "scaling": "yarn", "norm": True},
        # The first tokens of one conversation.
        {"name": "attend_1x100", "kind": "attend", "seqs": 1, "len_lo": 100, "len_hi": 100, "page": 64, "elem": "f16",
         "heads": 32, "kv_heads": 4, "dim": 128},
        # A few requests with narrow heads and small pages, in full precision.
        {"name": "attend_7x1501_f32", "kind": "attend", "seqs": 7, "len_lo": 0, "len_hi": 1501, "page": 16,
         "elem": "f32", "heads": 28, "kv_heads": 4, "dim": 64},
        # One request behind a very long document: the split over its length counts.
        {"name": "attend_1x131000", "kind": "attend", "seqs": 1, "len_lo": 131000, "len_hi": 131000, "page": 64,
         "elem": "f16", "heads": 32, "kv_heads": 4, "dim": 128},
        # A full server: many requests of every length, the pages' bytes count.
        {"name": "attend_64x16000", "kind": "attend", "seqs": 64, "len_lo": 1, "len_hi": 16000, "page": 64,
         "elem": "f16", "heads": 32, "kv_heads": 4, "dim": 128},
        # A chat's step of one layer.
        {"name": "step_1x4096", "kind": "step", "seqs": 1, "len_lo": 4096, "len_hi": 4096, "page": 64, "elem": "f16",
         "heads": 32, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half", "scaling": "none"},
        # A batch's step of one layer over 8-bit pages, past the trained context.
        {"name": "step_32x8192_q8", "kind": "step", "seqs": 32, "len_lo": 10, "len_hi": 8192, "page": 128,
         "elem": "q8_0", "heads": 32, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half", "scaling": "yarn"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["rotate", "append", "append", "attend", "attend", "attend", "step", "step"])
    kv_heads, group = rng.choice([(4, 8), (4, 8), (2, 8), (8, 4), (4, 7), (8, 1), (1, 16)])
    dim = rng.choice([128, 128, 128, 64, 96, 256] if kind != "rotate" else [128, 128, 64, 80, 96, 256])
    rot = rng.choice([dim, dim, dim // 2, 32])
    position = {"rot": rot, "layout": rng.choice(["half", "half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"])}
    if kind == "rotate":
        heads = rng.choice([kv_heads, kv_heads * group, kv_heads * (group + 1)])
        most = max(1, min(8192, 4096 * 36 * 128 // (heads * dim)))
        return {"kind": kind, "rows": _log(rng, 1, most), "heads": heads, "dim": dim, **position,
                "far": _log(rng, 8192, 131072), "spread": rng.random() < 0.5}
    case = {"kind": kind, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 32, 64, 128]), "elem": rng.choice(["f16", "f16", "f32", "q8_0", "q8_0"])}
    wide = max(1.0, kv_heads * dim / 512) * (2 if case["elem"] == "f32" else 1)
    if kind == "append":
        case.update(position, seqs=_log(rng, 1, 64), norm=rng.random() < 0.5, far=_log(rng, 1024, 100000))
        case["rows_hi"] = rng.choice([1, _log(rng, 1, max(1, min(1000, int(5000 / wide) // case["seqs"])))])
        case["rows_lo"] = rng.randint(min(1, case["rows_hi"]), case["rows_hi"])
        return case
    case["seqs"] = rng.choice([1, _log(rng, 1, 128), _log(rng, 1, 128)])
    most = min(131000 if kind == "attend" else 16000, int(500000 / wide) // case["seqs"])
    case["len_hi"] = _log(rng, 1, most)
    case["len_lo"] = rng.choice([0 if kind == "attend" else 1, min(100, case["len_hi"]), case["len_hi"]])
    if kind == "step":
        case.update(position)
    return case


# ---- sizes ------------------------------------------------------------------

def _spread_over(lo, hi, n):
    """n whole numbers over lo .. hi, hi among them."""
    out = [lo + (i * 7919) % (hi - lo + 1) for i in range(n)]
    out[-1] = hi
    return out


def _lens(case):
    """Rows each sequence attends (a step's own row among them)."""
    return _spread_over(case["len_lo"], case["len_hi"], case["seqs"])


def _runs(case):
    """The (first position, rows) of each sequence's appended rows."""
    rows = _spread_over(case["rows_lo"], case["rows_hi"], case["seqs"])
    return [((i * 104729 + 4095) % case["far"], n) for i, n in enumerate(rows)]


def _elem_bytes(elem):
    return {"f32": 4.0, "f16": 2.0, "q8_0": 34 / 32}[elem]


def work(case):
    if case["kind"] == "rotate":
        n = case["rows"] * case["heads"]
        return {"bytes": 8.0 * n * case["dim"] + 4.0 * case["rows"], "flops": 3.0 * n * case["rot"]}
    kv_dim, q_dim, es = case["kv_heads"] * case["dim"], case["heads"] * case["dim"], _elem_bytes(case["elem"])
    if case["kind"] == "append":
        n = sum(n for _, n in _runs(case)) * kv_dim
        back = 4.0 if case["elem"] == "f32" else 2.0
        return {"bytes": 2.0 * n * (4 + es + back), "flops": 8.0 * n}
    n, held = case["seqs"], sum(_lens(case))
    moved = 2 * held * kv_dim * es + 8.0 * n * q_dim
    if case["kind"] == "step":
        moved += n * kv_dim * (8 + 2 * (4 if case["elem"] == "f32" else 2))
    return {"bytes": moved, "flops": 4.0 * q_dim * held}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6007 + 11)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _keys(g, rows, heads, dim):
    """Keys as a model has them: a few channels of each head are much larger than the rest."""
    x = _randn(g, rows, heads, dim)
    x[..., 5::37] *= 6.0
    return x.reshape(rows, heads * dim)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _pages(g, case, longest):
    """A table of scattered pages, of a pool with some to spare: [sequences][pages], pages in the pool."""
    per_seq = -(-longest // case["page"])
    n = case["seqs"] * per_seq
    ids = torch.randperm(n + 3, generator=g, device="cuda")[:n]
    return ids.to(torch.int32).reshape(case["seqs"], per_seq).contiguous(), n + 3


def _inputs(case, seed):
    g, s = _gen(seed), {}
    if case["kind"] == "rotate":
        s["x"] = _randn(g, case["rows"], case["heads"] * case["dim"])
        if case["spread"]:
            s["at"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        else:
            first = max(0, case["far"] - case["rows"])
            s["at"] = torch.arange(first, first + case["rows"], device="cuda", dtype=torch.int32)
        return s
    h, d = case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        runs = _runs(case)
        s["table"], s["pool"] = _pages(g, case, max(at + n for at, n in runs))
        s["at"] = _ints([at + i for at, n in runs for i in range(n)])
        s["seq"] = _ints([i for i, (_, n) in enumerate(runs) for _ in range(n)])
        total = s["at"].shape[0]
    else:
        lens = _lens(case)
        s["table"], s["pool"] = _pages(g, case, max(lens))
        s["lens"] = _ints(lens)
        held = [n - 1 for n in lens] if case["kind"] == "step" else lens
        s["old_at"] = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in held])
        s["old_seq"] = torch.repeat_interleave(torch.arange(len(held), device="cuda", dtype=torch.int32),
                                               torch.tensor(held, device="cuda"))
        s["old_k"] = _keys(g, sum(held), h, d)
        s["old_v"] = _randn(g, sum(held), h * d)
        s["q"] = _randn(g, case["seqs"], case["heads"] * d)
        s["at"], s["seq"] = s["lens"] - 1, torch.arange(case["seqs"], device="cuda", dtype=torch.int32)
        total = case["seqs"]
    if case["kind"] != "attend":
        s["k"], s["v"] = _keys(g, total, h, d), _randn(g, total, h * d)
        s["qw"] = 1.0 + 0.1 * _randn(g, d)
        s["kw"] = 1.0 + 0.1 * _randn(g, d)
    return s


THETA = 1e6
FACTOR = 4.0
TRAINED = 32768


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import ramvamp_amd as rv

        if "rot" in case:
            s["rope"] = rv.Rope(case["dim"], THETA, rotary_dim=case["rot"], layout=case["layout"],
                                scaling=case["scaling"], factor=FACTOR, trained_positions=TRAINED)
        if case["kind"] == "rotate":
            s["out"] = torch.empty_like(s["x"])
        else:
            s["cache"] = rv.PagedKvCache(1, case["kv_heads"], case["dim"], s["pool"], case["page"], case["elem"])
            if "old_k" in s:
                s["cache"].append_rows(0, s["old_k"], s["old_v"], s["table"], s["old_at"], s["old_seq"])
                s["out"] = torch.empty_like(s["q"])
            s["cache"].synchronize()
    else:
        if "rot" in case:
            s["freq"], s["gain"] = _frequencies(case)
        if case["kind"] != "rotate":
            s["planes"] = [_empty(case, s["pool"]), _empty(case, s["pool"])]
            if "old_k" in s:
                _put(s, s["old_k"], s["old_v"], s["old_at"], s["old_seq"])
    for name in ("old_k", "old_v"):  # the pages hold them now
        s.pop(name, None)
    return s


# ---- the plain forms --------------------------------------------------------

def _frequencies(case):
    """Each pair's angle per position in 64 bits, and what cosine and sine are times."""
    r, base, gain = case["rot"], THETA, 1.0
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    if case["scaling"] == "ntk":
        base *= FACTOR ** (r / (r - 2))
    f = torch.exp(i * (-2.0 * math.log(base) / r))
    if case["scaling"] == "linear":
        f = f / FACTOR
    if case["scaling"] == "yarn":
        def pair_of(turns):  # the pair that makes so many turns within the trained positions
            return r * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), r - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / FACTOR * ramp
        gain = 0.1 * math.log(FACTOR) + 1
    return f, gain


def _rotated(s, x, at):
    """x [rows][heads][dim] at the positions."""
    case = s["case"]
    r, angle = case["rot"], at.double().unsqueeze(1) * s["freq"]
    c = (torch.cos(angle) * s["gain"]).float().unsqueeze(1)
    n = (torch.sin(angle) * s["gain"]).float().unsqueeze(1)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (
        slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., first], x[..., second]
    y = x.clone()
    y[..., first] = a * c - b * n
    y[..., second] = a * n + b * c
    return y


def _normed(x, weight):
    mean = (x.double() ** 2).sum(dim=-1, keepdim=True) / x.shape[-1]
    return x * (1.0 / torch.sqrt(mean + float(torch.tensor(EPS)))).float() * weight


def _heads(x, dim):
    return x.reshape(x.shape[0], -1, dim)


def _cut(x):
    """Values in blocks of 32: their codes and scales."""
    b = x.reshape(-1, BLOCK)
    step = b.abs().amax(dim=1) / torch.full((), 127.0, device=x.device).expand(b.shape[0])
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    y = b * inv.unsqueeze(1)
    whole = torch.trunc(y)
    codes = whole + torch.sign(y) * ((y - whole).abs() >= 0.5)
    return codes.to(torch.int8).reshape(x.shape), step.to(torch.float16).reshape(*x.shape[:-1], -1)


def _empty(case, pages):
    """One plane of the pool: every page's rows [pages * page][kv heads][dim]."""
    shape = (pages * case["page"], case["kv_heads"], case["dim"])
    if case["elem"] == "q8_0":
        return [torch.zeros(shape, device="cuda", dtype=torch.int8),
                torch.zeros(*shape[:2], case["dim"] // BLOCK, device="cuda", dtype=torch.float16)]
    return [torch.zeros(shape, device="cuda", dtype=torch.float16 if case["elem"] == "f16" else torch.float32)]


def _slots(s, at, seq):
    page = s["case"]["page"]
    return s["table"][seq.long(), (at // page).long()].long() * page + at % page


def _put(s, k, v, at, seq):
    slots, case = _slots(s, at, seq), s["case"]
    for plane, x in zip(s["planes"], (k, v)):
        x = _heads(x, case["dim"])
        held = _cut(x) if case["elem"] == "q8_0" else (x.to(plane[0].dtype),)
        for p, y in zip(plane, held):
            p[slots] = y


def _get(s, plane, slots):
    """Rows of a plane as the values they stand for, in the type that holds those."""
    x = plane[0][slots]
    if s["case"]["elem"] != "q8_0":
        return x
    b = x.float().reshape(*x.shape[:-1], -1, BLOCK) * plane[1][slots].float().unsqueeze(-1)
    return b.reshape(x.shape).to(torch.float16)


def _read_back(s):
    slots = _slots(s, s["at"], s["seq"])
    return tuple(_get(s, p, slots).reshape(slots.shape[0], -1) for p in s["planes"])


def _attended(s, q):
    """Softmax attention of q [sequences][heads][dim] over each sequence's pages."""
    case = s["case"]
    n, kvh, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    g, longest = case["heads"] // kvh, max(case["len_hi"], 1)
    t = torch.arange(longest, device="cuda")
    slots = s["table"].long()[:, t // page] * page + t % page
    dead = (t >= s["lens"].unsqueeze(1)).reshape(n, 1, longest, 1)
    k, v = (_get(s, p, slots).permute(0, 2, 1, 3).float() for p in s["planes"])
    k, v = k.masked_fill(dead, 0).contiguous(), v.masked_fill(dead, 0).contiguous()
    qt = q.reshape(n, kvh, g, d).transpose(2, 3).contiguous()
    x = (k @ qt * d ** -0.5).masked_fill(dead, -math.inf)
    top = x.amax(dim=2, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(dim=2).unsqueeze(3)
    o = p.transpose(2, 3).contiguous() @ v
    return torch.where(total > 0, o / total, torch.zeros_like(o)).reshape(n, kvh * g * d)


def _plain(s):
    case, d = s["case"], s["case"]["dim"]
    if case["kind"] == "rotate":
        return _rotated(s, _heads(s["x"], d), s["at"]).reshape(s["x"].shape)
    if case["kind"] == "attend":
        return _attended(s, _heads(s["q"], d))
    k = _heads(s["k"], d)
    if case["kind"] == "step" or case["norm"]:
        k = _normed(k, s["kw"])
    _put(s, _rotated(s, k, s["at"]), s["v"], s["at"], s["seq"])
    if case["kind"] == "append":
        return _read_back(s)
    q = _rotated(s, _normed(_heads(s["q"], d), s["qw"]), s["at"])
    return (_attended(s, q), *_read_back(s))


# ---- the framework's calls --------------------------------------------------

def _own(s):
    import ramvamp_amd as rv

    case = s["case"]
    if case["kind"] == "rotate":
        return rv.rope_rows(s["x"], s["at"], s["rope"], s["out"])
    cache, scale = s["cache"], case["dim"] ** -0.5
    if case["kind"] == "attend":
        return rv.paged_attention(s["q"], cache, 0, s["table"], s["lens"], scale, s["out"])
    if case["kind"] == "append":
        cache.append_rows(0, s["k"], s["v"], s["table"], s["at"], s["seq"], rope=s["rope"],
                          k_norm_w=s["kw"] if case["norm"] else None, eps=EPS)
        return cache.read_rows(0, s["table"], s["at"], s["seq"])
    rv.paged_decode_step(cache, 0, s["q"], s["k"], s["v"], s["qw"], s["kw"], EPS, s["rope"], s["table"], s["at"],
                         scale, s["out"])
    return (s["out"], *cache.read_rows(0, s["table"], s["at"]))


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ------------------------------------------------

def _turned64(case, x, at, stored):
    """x [rows][heads][dim] in 64 bits, rotated pair by pair. What is to be stored in
    fewer bits is rounded to 32 where the definition says so, since a value next to
    a border of its format would otherwise fall on the other side."""
    fit = (lambda y: y.float().double()) if stored else (lambda y: y)
    r, y = case["rot"], x.clone()
    pos = at.double().reshape(-1, 1)
    low = r * math.log(TRAINED / (64 * math.pi)) / math.log(THETA) / 2
    high = r * math.log(TRAINED / (2 * math.pi)) / math.log(THETA) / 2
    low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
    for i in range(r // 2):
        f, gain = THETA ** (-2 * i / r), 1.0
        if case["scaling"] == "linear":
            f /= FACTOR
        elif case["scaling"] == "ntk":
            f = (THETA * FACTOR ** (r / (r - 2))) ** (-2 * i / r)
        elif case["scaling"] == "yarn":
            share = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f, gain = f * (1 - share) + f / FACTOR * share, 1 + 0.1 * math.log(FACTOR)
        c, n = fit(gain * torch.cos(pos * f)), fit(gain * torch.sin(pos * f))
        j, k = (i, i + r // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        y[..., j] = fit(fit(x[..., j] * c) - fit(x[..., k] * n))
        y[..., k] = fit(fit(x[..., j] * n) + fit(x[..., k] * c))
    return y


def _scaled64(x, weight, stored):
    fit = (lambda y: y.float().double()) if stored else (lambda y: y)
    eps = float(torch.tensor(EPS, dtype=torch.float32))
    inv = fit(1.0 / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps))
    return fit(fit(x * inv) * weight.double())


def _held64(x, elem):
    """A stored row's values, the format's own steps rounded to 32 bits as it says."""
    if elem == "f32":
        return x.float().double()
    if elem == "f16":
        return x.float().half().double()
    b = x.float().double().reshape(-1, BLOCK)
    step = (b.abs().amax(1) / 127.0).float()
    inv = torch.where(step > 0, (1.0 / step.double()).float(), torch.zeros_like(step)).double()
    y = (b * inv.unsqueeze(1)).float().double()
    codes = torch.floor(y.abs() + 0.5) * torch.sign(y)
    return (codes * step.half().double().unsqueeze(1)).half().double().reshape(x.shape)


def exact(case, seed):
    s, d = _inputs(case, seed), case["dim"]
    if case["kind"] == "rotate":
        x = s["x"].double().reshape(case["rows"], case["heads"], d)
        return _turned64(case, x, s["at"], False).reshape(s["x"].shape)
    kvh, elem = case["kv_heads"], case["elem"]
    if case["kind"] != "attend":
        k = s["k"].double().reshape(-1, kvh, d)
        if case["kind"] == "step" or case["norm"]:
            k = _scaled64(k, s["kw"], True)
        k = _held64(_turned64(case, k, s["at"], True), elem).reshape(-1, kvh * d)
        v = _held64(s["v"], elem)
        if case["kind"] == "append":
            return k, v
    q = s["q"].double().reshape(case["seqs"], case["heads"], d)
    if case["kind"] == "step":
        q = _turned64(case, _scaled64(q, s["qw"], False), s["at"], False)
    out, at = torch.zeros_like(q), 0
    for i, length in enumerate(_lens(case)):
        old = length - 1 if case["kind"] == "step" else length
        ks, vs = _held64(s["old_k"][at:at + old], elem), _held64(s["old_v"][at:at + old], elem)
        at += old
        if case["kind"] == "step":
            ks, vs = torch.cat([ks, k[i:i + 1]]), torch.cat([vs, v[i:i + 1]])
        if length == 0:
            continue
        for h in range(kvh):
            part, mine = slice(h * d, (h + 1) * d), slice(h * case["heads"] // kvh, (h + 1) * case["heads"] // kvh)
            x = q[i, mine] @ ks[:, part].T.contiguous() * (1.0 / math.sqrt(d))
            out[i, mine] = torch.softmax(x, dim=1) @ vs[:, part]
    out = out.reshape(case["seqs"], -1)
    return (out, k, v) if case["kind"] == "step" else out
