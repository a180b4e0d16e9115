"""The quantized cache, the attention that reads it, and decode for a batch that
shares a prefix, as timed cases.

The shapes are the model's attention (32 query heads over 4 kv heads of 128)
and neighbours of it (other head counts), at the lengths a serving loop meets.
A case is a dict of plain values; its ``kind`` picks the operator:

- ``write``: rows appended to a Q8_0 cache and read back;
- ``decode``: one token's attention over a Q8_0 cache;
- ``rows``: a chunk's causal attention over a Q8_0 cache, full precision;
- ``shared``: one token of each of ``seqs`` sequences, which attend a prefix
  they share (``ctx`` rows of one cache) and ragged rows of their own.

A Q8_0 cache keeps a row in blocks of 32 values: the block's scale is its
largest magnitude over 127 and a value's code its product with the scale's
reciprocal, rounded half away from zero, each step in 32 bits; the scale is
stored in f16. A stored value reads as the f16 nearest to scale times code.
"""
from __future__ import annotations

import math

import torch

own = False

DIM = 128
SCALE = DIM ** -0.5
BLOCK = 32


def listed():
    return [
        # One token's rows into a layer of the cache and back: launches count.
        {"name": "write_1_at_4095", "kind": "write", "rows": 1, "ctx": 4095, "heads": 32, "kv_heads": 4},
        # A long prompt's chunk written whole.
        {"name": "write_4096_at_0", "kind": "write", "rows": 4096, "ctx": 0, "heads": 32, "kv_heads": 4},
        # A token early in a conversation.
        {"name": "decode_100", "kind": "decode", "ctx": 100, "heads": 32, "kv_heads": 4},
        # A token just past the model's default context.
        {"name": "decode_4097", "kind": "decode", "ctx": 4097, "heads": 32, "kv_heads": 4},
        # A token behind a very long document: the cache's bytes are what counts.
        {"name": "decode_131000", "kind": "decode", "ctx": 131000, "heads": 32, "kv_heads": 4},
        # A follow-up turn of a chat: a ragged few rows behind what is cached.
        {"name": "rows_77_at_901", "kind": "rows", "rows": 77, "ctx": 901, "heads": 32, "kv_heads": 4},
        # A chunk behind a reused prefix.
        {"name": "rows_512_at_3449", "kind": "rows", "rows": 512, "ctx": 3449, "heads": 32, "kv_heads": 4},
        # A late chunk of a long prompt: the largest products.
        {"name": "rows_1000_at_12000", "kind": "rows", "rows": 1000, "ctx": 12000, "heads": 32, "kv_heads": 4},
        # A few samples of one prompt, in a cache of full precision, at odd sizes.
        {"name": "shared_7x1501_f32", "kind": "shared", "seqs": 7, "ctx": 1501, "tail_lo": 1, "tail_hi": 60,
         "elem": "f32", "heads": 32, "kv_heads": 4},
        # Requests behind a long system prompt, whose own turns weigh about as much as it does.
        {"name": "shared_16x4096_q8", "kind": "shared", "seqs": 16, "ctx": 4096, "tail_lo": 0, "tail_hi": 2000,
         "elem": "q8_0", "heads": 32, "kv_heads": 4},
        # Many questions about one document.
        {"name": "shared_32x8192_q8", "kind": "shared", "seqs": 32, "ctx": 8192, "tail_lo": 1, "tail_hi": 300,
         "elem": "q8_0", "heads": 32, "kv_heads": 4},
        # The same at the model's own cache format, longer and wider: the largest shared product.
        {"name": "shared_64x16000_f16", "kind": "shared", "seqs": 64, "ctx": 16000, "tail_lo": 1, "tail_hi": 700,
         "elem": "f16", "heads": 32, "kv_heads": 4},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["write", "decode", "decode", "rows", "rows", "shared", "shared", "shared"])
    kv_heads, group = rng.choice([(4, 8), (4, 8), (2, 8), (8, 4), (4, 7), (8, 1)])
    case = {"kind": kind, "heads": kv_heads * group, "kv_heads": kv_heads}
    if kind == "write":
        case.update(rows=_log(rng, 1, 4096), ctx=_log(rng, 1, 8192))
    elif kind == "decode":
        case.update(ctx=_log(rng, 1, 65000))
    elif kind == "rows":
        case.update(rows=_log(rng, 2, 1000), ctx=rng.choice([0, _log(rng, 1, 12000)]))
    else:
        lo = rng.choice([0, 1, 10])
        case.update(seqs=_log(rng, 2, 64), ctx=_log(rng, 64, 16000), tail_lo=lo, tail_hi=lo + _log(rng, 1, 700),
                    elem=rng.choice(["q8_0", "q8_0", "f16", "f16", "f32"]))
        if case["elem"] == "f32":
            case["ctx"] = min(case["ctx"], 4000)
    return case


# ---- sizes ------------------------------------------------------------------

def _tails(case):
    """Each sequence's own rows: ragged over the case's range, its ends among them."""
    span = case["tail_hi"] - case["tail_lo"] + 1
    lens = [case["tail_lo"] + (i * 7919) % span for i in range(case["seqs"])]
    lens[-1] = case["tail_hi"]
    return lens


def _elem_bytes(elem):
    return {"f32": 4.0, "f16": 2.0, "q8_0": 34 / 32}[elem]


def work(case):
    kv_dim, q_dim = case["kv_heads"] * DIM, case["heads"] * DIM
    if case["kind"] == "write":
        n = 2 * case["rows"] * kv_dim
        return {"bytes": n * (4 + 4 + 34 / 32), "flops": 6.0 * n}
    if case["kind"] == "decode":
        rows, seen, held = 1, case["ctx"], case["ctx"]
        es = 34 / 32
    elif case["kind"] == "rows":
        rows = case["rows"]
        held = case["ctx"] + rows
        seen = rows * case["ctx"] + rows * (rows + 1) // 2
        es = 34 / 32
    else:
        rows, tails = case["seqs"], sum(_tails(case))
        held = case["ctx"] + tails
        seen = rows * case["ctx"] + tails
        es = _elem_bytes(case["elem"])
    return {"bytes": 2 * held * kv_dim * es + 2 * 4 * rows * q_dim, "flops": 4.0 * q_dim * seen}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _keys(g, rows, kv_heads):
    """Keys as a model has them: a few channels of each head are much larger than the rest."""
    x = _randn(g, rows, kv_heads, DIM)
    x[..., 5::37] *= 6.0
    return x.reshape(rows, kv_heads * DIM)


def _values(g, rows, kv_heads):
    return _randn(g, rows, kv_heads * DIM)


def _rows_of(case, seed):
    """The case's float rows: those cached before the call, and the call's own."""
    g, h = _gen(seed), case["kv_heads"]
    s = {}
    if case["kind"] == "write":
        s["k"], s["v"] = _keys(g, case["rows"], h), _values(g, case["rows"], h)
        return s
    held = case["ctx"] + (case["rows"] if case["kind"] == "rows" else 0)
    n = {"decode": 1, "rows": case.get("rows"), "shared": case.get("seqs")}[case["kind"]]
    s["k"], s["v"] = _keys(g, held, h), _values(g, held, h)
    s["q"] = _randn(g, n, case["heads"] * DIM)
    if case["kind"] == "shared":
        total = n * max(case["tail_hi"], 1)
        s["tk"], s["tv"] = _keys(g, total, h), _values(g, total, h)
    return s


def _cut(x):
    """Rows as the blocks of a Q8_0 cache: codes [rows][blocks][32], scales [rows][blocks]."""
    b = x.reshape(x.shape[0], -1, BLOCK)
    step = b.abs().amax(dim=2) / torch.full((), 127.0, device=x.device).expand(b.shape[:2])
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    y = b * inv.unsqueeze(2)
    whole = torch.trunc(y)
    codes = whole + torch.sign(y) * ((y - whole).abs() >= 0.5)
    return codes.to(torch.int8), step.to(torch.float16)


def _stored(x, elem):
    """What a cache of this type holds of the rows."""
    if elem == "q8_0":
        return _cut(x)
    return (x.to(torch.float16),) if elem == "f16" else (x,)


def prepare(case, seed):
    s = _rows_of(case, seed)
    s["case"] = case
    elem, h = case.get("elem", "q8_0"), case["kv_heads"]
    if case["kind"] == "shared":
        lens = _tails(case)
        s["lens"] = torch.tensor(lens, device="cuda")
    if own:
        import ramvamp_amd as rv

        if case["kind"] == "write":
            s["cache"] = rv.KvCache(1, h, DIM, case["ctx"] + case["rows"], "q8_0")
            if case["ctx"]:
                zeros = torch.zeros(case["ctx"], h * DIM, device="cuda")
                s["cache"].append_rows(0, zeros, zeros)
        else:
            s["cache"] = rv.KvCache(1, h, DIM, s["k"].shape[0], elem)
            s["cache"].append_rows(0, s["k"], s["v"])
            s["out"] = torch.empty_like(s["q"])
        if case["kind"] == "shared":
            room = max(case["tail_hi"], 1)
            s["own_rows"] = rv.KvCache(case["seqs"], h, DIM, room, elem)
            for i, n in enumerate(lens):
                if n:
                    s["own_rows"].append_rows(i, s["tk"][i * room:i * room + n], s["tv"][i * room:i * room + n])
            s["own_rows"].synchronize()
        s["cache"].synchronize()
    elif case["kind"] != "write":
        s["ks"], s["vs"] = _stored(s["k"], elem), _stored(s["v"], elem)
        if case["kind"] == "shared":
            s["tks"], s["tvs"] = _stored(s["tk"], elem), _stored(s["tv"], elem)
    if case["kind"] != "write":
        for name in ("k", "v", "tk", "tv"):  # the caches hold them now
            s.pop(name, None)
    return s


# ---- the plain forms --------------------------------------------------------

def _value(stored, kv_heads):
    """The values a cache's rows stand for, [kv_heads][rows][DIM], in 32 bits."""
    if len(stored) == 2:
        codes, scales = stored
        x = (codes.float() * scales.float().unsqueeze(2)).to(torch.float16)
    else:
        x = stored[0]
    return x.float().reshape(x.shape[0], kv_heads, DIM).transpose(0, 1)


def _softmax_times(scores, values):
    """softmax over the last axis of ``scores``, times ``values``; -inf is masked."""
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top)
    return (p @ values) / p.sum(dim=-1, keepdim=True)


def _plain(s):
    case = s["case"]
    kvh, heads = case["kv_heads"], case["heads"]
    g = heads // kvh
    if case["kind"] == "write":
        back = []
        for x in (s["k"], s["v"]):
            codes, scales = _cut(x)
            back.append((codes.float() * scales.float().unsqueeze(2)).to(torch.float16).float().reshape(x.shape))
        return tuple(back)
    n = s["q"].shape[0]
    q = s["q"].reshape(n, kvh, g, DIM).permute(1, 0, 2, 3).reshape(kvh, n * g, DIM)
    k, v = _value(s["ks"], kvh), _value(s["vs"], kvh)
    scores = (q @ k.transpose(1, 2).contiguous()) * SCALE
    if case["kind"] == "rows":
        at = torch.arange(k.shape[1], device="cuda")
        limit = case["ctx"] + torch.arange(n, device="cuda").repeat_interleave(g)
        scores = scores.masked_fill(at > limit.unsqueeze(1), -math.inf)
    if case["kind"] == "shared":
        room = max(case["tail_hi"], 1)
        tk = _value(s["tks"], kvh).reshape(kvh, n, room, DIM)
        tv = _value(s["tvs"], kvh).reshape(kvh, n, room, DIM)
        mine = (q.reshape(kvh, n, g, DIM) @ tk.transpose(2, 3).contiguous()) * SCALE
        empty = torch.arange(room, device="cuda") >= s["lens"].reshape(1, n, 1, 1)
        mine = mine.masked_fill(empty, -math.inf)
        top = torch.maximum(scores.amax(dim=-1), mine.amax(dim=-1).reshape(kvh, n * g)).unsqueeze(2)
        p, t = torch.exp(scores - top), torch.exp(mine - top.reshape(kvh, n, g, 1))
        sums = p.sum(dim=-1) + t.sum(dim=-1).reshape(kvh, n * g)
        o = (p @ v + (t @ tv).reshape(kvh, n * g, DIM)) / sums.unsqueeze(2)
    else:
        o = _softmax_times(scores, v)
    return o.reshape(kvh, n, g, DIM).permute(1, 0, 2, 3).reshape(n, heads * DIM)


# ---- the framework's calls --------------------------------------------------

def _own(s):
    import ramvamp_amd as rv

    case, kv = s["case"], s["cache"]
    if case["kind"] == "write":
        kv.truncate(case["ctx"])
        kv.append_rows(0, s["k"], s["v"])
        return kv.read_rows(0, case["ctx"], case["rows"])
    if case["kind"] == "decode":
        rv.decode_attention(s["q"], kv, 0, SCALE, None, s["out"])
    elif case["kind"] == "rows":
        rv.attention_at_rows(s["q"], kv, 0, case["ctx"], SCALE, s["out"])
    else:
        rv.decode_attention_shared(s["q"], kv, 0, case["ctx"], s["own_rows"], 0, SCALE, s["out"])
    return s["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ------------------------------------------------

def _held64(x, elem):
    """A stored row's values. The format rounds the step, its reciprocal and a value's
    product with it to 32 bits and the scale to f16, so this does too."""
    if elem == "f32":
        return x.double()
    if elem == "f16":
        return x.half().double()
    b = x.double().reshape(x.shape[0], -1, BLOCK)
    step = (b.abs().amax(2) / 127.0).float()
    inv = torch.where(step > 0, (1.0 / step.double()).float(), torch.zeros_like(step)).double()
    y = (b * inv.unsqueeze(2)).float().double()
    codes = torch.floor(y.abs() + 0.5) * torch.sign(y)
    return (codes * step.half().double().unsqueeze(2)).half().double().reshape(x.shape)


def exact(case, seed):
    s = _rows_of(case, seed)
    elem, kvh, heads = case.get("elem", "q8_0"), case["kv_heads"], case["heads"]
    g = heads // kvh
    if case["kind"] == "write":
        return _held64(s["k"], elem), _held64(s["v"], elem)
    k, v, q = _held64(s["k"], elem), _held64(s["v"], elem), s["q"].double()
    n = q.shape[0]
    out = torch.empty(n, heads, DIM, device="cuda", dtype=torch.float64)
    shared = case["kind"] == "shared"
    if shared:
        room, lens = max(case["tail_hi"], 1), _tails(case)
        tk, tv = _held64(s["tk"], elem), _held64(s["tv"], elem)
    for h in range(heads):
        part = slice((h // g) * DIM, (h // g + 1) * DIM)
        qh = q[:, h * DIM:(h + 1) * DIM] * SCALE
        x = qh @ k[:, part].T.contiguous()
        if case["kind"] == "rows":
            for r in range(n):
                x[r, case["ctx"] + r + 1:] = -math.inf
        if not shared:
            out[:, h] = torch.softmax(x, dim=1) @ v[:, part]
            continue
        own_x = torch.full((n, room), -math.inf, device="cuda", dtype=torch.float64)
        for i, m in enumerate(lens):
            own_x[i, :m] = tk[i * room:i * room + m, part] @ qh[i]
        w = torch.softmax(torch.cat([x, own_x], dim=1), dim=1)
        out[:, h] = w[:, :x.shape[1]] @ v[:, part]
        for i, m in enumerate(lens):
            out[i, h] += w[i, x.shape[1]:x.shape[1] + m] @ tv[i * room:i * room + m, part]
    return out.reshape(n, heads * DIM)
