"""Rotary positions, the paged cache's rows, attention over its pages and a
batch's step, against their definitions in 64 bits."""
import threading

import numpy as np
import pytest

import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from rows_util import EPS32, attend, check, stored

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e6


def ints(x):
    torch = torch_cuda()
    return torch.tensor(np.asarray(x, np.int64).astype(np.int32), device="cuda")


def scale_of(hd):
    return float(np.float32(1.0) / np.sqrt(np.float32(hd)))


def rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[:, 5::37] *= 6
    return x


# ---- rotary positions -------------------------------------------------------------

def turns(rope, pos):
    """Cosine and sine of each pair, rounded to 32 bits, [rows][pairs]."""
    f, gain = rope.frequencies()
    a = np.asarray(pos, np.float64)[:, None] * f
    return (gain * np.cos(a)).astype(np.float32), (gain * np.sin(a)).astype(np.float32)


def rotated(x, c, s, r, layout):
    """x [rows][heads][dim] in f64 by the f32 cosines and sines given."""
    x = np.asarray(x, np.float64)
    c, s = c[:, None].astype(np.float64), s[:, None].astype(np.float64)
    y = x.copy()
    a, b = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def rotation_bound(x, r, layout, gain=1.0):
    """Three roundings of f32 in each value (two products, their sum), and cosine
    and sine at most one step of f32 apart from the host's: 2 half steps each."""
    x = np.abs(np.asarray(x, np.float64))
    b = np.zeros_like(x)
    p, q = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    both = (x[..., p] + x[..., q]) * gain
    b[..., p] = b[..., q] = both * 4 * EPS32 + 2.0 ** -148
    return b


@pytest.mark.parametrize("hd,r,layout,scaling", [
    (128, 128, "half", "none"), (128, 128, "interleaved", "yarn"), (80, 32, "interleaved", "linear"),
    (80, 20, "half", "ntk"), (96, 96, "half", "linear"), (64, 2, "half", "none"), (64, 2, "interleaved", "none"),
    (7, 6, "half", "ntk"), (7, 6, "interleaved", "none"), (21, 14, "half", "yarn"), (512, 512, "half", "none"),
    (512, 510, "interleaved", "yarn"), (256, 64, "half", "none"), (33, 32, "half", "none"),
])
@pytest.mark.parametrize("n,heads", [(1, 1), (1, 36), (3, 5), (70, 2), (1030, 3)])
def test_rope_rows(hd, r, layout, scaling, n, heads):
    torch = torch_cuda()
    say(f"case rope {(hd, r, layout, scaling, n, heads)}")
    rng = np.random.default_rng(hd + r + n)
    rope = rv.Rope(hd, THETA, r, layout, scaling, factor=4.0, trained_positions=32768)
    pos = rng.integers(0, 200000, n)
    pos[0] = 0 if n % 2 else 131071
    if n > 2:
        pos[1:3] = [-5, 2 ** 31 - 1]
    x = rng.standard_normal((n, heads * hd)).astype(np.float32)
    got = host(rv.rope_rows(dev(x), ints(pos), rope)).reshape(n, heads, hd)
    xh = x.reshape(n, heads, hd)
    c, s = turns(rope, pos)
    err = np.abs(got - rotated(xh, c, s, r, layout))
    gain = rope.frequencies()[1]
    assert np.all(err <= rotation_bound(xh, r, layout, gain)), float(err.max())
    assert np.array_equal(got[..., r:], xh[..., r:])
    # In place, and as columns of a wider buffer beside the input's own: the same bits.
    wide = torch.full((n, 2 * heads * hd + 5), 7.0, device="cuda")
    a, b = wide[:, 1:1 + heads * hd], wide[:, 2 + heads * hd:2 + 2 * heads * hd]
    a.copy_(dev(x))
    rv.rope_rows(a, ints(pos), rope, b)
    assert np.array_equal(host(b).reshape(got.shape).view(np.uint32), got.view(np.uint32))
    assert np.array_equal(host(a), x)
    rv.rope_rows(a, ints(pos), rope, a)
    w = host(wide)
    assert np.array_equal(w[:, 1:1 + heads * hd].copy().view(np.uint32), got.reshape(n, -1).view(np.uint32))
    assert np.all(w[:, 0] == 7) and np.all(w[:, 1 + heads * hd] == 7) and np.all(w[:, 2 + 2 * heads * hd:] == 7)


def test_rope_rows_special_values():
    """Infinities and NaNs stay in their pairs; a rotation back returns the rows."""
    torch = torch_cuda()
    say("case rope special values")
    rope = rv.Rope(64, THETA, 32)
    x = np.random.default_rng(0).standard_normal((4, 64)).astype(np.float32)
    bad = x.copy()
    bad[0, 3], bad[1, 20], bad[2, 40] = np.inf, np.nan, np.nan
    y, z = host(rv.rope_rows(dev(x), ints([5, 6, 7, 8]), rope)), host(rv.rope_rows(dev(bad), ints([5, 6, 7, 8]), rope))
    touched = np.zeros((4, 64), bool)
    touched[0, [3, 19]] = touched[1, [4, 20]] = touched[2, 40] = True
    assert np.array_equal(y[~touched], z[~touched]) and not np.any(np.isfinite(z[touched]))
    back = host(rv.rope_rows(rv.rope_rows(dev(x), ints([9] * 4), rope), ints([-9] * 4), rope))
    # Twice the bound of one turn, the second over values at most sqrt(2) times as large.
    assert np.all(np.abs(back - x) <= 12 * EPS32 * np.abs(x).max() * 2)
    assert rv.rope_rows(torch.empty(0, 64, device="cuda"), ints([]), rope).shape == (0, 64)


def test_rope_rows_on_a_side_stream_and_in_a_graph():
    torch = torch_cuda()
    say("case rope stream and graph")
    rope = rv.Rope(128, THETA)
    x, at = dev(np.random.default_rng(1).standard_normal((300, 512))), ints(np.arange(300))
    want = host(rv.rope_rows(x, at, rope))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = rv.rope_rows(x, at, rope)
    side.synchronize()
    assert np.array_equal(host(y), want)
    out, g = torch.empty_like(x), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rv.rope_rows(x, at, rope, out)
    for i in range(4):
        at.add_(1)
        out.fill_(float("nan"))
        g.replay()
        assert np.array_equal(host(out), host(rv.rope_rows(x, at, rope)))


# ---- rows in and out ----------------------------------------------------------------

def everything(cache, layer=0):
    """All rows of a layer, (k, v) [pages * page_rows][kv_dim]."""
    n = cache.n_pages * cache.page_rows
    ident = ints(np.arange(cache.n_pages)[None])
    k, v = cache.read_rows(layer, ident, ints(np.arange(n)), ints(np.zeros(n)))
    cache.device_status()
    return host(k), host(v)


def tables(rng, n_seqs, pages, spare=3):
    ids = rng.permutation(n_seqs * pages + spare)
    return ids[:n_seqs * pages].reshape(n_seqs, pages), n_seqs * pages + spare


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,hd,page", [(4, 128, 64), (1, 32, 8), (2, 96, 16), (3, 256, 32), (2, 512, 8),
                                          (2, 20, 8), (1, 7, 16), (5, 1, 8)])
def test_rows_come_back_as_stored_and_nothing_else_changes(elem, n_kv, hd, page):
    torch = torch_cuda()
    if elem == "q8_0" and hd % 32:
        pytest.skip("Q8_0 rows are blocks of 32")
    say(f"case rows {(elem, n_kv, hd, page)}")
    rng = np.random.default_rng(hd + page)
    table, pool = tables(rng, 3, 4)
    c = rv.PagedKvCache(2, n_kv, hd, pool, page, elem)
    n, kvd = 37, n_kv * hd
    flat = rng.permutation(3 * 4 * page)[:n]  # distinct places
    seq, pos = flat // (4 * page), flat % (4 * page)
    k, v = rows(rng, n, kvd), rows(rng, n, kvd)
    k[0, 0], v[1, 0], k[2, 0], v[3, 0], k[4, 0] = np.inf, np.nan, 7e4, -7e4, 1e-6
    c.append_rows(1, dev(k), dev(v), ints(table), ints(pos), ints(seq))
    gk, gv = c.read_rows(1, ints(table), ints(pos), ints(seq))
    assert gk.dtype == (torch.float32 if elem == "f32" else torch.float16)
    with np.errstate(over="ignore"):
        wk, wv = stored(k, elem), stored(v, elem)
    assert np.array_equal(host(gk).astype(np.float32), wk, equal_nan=True)
    assert np.array_equal(host(gv).astype(np.float32), wv, equal_nan=True)
    for got, want in zip(everything(c, 1), (wk, wv)):
        full = np.zeros((pool * page, kvd), np.float32)
        full[table[seq, pos // page] * page + pos % page] = want
        assert np.array_equal(got.astype(np.float32), full, equal_nan=True)
    for got in everything(c, 0):
        assert not np.any(got)
    only = torch.full((n, kvd), 3.0, dtype=gk.dtype, device="cuda")
    c.read_rows(1, ints(table), ints(pos), ints(seq), v=only)
    assert np.array_equal(host(only).astype(np.float32), wv, equal_nan=True)


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("skip", [1, 2, 3])
def test_rows_into_tensors_at_any_element(elem, skip):
    """k and v views that begin at an element's boundary alone; then V alone."""
    torch = torch_cuda()
    say(f"case rows at any element {(elem, skip)}")
    rng = np.random.default_rng(skip)
    c = rv.PagedKvCache(1, 2, 32, 3, 8, elem)
    k, v = rows(rng, 5, 64), rows(rng, 5, 64)
    t, at, seq = ints([[2, 0]]), ints([3, 9, 0, 12, 7]), ints([0] * 5)
    wide = torch.full((2 * 5 * 64 + 16,), 9.0, device="cuda")
    kin, vin = wide[skip:skip + 320].view(5, 64), wide[skip + 320:skip + 640].view(5, 64)
    kin.copy_(dev(k)), vin.copy_(dev(v))
    c.append_rows(0, kin, vin, t, at, seq)
    dt = torch.float32 if elem == "f32" else torch.float16
    buf = torch.full((2 * 320 + 16,), 9.0, device="cuda", dtype=dt)
    gk, gv = buf[skip:skip + 320].view(5, 64), buf[skip + 320:skip + 640].view(5, 64)
    c.read_rows(0, t, at, seq, k=gk, v=gv)
    assert np.array_equal(host(gk).astype(np.float32), stored(k, elem))
    assert np.array_equal(host(gv).astype(np.float32), stored(v, elem))
    assert torch.all(buf[:skip] == 9) and torch.all(buf[skip + 640:] == 9)
    gk.fill_(5)
    got = c.read_rows(0, t, at, seq, v=gv)
    assert got[0] is None and torch.all(gk == 5) and np.array_equal(host(gv).astype(np.float32), stored(v, elem))


def test_padding_and_refused_rows_write_nothing_and_are_recorded():
    torch = torch_cuda()
    say("case refused rows")
    rng = np.random.default_rng(3)
    c = rv.PagedKvCache(1, 2, 64, 6, 8, "f16")
    table = ints([[0, 1, 99], [2, -1, 3]])  # two entries name no page
    k, v = rows(rng, 8, 128), rows(rng, 8, 128)
    pos, seq = [0, -1, 17, 9, 24, 3, 3, 23], [0, 0, 0, 1, 0, 2, -7, 1]
    c.append_rows(0, dev(k), dev(v), table, ints(pos), ints(seq))
    with pytest.raises(rv.KvError) as e:
        c.device_status()
    assert e.value.variant in ("PageOutOfRange", "SequenceOutOfRange", "PositionOutOfTable")
    c.device_status()  # read once
    got = everything(c)
    for g, x in zip(got, (k, v)):
        want = np.zeros((48, 128), np.float32)
        want[0], want[3 * 8 + 7] = stored(x[0:1], "f16")[0], stored(x[7:8], "f16")[0]
        assert np.array_equal(g.astype(np.float32), want)
    for p, s, variant, fields in [
            (17, 0, "PageOutOfRange", dict(layer=0, row=0, page=99, n_pages=6)),
            (9, 1, "PageOutOfRange", dict(layer=0, row=0, page=2 ** 32 - 1, n_pages=6)),
            (24, 0, "PositionOutOfTable", dict(layer=0, row=0, position=24, positions=24)),
            (3, 2, "SequenceOutOfRange", dict(layer=0, row=0, sequence=2, n_seqs=2))]:
        c.append_rows(0, dev(k[:1]), dev(v[:1]), table, ints([p]), ints([s]))
        with pytest.raises(rv.KvError) as e:
            c.device_status()
        assert e.value.variant == variant and {f: e.value.fields[f] for f in fields} == fields
        out = [torch.full((1, 128), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        c.read_rows(0, table, ints([p]), ints([s]), *out)
        with pytest.raises(rv.KvError) as e:
            c.device_status()
        assert e.value.variant == variant and not host(out[0]).any() and not host(out[1]).any()
    out = c.read_rows(0, table, ints([-1, 0]))
    assert not host(out[0])[0].any() and np.array_equal(host(out[0])[1], got[0][16])
    c.device_status()
    for g, w in zip(everything(c), got):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("n_kv,hd,r,layout,scaling", [
    (4, 128, 128, "half", "none"), (4, 128, 64, "interleaved", "ntk"), (2, 96, 96, "half", "yarn"),
    (1, 64, 10, "half", "linear"), (2, 20, 14, "interleaved", "none"), (1, 512, 512, "half", "yarn"),
    (9, 256, 32, "interleaved", "none"), (2, 9, 8, "half", "none"),
])
def test_append_norms_and_rotates(norm, n_kv, hd, r, layout, scaling):
    torch = torch_cuda()
    say(f"case append {(norm, n_kv, hd, r, layout, scaling)}")
    rng = np.random.default_rng(hd + r)
    rope = rv.Rope(hd, THETA, r, layout, scaling, factor=4.0, trained_positions=32768)
    n, page, kvd = 19, 16, n_kv * hd
    table, pool = tables(rng, 2, 4)
    pos, seq = np.concatenate([np.arange(40, 50), np.arange(3, 12)]), np.repeat([0, 1], [10, 9])
    k, v, w = rows(rng, n, kvd), rows(rng, n, kvd), (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    qkv = torch.zeros(n, 2 * kvd + 3, device="cuda")  # strided rows
    qkv[:, 1:1 + kvd], qkv[:, 2 + kvd:2 + 2 * kvd] = dev(k), dev(v)
    kw = dict(k_norm_w=dev(w), eps=EPS) if norm else {}
    read = {}
    for elem in ("f32", "f16") + (("q8_0",) if hd % 32 == 0 else ()):
        c = rv.PagedKvCache(1, n_kv, hd, pool, page, elem)
        c.append_rows(0, qkv[:, 1:1 + kvd], qkv[:, 2 + kvd:2 + 2 * kvd], ints(table), ints(pos), ints(seq), rope=rope,
                      **kw)
        gk, gv = c.read_rows(0, ints(table), ints(pos), ints(seq))
        c.device_status()
        read[elem] = host(gk).astype(np.float32)
        assert np.array_equal(host(gv).astype(np.float32), stored(v, elem))
    x = k.reshape(n, n_kv, hd).astype(np.float64)
    slack = 0.0
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPS))) * w
        slack = 4 * EPS32  # the reciprocal root, its two products: half a step each, and one spare
    c, s = turns(rope, pos)
    want = rotated(x, c, s, r, layout)
    gain = rope.frequencies()[1]
    turned = np.zeros_like(x)
    turned[..., :r] = rotation_bound(x, r, layout, gain)[..., :r] * (1 + slack / EPS32 / 4)
    bound = turned + slack * np.abs(x)
    got = read["f32"].reshape(n, n_kv, hd)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))
    # The other types hold the roundings of those very rows.
    for elem in read:
        assert np.array_equal(read[elem], stored(read["f32"], elem)), elem


def test_rows_are_those_of_the_linear_cache():
    """Whole heads in NeoX order without scaling: the row that KvCache's step stores."""
    say("case linear cache rows")
    rng = np.random.default_rng(5)
    n, k, v = 6, rows(rng, 6, 512), rows(rng, 6, 512)
    w = (1 + 0.1 * rng.standard_normal(128)).astype(np.float32)
    q = rows(rng, n, 4096)
    kv, out = rv.KvCache(1, 4, 128, 8, "f32"), dev(np.zeros((n, 4096)))
    rv.prefill_chunk(kv, 0, dev(q), dev(k), dev(v), dev(w), dev(w), EPS, THETA, 0, scale_of(128), out)
    c = rv.PagedKvCache(1, 4, 128, 2, 8, "f32")
    c.append_rows(0, dev(k), dev(v), ints([[1, 0]]), ints(np.arange(n)), ints(np.zeros(n)), rope=rv.Rope(128, THETA),
                  k_norm_w=dev(w), eps=EPS)
    gk, gv = c.read_rows(0, ints([[1, 0]]), ints(np.arange(n)), ints(np.zeros(n)))
    wk, wv = kv.read_rows(0, 0, n)
    # The mean of squares is summed in another order in f64: at most a step of f32.
    assert np.all(np.abs(host(gk) - host(wk)) <= 2.0 ** -22 * np.abs(host(wk)).max())
    assert np.array_equal(host(gv), host(wv))


# ---- attention ----------------------------------------------------------------------------

def filled(rng, elem, n_kv, hd, page, lens, junk=True, extra=0):
    """A cache whose pages hold NaN rows wherever no sequence has a row, the
    sequences' rows, their table, and their values."""
    kvd = n_kv * hd
    per = max(1, -(-(max(lens) + extra) // page))
    table, pool = tables(rng, len(lens), per)
    c = rv.PagedKvCache(2, n_kv, hd, pool, page, elem)
    if junk:
        n = pool * page
        bad = np.full((n, kvd), np.nan, np.float32)
        bad[::3] = np.inf
        c.append_rows(1, dev(bad), dev(bad), ints(np.arange(pool)[None]), ints(np.arange(n)), ints(np.zeros(n)))
    own = []
    for i, m in enumerate(lens):
        k, v = rows(rng, m, kvd), rows(rng, m, kvd)
        if m:
            c.append_rows(1, dev(k), dev(v), ints(table), ints(np.arange(m)), ints(np.full(m, i)))
        own.append((stored(k, elem), stored(v, elem)))
    c.device_status()
    return c, table, own


def expect(q, own, n_kv, hd, scale=None):
    outs, a, vmax = [], 0.0, 1e-30
    for i, (k, v) in enumerate(own):
        if not len(k):
            outs.append(np.zeros(q.shape[1]))
            continue
        w, ai = attend(q[i], k, v, n_kv, hd, scale_of(hd) if scale is None else scale)
        outs.append(w)
        a, vmax = max(a, ai), max(vmax, float(np.abs(v).max()))
    return np.stack(outs), a, vmax


SHAPES = [
    (4, 8, 128, 64, [100]),
    (4, 8, 128, 16, [1]),
    (4, 8, 128, 64, [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000]),
    (4, 8, 128, 8, [5000, 3]),
    (2, 8, 128, 1024, [2500, 0, 1100]),
    (8, 1, 128, 32, [200, 77]),
    (4, 7, 128, 32, [300, 1, 40]),
    (1, 16, 128, 16, [700, 129]),
    (1, 17, 128, 16, [300]),
    (1, 40, 128, 64, [60, 10, 260]),
    (4, 4, 64, 16, [0, 150, 1501]),
    (2, 2, 96, 32, [130, 64, 1]),
    (2, 3, 256, 32, [140, 500]),
    (1, 2, 80, 8, [90, 300]),
    (1, 4, 192, 16, [33, 200]),
    (1, 2, 512, 16, [33, 200]),
    (2, 5, 20, 8, [60, 7]),
    (1, 3, 7, 16, [20]),
    (3, 1, 8, 8, [150]),
    (1, 1, 32, 8, [1, 9]),
]


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,group,hd,page,lens", SHAPES)
def test_paged_attention(elem, n_kv, group, hd, page, lens):
    torch = torch_cuda()
    if elem == "q8_0" and hd % 32:
        pytest.skip("Q8_0 rows are blocks of 32")
    say(f"case paged attention {(elem, n_kv, group, hd, page, lens)}")
    rng = np.random.default_rng(sum(lens) + hd)
    c, table, own = filled(rng, elem, n_kv, hd, page, lens)
    q = rng.standard_normal((len(lens), n_kv * group * hd)).astype(np.float32)
    out = torch.full((len(lens) + 2, q.shape[1]), 9.0, device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale_of(hd), out[:len(lens)])
    c.device_status()
    want, a, vmax = expect(q, own, n_kv, hd)
    got = host(out)
    assert np.all(got[len(lens):] == 9)
    for i in range(len(lens)):
        check(got[i], want[i], a, vmax, f"sequence {i}")
        if lens[i] == 0:
            assert not got[i].any()
    again = torch.empty_like(out[:len(lens)])
    rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale_of(hd), again)
    assert np.array_equal(host(again).view(np.uint32), got[:len(lens)].copy().view(np.uint32))


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_many_ragged_sequences(elem):
    torch = torch_cuda()
    say(f"case many sequences {elem}")
    rng = np.random.default_rng(11)
    lens = [int(x) for x in rng.integers(0, 400, 300)]
    lens[7], lens[299] = 9000, 0
    n_kv, group, hd = 2, 4, 64
    c, table, own = filled(rng, elem, n_kv, hd, 32, lens, junk=False)
    q = rng.standard_normal((300, n_kv * group * hd)).astype(np.float32)
    out = torch.empty(300, q.shape[1], device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale_of(hd), out)
    want, a, vmax = expect(q, own, n_kv, hd)
    for i in range(300):
        check(host(out)[i], want[i], a, vmax, f"sequence {i}")


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,group,hd,page,lens", [
    (4, 8, 128, 64, [9000, 1, 300]), (1, 4, 128, 64, [40000]), (2, 17, 64, 16, [5000, 70]), (1, 2, 192, 16, [6000]),
    (1, 2, 512, 16, [700, 90])])
def test_joins_across_xcds_alone(elem, n_kv, group, hd, page, lens):
    """The joins of a device that does not deal workgroups to its XCDs in turn."""
    torch = torch_cuda()
    say(f"case joins {(elem, n_kv, group, hd, lens)}")
    rng = np.random.default_rng(hd + lens[0])
    c, table, own = filled(rng, elem, n_kv, hd, page, lens)
    q = rng.standard_normal((len(lens), n_kv * group * hd)).astype(np.float32)
    want, a, vmax = expect(q, own, n_kv, hd)
    got = []
    for join in (2, 0, 2):
        c.set_tuning(rv.RV_TUNE_PAGED_JOIN, join)
        out = torch.full(q.shape, 9.0, device="cuda")
        rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale_of(hd), out)
        got.append(host(out))
        for i in range(len(lens)):
            check(got[-1][i], want[i], a, vmax, f"join {join} sequence {i}")
    assert np.array_equal(got[0].view(np.uint32), got[2].view(np.uint32))
    with pytest.raises(rv.RamvampError):
        c.set_tuning(2, 0)


@pytest.mark.parametrize("hd", [64, 20])
def test_mostly_empty_batches(hd):
    """Few sequences with rows between many without, refused ones among those."""
    torch = torch_cuda()
    say(f"case mostly empty {hd}")
    rng = np.random.default_rng(13)
    n, n_kv, group = 1500, 2, 4
    for live in ([0], [1499], [63, 64], [5, 128, 700, 1100, 1498], []):
        lens = np.zeros(n, int)
        lens[live] = rng.integers(1, 700, len(live))
        refused = [i for i in (2, 66, 900, 1497) if i not in live]
        c, table, own = filled(rng, "f16", n_kv, hd, 16, lens[live] if live else [1], junk=False)
        wide = np.full((n, table.shape[1]), -7)
        wide[live] = table[:len(live)]
        asked = lens.copy()
        asked[refused] = -3
        q = rng.standard_normal((n, n_kv * group * hd)).astype(np.float32)
        out = torch.full(q.shape, 9.0, device="cuda")
        rv.paged_attention(dev(q), c, 1, ints(wide), ints(asked), scale_of(hd), out)
        with pytest.raises(rv.KvError) as e:
            c.device_status()
        assert e.value.variant == "PositionOutOfTable"
        got = host(out)
        assert np.isnan(got[refused]).all()
        if live:
            want, a, vmax = expect(q[live], own, n_kv, hd)
            for j, i in enumerate(live):
                check(got[i], want[j], a, vmax, f"sequence {i}")
        rest = np.ones(n, bool)
        rest[live] = rest[refused] = False
        assert not got[rest].any()


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("hd", [128, 20])
def test_long_split_keeps_small_weights(elem, hd):
    """A first row far above the rest, whose weights are small and many: each counts."""
    torch = torch_cuda()
    if elem == "q8_0" and hd % 32:
        pytest.skip("Q8_0 rows are blocks of 32")
    say(f"case small weights {(elem, hd)}")
    n = 40000
    k = np.zeros((n, hd), np.float32)
    v = np.ones((n, hd), np.float32)
    k[0, 0], v[0] = 1.0, 0.0
    c = rv.PagedKvCache(1, 1, hd, n // 64, 64, elem)
    table = ints(np.random.default_rng(0).permutation(n // 64)[None])
    c.append_rows(0, dev(k), dev(v), table, ints(np.arange(n)), ints(np.zeros(n)))
    q = np.zeros((1, 4 * hd), np.float32)
    gaps = np.array([4.0, 12.0, 16.0, 20.0])  # the first row's score above the others'
    q[0, ::hd] = gaps / scale_of(hd)
    out = torch.empty(1, 4 * hd, device="cuda")
    rv.paged_attention(dev(q), c, 0, table, ints([n]), scale_of(hd), out)
    first = stored(k[:1], elem)[0, 0] * np.float32(gaps / scale_of(hd)).astype(np.float64) * scale_of(hd)
    rest = (n - 1) * np.exp(-first)
    one = stored(v[1:2], elem)[0, 0].astype(np.float64)
    want = one * rest / (1 + rest)
    got = host(out).reshape(4, hd)
    # The score's own error (its scaling, split and sum: 2^-21 of it) moves a weight by
    # as much times the score; the rest as in check().
    for j in range(4):
        bound = want[j] * (2 * gaps[j] * 2.0 ** -21 + 2.0 ** -21 + 96 * EPS32)
        assert np.all(np.abs(got[j] - want[j]) <= bound), (j, float(np.abs(got[j] - want[j]).max()), bound)


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("hd", [64, 128, 256, 192, 20])
def test_long_sums_keep_small_weights(elem, hd):
    """As above where a workgroup has whole sequences: 300 over one's pages. Of the two kv
    heads' values one has the first row apart, the other the rest."""
    torch = torch_cuda()
    if elem == "q8_0" and hd % 32:
        pytest.skip("Q8_0 rows are blocks of 32")
    say(f"case long sums {(elem, hd)}")
    n, seqs = 130000, 300
    c = rv.PagedKvCache(1, 2, hd, -(-n // 64), 64, elem)
    k, v = torch.zeros(n, 2 * hd, device="cuda"), torch.ones(n, 2 * hd, device="cuda")
    k[0, 0] = k[0, hd] = 1.0
    v[0, :hd] = 0.0
    v[1:, hd:] = 0.0
    table = ints(np.random.default_rng(0).permutation(-(-n // 64))[None])
    c.append_rows(0, k, v, table, ints(np.arange(n)), ints(np.zeros(n)))
    gaps = np.array([24.5, 27.5, 29.5, 31.5]) * np.log(2)  # the first row's score above the others'
    q = np.zeros((2, 4, hd), np.float32)
    q[:, :, 0] = gaps / scale_of(hd)
    q = np.tile(q.reshape(1, -1), (seqs, 1))
    out = torch.empty(seqs, 8 * hd, device="cuda")
    rv.paged_attention(dev(q), c, 0, table.repeat(seqs, 1), ints([n] * seqs), scale_of(hd), out)
    one = stored(np.ones((1, 32), np.float32), elem)[0, 0].astype(np.float64)
    first = one * np.float32(gaps / scale_of(hd)).astype(np.float64) * scale_of(hd)
    rest = (n - 1) * np.exp(-first)
    want = np.stack([one * rest / (1 + rest), one / (1 + rest)])
    # The weights as in the test above, and check()'s 96 half steps of the largest value.
    bound = rest / (1 + rest) * (2 * gaps + 1) * 2.0 ** -21 + 96 * EPS32
    err = np.abs(host(out).reshape(seqs, 2, 4, hd) - want[None, :, :, None]).max((0, 3))
    assert np.all(err <= bound), (err, bound)


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("mag", [1e-20, 1e-6, 1e6, 1e15])
def test_queries_of_any_magnitude(elem, mag):
    """q times mag, the scale divided by it: the same output."""
    torch = torch_cuda()
    say(f"case magnitude {(elem, mag)}")
    rng = np.random.default_rng(4)
    lens = [300, 20]
    c, table, own = filled(rng, elem, 2, 128, 16, lens)
    q = (rng.standard_normal((2, 2 * 4 * 128)) * mag).astype(np.float32)
    scale = float(np.float32(scale_of(128) / mag))
    out = torch.empty(2, q.shape[1], device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale, out)
    want, a, vmax = expect(q, own, 2, 128, scale)
    check(host(out), want, a, vmax, "all")


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales(scale):
    torch = torch_cuda()
    say(f"case scale {scale}")
    rng = np.random.default_rng(6)
    c, table, own = filled(rng, "f16", 2, 128, 16, [200])
    q = rng.standard_normal((1, 1024)).astype(np.float32)
    out = torch.empty(1, 1024, device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(table), ints([200]), scale, out)
    want, a, vmax = expect(q, own, 2, 128, scale)
    check(host(out), want, a, vmax, "all")


def test_zero_and_nonfinite_queries():
    torch = torch_cuda()
    say("case zero and non-finite queries")
    rng = np.random.default_rng(6)
    c, table, own = filled(rng, "f16", 1, 128, 16, [200])
    q = rng.standard_normal((1, 512)).astype(np.float32)
    q[0, :128] = 0
    q[0, 130] = np.nan
    q[0, 300] = np.inf
    out = torch.empty(1, 512, device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(table), ints([200]), scale_of(128), out)
    got = host(out).reshape(4, 128)
    mean = own[0][1].astype(np.float64).mean(0)
    assert np.all(np.abs(got[0] - mean) <= 2.0 ** -17 * np.abs(own[0][1]).max())
    assert np.isnan(got[1:3]).all()
    want, a, vmax = expect(q[:, 384:], own, 1, 128)
    check(got[3], want[0], a, vmax, "the head beside them")


def test_a_nonfinite_row_stays_in_its_head_and_sequence():
    torch = torch_cuda()
    say("case non-finite rows")
    rng = np.random.default_rng(8)
    for elem in ("f16", "f32", "q8_0"):
        c, table, own = filled(rng, elem, 2, 128, 16, [200, 90])
        bad = rows(rng, 1, 256)
        bad[0, 5] = np.nan  # kv head 0
        c.append_rows(1, dev(bad), dev(rows(rng, 1, 256)), ints(table), ints([77]), ints([0]))
        q = rng.standard_normal((2, 1024)).astype(np.float32)
        out = torch.empty(2, 1024, device="cuda")
        rv.paged_attention(dev(q), c, 1, ints(table), ints([200, 90]), scale_of(128), out)
        got = host(out)
        assert np.isnan(got[0, :512]).all() and np.isfinite(got[0, 512:]).all()
        want, a, vmax = expect(q[1:], own[1:], 2, 128)
        check(got[1], want[0], a, vmax, "the sequence beside it")


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("hd", [128, 64, 20, 512])
@pytest.mark.parametrize("n,at", [(1, 0), (200, 0), (200, 4), (200, 16), (200, 199), (6000, 3000)])
def test_a_nan_anywhere_reaches_the_output(elem, hd, n, at):
    """A row of NaN, the first that a wave sees or its last, in K or in V."""
    torch = torch_cuda()
    if elem == "q8_0" and hd % 32:
        pytest.skip("Q8_0 rows are blocks of 32")
    say(f"case NaN {(elem, hd, n, at)}")
    rng = np.random.default_rng(n + at)
    c, table, own = filled(rng, elem, 2, hd, 16, [n, 90])
    q = rng.standard_normal((2, 4 * hd)).astype(np.float32)
    row = np.full((1, 2 * hd), np.nan, np.float32)
    row[:, hd:] = 1.0  # kv head 1 stays sound
    for bad_k in (True, False):
        fine = np.ones((1, 2 * hd), np.float32)
        c.append_rows(1, dev(row if bad_k else fine), dev(fine if bad_k else row), ints(table), ints([at]), ints([0]))
        out = torch.empty(2, 4 * hd, device="cuda")
        rv.paged_attention(dev(q), c, 1, ints(table), ints([n, 90]), scale_of(hd), out)
        got = host(out)
        assert np.isnan(got[0, :2 * hd]).all() and np.isfinite(got[0, 2 * hd:]).all()
        want, a, vmax = expect(q[1:], own[1:], 2, hd)
        check(got[1], want[0], a, vmax, "the sequence beside it")


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("hd", [128, 32])
def test_refused_sequences(elem, hd):
    """Bad pages and lengths: NaN for their sequence, recorded, the others as without them."""
    torch = torch_cuda()
    say(f"case refused sequences {(elem, hd)}")
    rng = np.random.default_rng(9)
    lens = [100, 60, 300, 50, 40]
    c, table, own = filled(rng, elem, 2, hd, 16, lens)
    q = rng.standard_normal((5, 8 * hd)).astype(np.float32)
    bad = table.copy()
    bad[0, 2] = -1
    bad[2, 18] = 2 ** 31 - 1  # its last page
    bad[3, 4:] = -9           # entries past its rows are not looked at
    asked = [100, -1, 300, 50, table.shape[1] * 16 + 1]
    out = torch.full((5, 8 * hd), 3.0, device="cuda")
    rv.paged_attention(dev(q), c, 1, ints(bad), ints(asked), scale_of(hd), out)
    with pytest.raises(rv.KvError) as e:
        c.device_status()
    assert e.value.variant in ("PageOutOfRange", "PositionOutOfTable") and e.value.fields["layer"] == 1
    got = host(out)
    assert np.isnan(got[[0, 1, 2, 4]]).all()
    want, a, vmax = expect(q, own, 2, hd)
    check(got[3], want[3], a, vmax, "the sound one")
    rv.paged_attention(dev(q), c, 1, ints(table), ints(lens), scale_of(hd), out)
    c.device_status()
    for i in range(5):
        check(host(out)[i], want[i], a, vmax, f"sequence {i}")


def test_strided_views_and_shared_pages():
    torch = torch_cuda()
    say("case strides and shared pages")
    rng = np.random.default_rng(10)
    c, table, own = filled(rng, "f16", 2, 128, 16, [200, 90])
    wide = np.full((6, table.shape[1] + 3), -5)
    both = np.stack([table[0], table[0], table[1]])  # two sequences on one's pages
    wide[::2, 1:1 + table.shape[1]] = both
    t = ints(wide)[::2, 1:1 + table.shape[1]]
    q = rng.standard_normal((3, 1024)).astype(np.float32)
    buf = torch.full((3, 2 * 1024 + 7), 4.0, device="cuda")
    qv, ov = buf[:, 3:1027], buf[:, 1027:2051]
    qv.copy_(dev(q))
    rv.paged_attention(qv, c, 1, t, ints([200, 64, 90]), scale_of(128), ov)
    c.device_status()
    want, a, vmax = expect(q, [own[0], (own[0][0][:64], own[0][1][:64]), own[1]], 2, 128)
    check(host(ov), want, a, vmax, "all")
    w = host(buf)
    assert np.all(w[:, :3] == 4) and np.all(w[:, 2051:] == 4) and np.array_equal(w[:, 3:1027], q)


def test_pages_past_4_gib():
    torch = torch_cuda()
    say("case pages past 4 GiB")
    rng = np.random.default_rng(12)
    n_kv, hd, page = 8, 128, 1024
    for elem, pool in (("f16", 2300), ("q8_0", 4300), ("f32", 1200)):
        c = rv.PagedKvCache(1, n_kv, hd, pool, page, elem)
        table = np.array([[pool - 1, 0], [pool - 2, 1]])
        k, v = rows(rng, 2 * 1100, 1024), rows(rng, 2 * 1100, 1024)
        pos, seq = np.tile(np.arange(1100), 2), np.repeat([0, 1], 1100)
        c.append_rows(0, dev(k), dev(v), ints(table), ints(pos), ints(seq))
        gk, gv = c.read_rows(0, ints(table), ints(pos), ints(seq))
        assert np.array_equal(host(gk).astype(np.float32), stored(k, elem))
        assert np.array_equal(host(gv).astype(np.float32), stored(v, elem))
        q = rng.standard_normal((2, 4 * 1024)).astype(np.float32)
        out = torch.empty(2, 4096, device="cuda")
        rv.paged_attention(dev(q), c, 0, ints(table), ints([1100, 1099]), scale_of(hd), out)
        own = [(stored(k[:1100], elem), stored(v[:1100], elem)),
               (stored(k[1100:2199], elem), stored(v[1100:2199], elem))]
        want, a, vmax = expect(q, own, n_kv, hd)
        check(host(out), want, a, vmax, elem)
        c.close()


# ---- the batch's step, and all of it together ---------------------------------------------

def step_inputs(rng, n, n_kv, group, hd):
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    return rows(rng, n, n_kv * group * hd), rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd), w


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,group,hd,r,layout,lens", [
    (4, 8, 128, 128, "half", [0, 1, 63, 64, 300]), (2, 3, 64, 32, "interleaved", [5, -1, 0]),
    (1, 16, 96, 96, "half", [40]), (2, 1, 256, 64, "half", [7, 130]), (1, 2, 512, 512, "half", [9]),
])
def test_step_is_its_parts(elem, n_kv, group, hd, r, layout, lens):
    torch = torch_cuda()
    say(f"case step {(elem, n_kv, group, hd, r, layout, lens)}")
    rng = np.random.default_rng(hd + len(lens))
    rope = rv.Rope(hd, THETA, r, layout)
    n = len(lens)
    two = [filled(np.random.default_rng(1), elem, n_kv, hd, 16, [max(x, 0) for x in lens], extra=1) for _ in range(2)]
    (c, table, _), (d, _, _) = two
    q, k, v, (wq, wk) = step_inputs(rng, n, n_kv, group, hd)
    out = torch.full(q.shape, 3.0, device="cuda")
    rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), dev(wq), dev(wk), EPS, rope, ints(table), ints(lens),
                         scale_of(hd), out)
    c.device_status()
    d.append_rows(1, dev(k), dev(v), ints(table), ints(lens), rope=rope, k_norm_w=dev(wk), eps=EPS)
    for a, b in zip(everything(c, 1), everything(d, 1)):
        assert np.array_equal(a, b, equal_nan=True)
    # q as the step's: the same norm and rotation through a cache of q's heads.
    qc = rv.PagedKvCache(1, n_kv * group, hd, n, 8, "f32")
    at = np.array(lens)
    tab = np.tile(np.arange(n)[:, None], (1, max(1, (max(lens) + 8) // 8)))
    qc.append_rows(0, dev(q), dev(q), ints(tab), ints(at), rope=rope, k_norm_w=dev(wq), eps=EPS)
    qr, _ = qc.read_rows(0, ints(tab), ints(at))
    want = torch.empty_like(out)
    rv.paged_attention(qr, d, 1, ints(table), ints(at + 1), scale_of(hd), want)
    d.device_status()
    assert np.array_equal(host(out).view(np.uint32), host(want).view(np.uint32))
    for i in range(n):
        if lens[i] < 0:
            assert not host(out)[i].any()


def test_step_without_norm_or_rotation():
    torch = torch_cuda()
    say("case bare step")
    rng = np.random.default_rng(2)
    c, table, own = filled(rng, "f32", 2, 64, 16, [30, 0], extra=1)
    q, k, v, _ = step_inputs(rng, 2, 2, 4, 64)
    out = torch.empty(q.shape, device="cuda")
    rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), None, None, EPS, None, ints(table), ints([30, 0]),
                         scale_of(64), out)
    own = [(np.concatenate([o[0], k[i:i + 1]]), np.concatenate([o[1], v[i:i + 1]])) for i, o in enumerate(own)]
    want, a, vmax = expect(q, own, 2, 64)
    check(host(out), want, a, vmax, "all")


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_prompts_moved_to_pages_then_decoded_as_by_linear_caches(elem):
    """A serving loop: each prompt through KvCache's chunk, its rows moved to pages,
    then tokens of the whole batch; a linear cache a sequence does the same."""
    torch = torch_cuda()
    say(f"case serving loop {elem}")
    rng = np.random.default_rng(21)
    prompts, layers, tokens, n_kv, hd = [70, 9, 130], 2, 4, 4, 128
    n, kvd, qd = len(prompts), n_kv * hd, 32 * 128
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    table, pool = tables(rng, n, 9)
    pages = rv.PagedKvCache(layers, n_kv, hd, pool, 16, elem)
    lin = [rv.KvCache(layers, n_kv, hd, m + tokens, elem) for m in prompts]
    for i, m in enumerate(prompts):
        for layer in range(layers):
            out = dev(np.zeros((m, qd)))
            rv.prefill_chunk(lin[i], layer, dev(rows(rng, m, qd)), dev(rows(rng, m, kvd)), dev(rows(rng, m, kvd)),
                             dev(w[0]), dev(w[1]), EPS, THETA, 0, scale_of(hd), out)
            k, v = lin[i].read_rows(layer, 0, m)
            pages.append_rows(layer, k, v, ints(table), ints(np.arange(m)), ints(np.full(m, i)))
    rope, at = rv.Rope(hd, THETA), ints(prompts)
    for t in range(tokens):
        for layer in range(layers):
            q, k, v = rows(rng, n, qd), rows(rng, n, kvd), rows(rng, n, kvd)
            out, want = torch.empty(n, qd, device="cuda"), torch.empty(n, qd, device="cuda")
            rv.paged_decode_step(pages, layer, dev(q), dev(k), dev(v), dev(w[0]), dev(w[1]), EPS, rope, ints(table),
                                 at, scale_of(hd), out)
            for i, m in enumerate(prompts):
                rv.decode_step(lin[i], layer, dev(q[i]), dev(k[i]), dev(v[i]), dev(w[0]), dev(w[1]), EPS, THETA, m + t,
                               scale_of(hd), want[i])
            g, x = host(out).astype(np.float64), host(want).astype(np.float64)
            # Both within their own bounds of one value; two of a step of f16 (or of a
            # code) may fall apart where a row's last bit does, far less than this.
            assert np.linalg.norm(g - x) <= 2.0 ** -10 * np.linalg.norm(x)
        at.add_(1)
    pages.device_status()


@pytest.mark.parametrize("elem", ["f16", "q8_0"])
def test_captured_step_follows_positions_and_tables(elem):
    torch = torch_cuda()
    say(f"case captured step {elem}")
    rng = np.random.default_rng(31)
    lens = [30, 200, 15]
    (c, table, _), (d, _, _) = [filled(np.random.default_rng(1), elem, 4, 128, 16, lens, extra=8) for _ in range(2)]
    q, k, v, (wq, wk) = (x if isinstance(x, list) else dev(x) for x in step_inputs(rng, 3, 4, 8, 128))
    wq, wk, rope = dev(wq), dev(wk), rv.Rope(128, THETA)
    out, ref = torch.empty(3, 4096, device="cuda"), torch.empty(3, 4096, device="cuda")
    t = ints(table)
    at, at2 = ints(lens), ints(lens)

    def step(cache, where, into):
        rv.paged_decode_step(cache, 1, q, k, v, wq, wk, EPS, rope, t, where, scale_of(128), into)

    step(d, at2, ref)  # (allocates)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, at, out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(c, at, out)
        at.add_(1)
    at.copy_(ints(lens))
    for i in range(6):
        if i == 3:  # the last sequence leaves: padding from here on
            at[2] = -9
            at2[2] = -9
        for x in (q, k, v):
            x.mul_(1.01)
        out.fill_(float("nan"))
        g.replay()
        step(d, at2, ref)
        at2.add_(1)
        torch.cuda.synchronize()
        assert np.array_equal(host(out).view(np.uint32), host(ref).view(np.uint32)), f"replay {i}"
    for a, b in zip(everything(c, 1), everything(d, 1)):
        assert np.array_equal(a, b, equal_nan=True)


def test_graphs_over_one_cache_in_turn_while_its_workspace_grows():
    """Two captured batches, replayed alternately; then larger eager calls, which take
    new workspaces, and the graphs again."""
    torch = torch_cuda()
    say("case two graphs")
    rng = np.random.default_rng(51)
    lens = [9000, 700, 40, 3, 0]
    c, table, own = filled(rng, "f16", 2, 128, 16, lens)
    q = rng.standard_normal((5, 2 * 4 * 128)).astype(np.float32)
    t, n, qd = ints(table), ints(lens), dev(q)
    outs, graphs = [torch.empty(5, 1024, device="cuda") for _ in range(2)], []
    want, a, vmax = expect(q, own, 2, 128)
    torch.cuda.synchronize()
    call = lambda o, k: rv.paged_attention(qd[:k], c, 1, t[:k], n[:k], scale_of(128), o[:k])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(outs[0], 5)
    torch.cuda.current_stream().wait_stream(side)
    for o, k in zip(outs, (5, 1)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(o, k)
        graphs.append(g)
    for rep in range(4):
        for o in outs:
            o.fill_(float("nan"))
        for g in graphs:
            g.replay()
        if rep:
            # Sixteen heads a kv head, then a batch ten times as large.
            big = dev(rng.standard_normal((5, 2 * 16 * 128)))
            rv.paged_attention(big, c, 1, t, n, scale_of(128), torch.empty_like(big))
            many = ints(np.tile(table, (10 * rep, 1)))
            wide = qd.repeat(10 * rep, 1)
            o2 = rv.paged_attention(wide, c, 1, many, n.repeat(10 * rep), scale_of(128), torch.empty_like(wide))
            for i in range(50 * rep):
                check(host(o2)[i], want[i % 5], a, vmax, f"batch {i}")
        for i in range(5):
            check(host(outs[0])[i], want[i], a, vmax, f"replay {rep} sequence {i}")
        check(host(outs[1])[0], want[0], a, vmax, f"replay {rep} of one")
        assert torch.isnan(outs[1][1:]).all()


def test_rows_of_one_call_that_name_one_place():
    """Of two rows for one place it holds values of both; no other place changes."""
    say("case one place twice")
    rng = np.random.default_rng(52)
    c = rv.PagedKvCache(1, 2, 64, 2, 8, "f16")
    k, v = rows(rng, 6, 128), rows(rng, 6, 128)
    at = [3, 3, 3, 4, 3, 3]
    c.append_rows(0, dev(k), dev(v), ints([[1]]), ints(at), ints([0] * 6))
    (gk, gv) = (host(x) for x in c.read_rows(0, ints([[1]]), ints(range(8)), ints([0] * 8)))
    for got, x in ((gk, k), (gv, v)):
        x = x.astype(np.float16)
        assert np.array_equal(got[4], x[3]) and not got[[0, 1, 2, 5, 6, 7]].any()
        assert np.all(np.any(got[3] == x[[0, 1, 2, 4, 5]], axis=0))
    kp, _ = c.read_rows(0, ints([[0]]), ints(range(8)), ints([0] * 8))
    assert not host(kp).any()


def test_step_of_a_large_padded_batch():
    """More sequences than a wave has lanes, a third of them padding, into strided out."""
    torch = torch_cuda()
    say("case large step")
    rng = np.random.default_rng(53)
    n, n_kv, group, hd = 150, 2, 4, 64
    lens = rng.integers(0, 200, n)
    off = rng.random(n) < 0.3
    c, table, own = filled(rng, "q8_0", n_kv, hd, 16, lens, extra=1)
    q, k, v, _ = step_inputs(rng, n, n_kv, group, hd)
    wide = torch.full((n, q.shape[1] + 8), 9.0, device="cuda")
    out = wide[:, 4:4 + q.shape[1]]
    rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), None, None, EPS, None, ints(table), ints(np.where(off, -1, lens)),
                         scale_of(hd), out)
    c.device_status()
    new = [(np.concatenate([o[0], stored(k[i:i + 1], "q8_0")]), np.concatenate([o[1], stored(v[i:i + 1], "q8_0")]))
           for i, o in enumerate(own)]
    want, a, vmax = expect(q, new, n_kv, hd)
    got = host(out)
    for i in range(n):
        if off[i]:
            assert not got[i].any()
        else:
            check(got[i], want[i], a, vmax, f"sequence {i}")
    w = host(wide)
    assert np.all(w[:, :4] == 9) and np.all(w[:, -4:] == 9)


def test_a_captured_call_that_would_allocate_is_refused():
    torch = torch_cuda()
    say("case capture refused")
    c = rv.PagedKvCache(1, 2, 64, 4, 16, "f16")
    q, out = dev(np.zeros((1, 512))), dev(np.zeros((1, 512)))
    t, n = ints([[0]]), ints([0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q.add_(1)
        with pytest.raises(rv.DeviceError) as e:
            rv.paged_attention(q, c, 0, t, n, 1.0, out)
        assert e.value.variant == "Unsupported"
        with pytest.raises(rv.DeviceError):
            c.device_status()
    rv.paged_attention(q, c, 0, t, n, 1.0, out)
    c.device_status()


def test_streams_take_turns_and_caches_do_not_meet():
    """One cache from several streams in turn; two caches from two threads at once."""
    torch = torch_cuda()
    say("case streams and threads")
    rng = np.random.default_rng(41)
    lens = [500, 40]
    c, table, own = filled(rng, "f16", 4, 128, 64, lens)
    q = rng.standard_normal((2, 4096)).astype(np.float32)
    want, a, vmax = expect(q, own, 4, 128)
    t, n, qd = ints(table), ints(lens), dev(q)
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs.append(rv.paged_attention(qd, c, 1, t, n, scale_of(128), torch.empty(2, 4096, device="cuda")))
    torch.cuda.synchronize()
    for o in outs:
        check(host(o), want, a, vmax, "streams")
    two = [filled(np.random.default_rng(i), "f16", 4, 128, 64, lens) for i in range(2)]
    res, errs = [None, None], []

    def work(i):
        try:
            cache, tab, _ = two[i]
            s = torch.cuda.Stream()
            tt, nn = ints(tab), ints(lens)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                for _ in range(20):
                    res[i] = rv.paged_attention(qd, cache, 1, tt, nn, scale_of(128),
                                                torch.empty(2, 4096, device="cuda"))
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errs.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [x.start() for x in ts]
    [x.join() for x in ts]
    assert not errs
    for i in range(2):
        want, a, vmax = expect(q, two[i][2], 4, 128)
        check(host(res[i]), want, a, vmax, f"thread {i}")


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_step_of_a_fused_matrix(elem):
    """q, k and v as columns of one matrix, out over q: the bits of rows apart."""
    torch = torch_cuda()
    say(f"case fused matrix {elem}")
    rng = np.random.default_rng(54)
    lens, n_kv, group, hd = [70, 0, 300], 2, 4, 96
    two = [filled(np.random.default_rng(1), elem, n_kv, hd, 16, lens, extra=1) for _ in range(2)]
    (c, table, _), (d, _, _) = two
    q, k, v, (wq, wk) = step_inputs(rng, 3, n_kv, group, hd)
    rope = rv.Rope(hd, THETA, 48, "interleaved")
    args = (dev(wq), dev(wk), EPS, rope, ints(table), ints(lens), scale_of(hd))
    want = rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), *args, torch.empty(q.shape, device="cuda"))
    a, b = q.shape[1], k.shape[1]
    fused = torch.full((3, a + 2 * b + 3), 9.0, device="cuda")
    parts = [fused[:, 1:1 + a], fused[:, 1 + a:1 + a + b], fused[:, 1 + a + b:1 + a + 2 * b]]
    for x, y in zip(parts, (q, k, v)):
        x.copy_(dev(y))
    rv.paged_decode_step(d, 1, *parts, *args, parts[0])
    assert np.array_equal(host(parts[0]).copy().view(np.uint32), host(want).view(np.uint32))
    w = host(fused)
    assert np.all(w[:, 0] == 9) and np.all(w[:, -2:] == 9)
    assert np.array_equal(w[:, 1 + a:1 + a + b], k) and np.array_equal(w[:, 1 + a + b:-2], v)
    for x, y in zip(everything(c, 1), everything(d, 1)):
        assert np.array_equal(x, y, equal_nan=True)


def test_threads_take_turns_at_one_cache():
    """Two threads on streams of their own, one cache and one workspace; each appends to
    its own sequence and attends both."""
    torch = torch_cuda()
    say("case threads at one cache")
    rng = np.random.default_rng(42)
    lens = [5000, 3000]
    c, table, own = filled(rng, "f16", 4, 128, 64, lens)
    q = [rng.standard_normal((2, 4096)).astype(np.float32) for _ in range(2)]
    want = [expect(x, own, 4, 128) for x in q]
    t, n, qd = ints(table), ints(lens), [dev(x) for x in q]
    new = [(dev(own[i][0][-1:]), dev(own[i][1][-1:])) for i in range(2)]  # the last rows again
    last, seq = [ints([m - 1]) for m in lens], [ints([i]) for i in range(2)]
    torch.cuda.synchronize()
    outs, errs = [[], []], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    c.append_rows(1, *new[i], t, last[i], seq[i])
                    outs[i].append(rv.paged_attention(qd[i], c, 1, t, n, scale_of(128),
                                                      torch.empty(2, 4096, device="cuda")))
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errs.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [x.start() for x in ts]
    [x.join() for x in ts]
    assert not errs
    c.device_status()
    for i in range(2):
        for o in outs[i]:
            assert np.array_equal(host(o).view(np.uint32), host(outs[i][0]).view(np.uint32))
        check(host(outs[i][0]), *want[i], f"thread {i}")


def test_empty_calls():
    torch = torch_cuda()
    say("case empty calls")
    c = rv.PagedKvCache(1, 2, 64, 4, 16, "f16")
    none, t0 = ints([]), torch.empty(0, 0, dtype=torch.int32, device="cuda")
    e = lambda w, dt=torch.float32: torch.empty(0, w, dtype=dt, device="cuda")
    c.append_rows(0, e(128), e(128), t0, none)
    k, v = c.read_rows(0, t0, none)
    assert k.shape == v.shape == (0, 128)
    rv.paged_attention(e(256), c, 0, t0, none, 1.0, e(256))
    rv.paged_decode_step(c, 0, e(256), e(128), e(128), None, None, EPS, None, t0, none, 1.0, e(256))
    # A table of sequences without pages: every length but 0 is refused.
    out = torch.full((2, 256), 3.0, device="cuda")
    rv.paged_attention(torch.zeros(2, 256, device="cuda"), c, 0, torch.empty(2, 0, dtype=torch.int32, device="cuda"),
                       ints([0, 1]), 1.0, out)
    got = host(out)
    assert not got[0].any() and np.isnan(got[1]).all()
    with pytest.raises(rv.KvError):
        c.device_status()


def test_host_refusals():
    torch = torch_cuda()
    say("case host refusals")
    c = rv.PagedKvCache(2, 2, 64, 4, 16, "f16")
    f = lambda *s: torch.zeros(*s, device="cuda")
    t, one = ints([[0], [1]]), ints([0, 0])
    out = torch.full((2, 256), 3.0, device="cuda")
    for call, variant in [
            (lambda: rv.paged_attention(f(2, 200), c, 0, t, one, 1.0, f(2, 200)), "QLenIndivisible"),
            (lambda: rv.paged_attention(f(2, 192), c, 0, t, one, 1.0, f(2, 192)), "GqaGroupMismatch"),
            (lambda: rv.paged_attention(f(2, 256), c, 2, t, one, 1.0, out), "LayerOutOfRange"),
            (lambda: rv.paged_attention(f(3, 256), c, 0, t, ints([0] * 3), 1.0, f(3, 256)), "LengthMismatch"),
            (lambda: rv.paged_attention(out, c, 0, t, one, 1.0, out), "Unsupported"),
            (lambda: c.append_rows(2, f(2, 128), f(2, 128), t, one), "LayerOutOfRange"),
            (lambda: c.append_rows(0, f(3, 128), f(3, 128), t, ints([0] * 3)), "LengthMismatch"),
            (lambda: c.append_rows(0, f(2, 128), f(2, 128), t, one, rope=rv.Rope(128, THETA)), "LengthMismatch"),
            (lambda: c.append_rows(0, f(2, 128), f(2, 128), t, one, k_norm_w=f(63)), "LengthMismatch"),
            (lambda: c.read_rows(2, t, one), "LayerOutOfRange"),
            (lambda: c.read_rows(0, t, ints([0] * 3)), "LengthMismatch"),
            (lambda: rv.paged_decode_step(c, 0, f(2, 256), f(2, 128), f(2, 128), f(65), None, EPS, None, t, one, 1.0,
                                          out), "LengthMismatch"),
            (lambda: rv.paged_decode_step(c, 0, f(2, 256), f(2, 128), f(2, 128), None, None, EPS, rv.Rope(32, THETA),
                                          t, one, 1.0, out), "LengthMismatch"),
            (lambda: rv.paged_decode_step(c, 2, f(2, 256), f(2, 128), f(2, 128), None, None, EPS, None, t, one, 1.0,
                                          out), "LayerOutOfRange")]:
        with pytest.raises(rv.RamvampError) as e:
            call()
        assert e.value.variant == variant
    with pytest.raises(rv.DeviceError):
        rv.PagedKvCache(1, 2, 64, 4, 16, "f16", device=torch.cuda.device_count())
    with pytest.raises(rv.DeviceError):
        rv.PagedKvCache(1, 64, 128, 2 ** 20, 1024, "f32")  # 64 TiB
    # 2^21 pages of 1024 rows for each of 128 kv heads: 2^31 units.
    many = rv.PagedKvCache(1, 128, 8, 1, 1024, "f16")
    with pytest.raises(rv.RamvampError) as e:
        rv.paged_attention(f(1, 1024), many, 0, torch.zeros(1, 2 ** 21, dtype=torch.int32, device="cuda"), ints([1]), 1.0,
                           f(1, 1024))
    assert e.value.variant == "Unsupported"
    for call in [
            lambda: rv.paged_attention(f(2, 256).double(), c, 0, t, one, 1.0, out),
            lambda: rv.paged_attention(f(256, 2).T, c, 0, t, one, 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, t.long(), one, 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, t, one.long(), 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, ints([0, 1]), one, 1.0, out),
            lambda: rv.paged_attention(f(2, 256).cpu(), c, 0, t, one, 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, t.cpu(), one, 1.0, out),
            lambda: rv.paged_attention(f(512), c, 0, t, one, 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, t, ints([0]), 1.0, out),
            lambda: rv.paged_attention(f(2, 256), c, 0, t, one, 1.0, f(1, 256)),
            lambda: c.append_rows(0, f(2, 128), f(1, 128), t, one),
            lambda: c.append_rows(0, f(2, 64), f(2, 64), t, one),
            lambda: c.append_rows(0, f(2, 128), f(2, 128), t, one, ints([0])),
            lambda: c.append_rows(0, f(2, 128), f(2, 128), t, one, k_norm_w=f(64).double()),
            lambda: c.read_rows(0, t, one, k=f(2, 128)),
            lambda: c.read_rows(0, t, one, v=f(1, 128).half()),
            lambda: rv.paged_decode_step(c, 0, f(2, 256), f(1, 128), f(2, 128), None, None, EPS, None, t, one, 1.0,
                                         out),
            lambda: rv.rope_rows(f(2, 128), one, rv.Rope(64, THETA), f(2, 64))]:
        with pytest.raises((TypeError, ValueError)):
            call()
    assert np.all(host(out) == 3)
    for k, v in (everything(c, 0), everything(c, 1)):
        assert not k.any() and not v.any()


@pytest.mark.parametrize("back", [False, True])
def test_calls_behind_a_capture_wait_for_those_before_it(back):
    """A call on one stream, held up there, another captured on a second without a wait
    for the device, then one on a third, or on the second itself."""
    torch = torch_cuda()
    say(f"case behind a capture {back}")
    rng = np.random.default_rng(55)
    lens, n_kv, hd = [300, 40], 2, 128
    c, table, _ = filled(rng, "f16", n_kv, hd, 16, lens)
    k, v = rows(rng, 2, n_kv * hd), rows(rng, 2, n_kv * hd)
    t, n, last, seq = ints(table), ints(lens), ints([m - 1 for m in lens]), ints([0, 1])
    kd, vd, q = dev(k), dev(v), dev(rng.standard_normal((2, 2 * 4 * hd)))
    out = torch.empty(2, 2 * 4 * hd, device="cuda")
    gk, gv = (torch.zeros(2, n_kv * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    big = torch.ones(8192, 8192, device="cuda")
    first, second, third = (torch.cuda.Stream() for _ in range(3))
    with torch.cuda.stream(second):
        rv.paged_attention(q, c, 1, t, n, scale_of(hd), out)  # (allocates)
    with torch.cuda.stream(first):
        hold = big @ big
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        for _ in range(8):
            torch.mm(big, big, out=hold)
        c.append_rows(1, kd, vd, t, last, seq)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(second):
        g.capture_begin()
        rv.paged_attention(q, c, 1, t, n, scale_of(hd), out)
        g.capture_end()
    with torch.cuda.stream(second if back else third):
        c.read_rows(1, t, last, seq, k=gk, v=gv)
    torch.cuda.synchronize()
    assert np.array_equal(host(gk), k.astype(np.float16)) and np.array_equal(host(gv), v.astype(np.float16))
    out.fill_(float("nan"))
    g.replay()
    torch.cuda.synchronize()
    again = rv.paged_attention(q, c, 1, t, n, scale_of(hd), torch.empty_like(out))
    assert np.array_equal(host(out).view(np.uint32), host(again).view(np.uint32))


@pytest.mark.parametrize("hd", [128, 64, 96, 256, 192, 20, 512])
@pytest.mark.parametrize("lens", [[300, 1, 16], [9000], [70] * 300])
def test_values_at_the_end_of_the_range(hd, lens):
    """f32 pages whose values' sums pass the floats' range: averages of them do not."""
    torch = torch_cuda()
    say(f"case largest values {(hd, lens[:3])}")
    rng = np.random.default_rng(hd + len(lens))
    n_kv, group, page = 2, 4, 16
    top = float(np.finfo(np.float32).max)
    table, pool = tables(rng, len(lens), -(-max(lens) // page))
    c = rv.PagedKvCache(1, n_kv, hd, pool, page, "f32")
    own = []
    for i, n in enumerate(lens):
        k, v = rows(rng, n, n_kv * hd), rng.uniform(-1, 1, (n, n_kv * hd))
        v[:, :hd // 2] = 1.0  # half of kv head 0: all as large as can be
        v = (v * top).astype(np.float32)
        c.append_rows(0, dev(k), dev(v), ints(table), ints(np.arange(n)), ints(np.full(n, i)))
        own.append((k, v))
    q = rng.standard_normal((len(lens), n_kv * group * hd)).astype(np.float32)
    out = torch.empty(q.shape, device="cuda")
    rv.paged_attention(dev(q), c, 0, ints(table), ints(lens), scale_of(hd), out)
    got = host(out).astype(np.float64) / top
    assert np.isfinite(got).all()
    for i in range(0, len(lens), 1 if len(lens) < 4 else 29):
        k, v = own[i]
        want, a = attend(q[i], k, v / np.float64(top), n_kv, hd, scale_of(hd))
        check(got[i], want, a, 1.0, f"sequence {i}")
    # Once they are overwritten the rest is as it was, to its last bits.
    few = rows(rng, max(lens), n_kv * hd)
    two = rv.PagedKvCache(1, n_kv, hd, pool, page, "f32")
    for i, n in enumerate(lens):
        for x in (c, two):
            x.append_rows(0, dev(own[i][0]), dev(few[:n]), ints(table), ints(np.arange(n)), ints(np.full(n, i)))
    outs = [rv.paged_attention(dev(q), x, 0, ints(table), ints(lens), scale_of(hd), torch.empty_like(out)) for x in (c, two)]
    assert np.array_equal(host(outs[0]).view(np.uint32), host(outs[1]).view(np.uint32))


@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
def test_very_long_sums_keep_small_weights(hd):
    """1.5 million f32 rows to a workgroup, whose weights next to the first one's add up
    to nothing within one period of the sums, but not over all periods."""
    torch = torch_cuda()
    say(f"case very long sums {hd}")
    n, seqs = 1500000, 300
    c = rv.PagedKvCache(1, 2, hd, -(-n // 1024), 1024, "f32")
    k, v = torch.zeros(n, 2 * hd, device="cuda"), torch.ones(n, 2 * hd, device="cuda")
    k[0, 0] = k[0, hd] = 1.0
    v[1:, :hd] = -1.0  # kv head 0: the first row's value against all others'
    v[0, hd:] = 0.0    # kv head 1: the others' alone
    table = ints(np.random.default_rng(0).permutation(-(-n // 1024))[None])
    c.append_rows(0, k, v, table, ints(np.arange(n)), ints(np.zeros(n)))
    del k, v
    gaps = np.array([28.2, 32.2, 34.2, 36.2]) * np.log(2)  # the first row's score above the others'
    q = np.zeros((2, 4, hd), np.float32)
    q[:, :, 0] = gaps / scale_of(hd)
    q = np.tile(q.reshape(1, -1), (seqs, 1))
    out = torch.empty(seqs, 8 * hd, device="cuda")
    rv.paged_attention(dev(q), c, 0, table.repeat(seqs, 1), ints([n] * seqs), scale_of(hd), out)
    first = np.float32(gaps / scale_of(hd)).astype(np.float64) * scale_of(hd)
    rest = (n - 1) * np.exp(-first)
    want = np.stack([(1 - rest) / (1 + rest), rest / (1 + rest)])
    # A weight is off by the score's 2^-21 times the score, as in the tests above, which
    # moves an average of values 2 apart by twice as much; and check()'s 96 half steps.
    bound = 2 * rest / (1 + rest) * (2 * gaps + 1) * 2.0 ** -21 + 96 * EPS32
    err = np.abs(host(out).reshape(seqs, 2, 4, hd) - want[None, :, :, None]).max((0, 3))
    assert np.all(err <= bound), (err, bound)


@pytest.mark.parametrize("value", [1, 3, -7, 2 ** 40])
def test_join_values_that_mean_nothing_are_refused(value):
    torch_cuda()
    say(f"case join value {value}")
    c = rv.PagedKvCache(1, 2, 64, 4, 16, "f16")
    with pytest.raises(rv.DeviceError) as e:
        c.set_tuning(rv.RV_TUNE_PAGED_JOIN, value)
    assert e.value.variant == "Unsupported"
    c.set_tuning(rv.RV_TUNE_PAGED_JOIN, 0)


def test_outputs_over_what_is_still_read_are_refused():
    """Lengths, positions, tables and sequences inside the rows written; between the rows
    they are none of the call's business."""
    torch = torch_cuda()
    say("case outputs over what is read")
    c = rv.PagedKvCache(1, 2, 64, 8, 16, "f16")
    f = lambda *s: torch.zeros(*s, device="cuda")
    t, at = ints([[0], [1], [2]]), ints([0, 0, 0])
    as_ints = lambda x: x.view(torch.int32)
    wide = f(3, 256 + 8)
    out, flat = wide[:, :256], as_ints(wide).view(-1)
    q, k = f(3, 256), f(3, 128)
    step = lambda pos, tab, o, x=q, y=k, z=k: rv.paged_decode_step(c, 0, x, y, z, None, None, EPS, None, tab, pos, 0.125, o)
    for start in (0, 100, 255, 262, 264 * 2 + 253):  # (of 262's three the last is in a row)
        inside = flat[start:start + 3]
        for call in (lambda: rv.paged_attention(q, c, 0, t, inside, 0.125, out),
                     lambda: rv.paged_attention(q, c, 0, inside.view(3, 1), at, 0.125, out),
                     lambda: step(inside, t, out), lambda: step(at, inside.view(3, 1), out)):
            with pytest.raises(rv.DeviceError) as e:
                call()
            assert e.value.variant == "Unsupported"
    between = flat[264 + 257:264 + 260]
    rv.paged_attention(q, c, 0, t, between, 0.125, out)
    rv.paged_attention(q, c, 0, between.view(3, 1), at, 0.125, out)
    step(between, t, out)
    x = f(3, 256)
    rope = rv.Rope(64, THETA)
    rv.rope_rows(x, between, rope, out)
    with pytest.raises(rv.DeviceError):
        rv.rope_rows(x, flat[250:253], rope, out)
    half = lambda n: torch.zeros(n, dtype=torch.float16, device="cuda")
    kv = half(2 * 3 * 128)
    ok = kv[:384].view(3, 128), kv[384:].view(3, 128)
    c.read_rows(0, t, at, k=ok[0], v=ok[1])
    over = as_ints(ok[0]).view(-1)[10:13]
    for kw in (dict(k=ok[0], v=ok[0]), dict(k=ok[0], v=kv[100:484].view(3, 128))):
        with pytest.raises(rv.DeviceError):
            c.read_rows(0, t, at, **kw)
    for tab, pos, seq in ((t, over, None), (over.view(3, 1), at, None), (t, at, over)):
        with pytest.raises(rv.DeviceError):
            c.read_rows(0, tab, pos, seq, k=ok[0], v=ok[1])
    c.device_status()


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("over", ["q", "k", "v", "all"])
def test_step_over_its_inputs(elem, over):
    """out over any of q, k and v: the bits of a step with rows of its own."""
    torch = torch_cuda()
    say(f"case step over its inputs {(elem, over)}")
    rng = np.random.default_rng(56)
    lens, n_kv, group, hd = [70, 0, 300], 4, 1, 64
    (c, table, _), (d, _, _) = [filled(np.random.default_rng(1), elem, n_kv, hd, 16, lens, extra=1) for _ in range(2)]
    q, k, v, (wq, wk) = step_inputs(rng, 3, n_kv, group, hd)
    args = (dev(wq), dev(wk), EPS, rv.Rope(hd, THETA), ints(table), ints(lens), scale_of(hd))
    want = rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), *args, torch.empty(q.shape, device="cuda"))
    x = {"q": dev(q), "k": dev(k), "v": dev(v)}
    if over == "all":  # rows that overlap q's, k's and v's in one matrix
        fused = torch.cat([x["q"], x["k"], x["v"]], 1).contiguous()
        w = q.shape[1]
        x = {"q": fused[:, :w], "k": fused[:, w:2 * w], "v": fused[:, 2 * w:]}
        out = fused[:, w // 2:w // 2 + w]
    else:
        out = x[over]
    rv.paged_decode_step(d, 1, x["q"], x["k"], x["v"], *args, out)
    assert np.array_equal(host(out).copy().view(np.uint32), host(want).view(np.uint32))
    for a, b in zip(everything(c, 1), everything(d, 1)):
        assert np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,group,hd,r,layout,scaling,lens", [
    (4, 8, 128, 128, "half", "yarn", [0, 1, 63, 300, 4000]), (2, 3, 64, 32, "interleaved", "ntk", [5, -1, 129, 0]),
    (1, 16, 96, 96, "half", "none", [40, 700]), (2, 1, 256, 64, "interleaved", "linear", [7, 130]),
    (1, 2, 512, 512, "half", "none", [9]), (2, 4, 192, 100, "half", "yarn", [33, 0]),
])
def test_step_in_64_bits(elem, n_kv, group, hd, r, layout, scaling, lens):
    """A normed, rotated step against its definition, from the rows given to the output."""
    torch = torch_cuda()
    say(f"case step in 64 bits {(elem, n_kv, group, hd, r, layout, scaling, lens)}")
    rng = np.random.default_rng(hd + r + len(lens))
    n, at, page = len(lens), np.array(lens), 16
    rope = rv.Rope(hd, THETA, r, layout, scaling, factor=4.0, trained_positions=32768)
    gain = rope.frequencies()[1]
    c, table, own = filled(rng, elem, n_kv, hd, page, [max(x, 0) for x in lens], extra=1)
    q, k, v, (wq, wk) = step_inputs(rng, n, n_kv, group, hd)
    out = torch.full(q.shape, 3.0, device="cuda")
    rv.paged_decode_step(c, 1, dev(q), dev(k), dev(v), dev(wq), dev(wk), EPS, rope, ints(table), ints(lens),
                         scale_of(hd), out)
    gk, gv = (host(x).astype(np.float32) for x in c.read_rows(1, ints(table), ints(lens)))
    c.device_status()
    cos, sin = turns(rope, np.maximum(at, 0))

    def exact(x, w):
        """The normed and rotated rows, and how far 32 bits may be from them: the norm's
        reciprocal root and two products (half a step each, one spare), then the rotation."""
        x = x.reshape(n, -1, hd).astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPS))) * w
        off = 4 * EPS32 * np.abs(x)
        off[..., :r] = rotation_bound(x, r, layout, gain)[..., :r] * 2
        return rotated(x, cos, sin, r, layout), off

    (q64, q_off), (k64, k_off) = exact(q, wq), exact(k, wk)
    for got, want, off in ((gk, k64, k_off), (gv, v.reshape(n, n_kv, hd).astype(np.float64), 0.0)):
        got = got.reshape(n, n_kv, hd)
        if elem == "f32":
            bound = off + 0 * np.abs(want)
        elif elem == "f16":
            bound = off + 2.0 ** -11 * (np.abs(want) + off) + 2.0 ** -25
        else:  # half a code, what 32 bits take off or add to it, and the scale's and the value's f16
            top = np.abs(want + off).reshape(n, n_kv, -1, 32).max(-1).repeat(32, -1)
            bound = off + top / 127 * (0.5 + 2.0 ** -16) + 2 * 2.0 ** -11 * top + 2.0 ** -18
        for i in range(n):
            assert np.all(np.abs(got[i] - want[i]) <= bound[i]) if lens[i] >= 0 else not got[i].any()
    for i in range(n):
        if lens[i] < 0:
            assert not host(out)[i].any()
            continue
        ks, vs = np.concatenate([own[i][0], gk[i:i + 1]]), np.concatenate([own[i][1], gv[i:i + 1]])
        want, a = attend(q64[i].reshape(-1), ks, vs, n_kv, hd, scale_of(hd))
        # q's own error moves a score by at most its product with |k|: as much as a larger
        # A would at check()'s 37 half steps.
        kk = np.abs(ks.reshape(-1, n_kv, hd).astype(np.float64))
        moved = max(float((q_off[i].reshape(n_kv, group, hd)[j] @ kk[:, j].T).max()) for j in range(n_kv))
        check(host(out)[i], want, a + moved * scale_of(hd) / np.log(2) / (37 * EPS32), float(np.abs(vs).max()), f"sequence {i}")


def test_a_blocking_streams_capture_is_not_broken_by_the_hand_over():
    """A stream that the null stream waits for is captured while that holds a call: no
    event may be recorded on the null stream then, and the call behind the capture, on
    a third stream, waits for it all the same."""
    import ctypes

    from ramvamp_amd import _lib as L

    torch = torch_cuda()
    say("case blocking capture")
    hip = L.load()  # (its HIP runtime is the process's)
    rng = np.random.default_rng(57)
    lens, n_kv, hd = [300, 40], 2, 128
    c, table, _ = filled(rng, "f16", n_kv, hd, 16, lens)
    k, v = rows(rng, 2, n_kv * hd), rows(rng, 2, n_kv * hd)
    t, n, last, seq = ints(table), ints(lens), ints([m - 1 for m in lens]), ints([0, 1])
    kd, vd, q = dev(k), dev(v), dev(rng.standard_normal((2, 2 * 4 * hd)))
    out = torch.empty(2, 2 * 4 * hd, device="cuda")
    gk, gv = (torch.zeros(2, n_kv * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    big = torch.ones(8192, 8192, device="cuda")
    hold = big @ big
    rv.paged_attention(q, c, 1, t, n, scale_of(hd), out)  # (allocates)
    third = torch.cuda.Stream()
    blocking, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(blocking)) == 0
    second = torch.cuda.ExternalStream(blocking.value)
    torch.cuda.synchronize()
    for _ in range(8):
        torch.mm(big, big, out=hold)
    c.append_rows(1, kd, vd, t, last, seq)
    assert hip.hipStreamBeginCapture(blocking, 0) == 0
    with torch.cuda.stream(second):
        rv.paged_attention(q, c, 1, t, n, scale_of(hd), out)
    assert hip.hipStreamEndCapture(blocking, ctypes.byref(graph)) == 0 and graph.value
    with torch.cuda.stream(third):
        c.read_rows(1, t, last, seq, k=gk, v=gv)
    torch.cuda.synchronize()
    assert np.array_equal(host(gk), k.astype(np.float16)) and np.array_equal(host(gv), v.astype(np.float16))
    assert hip.hipGraphDestroy(graph) == 0
    c.synchronize()  # (on the null stream again)
    assert hip.hipStreamDestroy(blocking) == 0


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_calls_of_many_shapes_in_turn(elem):
    """Grids, batches and joins that differ from call to call, eager and replayed, share
    one cache's partials and tickets: each gives its own bits every time."""
    torch = torch_cuda()
    say(f"case many shapes in turn {elem}")
    rng = np.random.default_rng(58)
    n_kv, hd, lens = 2, 64, [9000, 1, 700, 0, 130, 4000] + [int(x) for x in rng.integers(0, 300, 200)]
    c, table, own = filled(rng, elem, n_kv, hd, 16, lens, junk=False)
    t, all_lens = ints(table), ints(lens)
    calls = []
    for k, group, join in ((1, 4, 0), (len(lens), 4, 0), (2, 1, 0), (6, 20, 0), (6, 4, 2), (3, 16, 0)):
        q = rng.standard_normal((k, n_kv * group * hd)).astype(np.float32)
        calls.append((k, join, dev(q), torch.empty(q.shape, device="cuda"), expect(q, own[:k], n_kv, hd)))

    def run(i):
        k, join, q, out, _ = calls[i]
        c.set_tuning(rv.RV_TUNE_PAGED_JOIN, join)
        rv.paged_attention(q, c, 1, t[:k], all_lens[:k], scale_of(hd), out)

    for i in sorted(range(len(calls)), key=lambda i: -calls[i][3].numel()):
        run(i)  # (allocates)
    torch.cuda.synchronize()
    bits = [host(x[3]).view(np.uint32) for x in calls]
    for b, (k, _, _, _, (want, a, vmax)) in zip(bits, calls):
        for s in range(k):
            check(b[s].view(np.float32), want[s], a, vmax, f"sequence {s} of {k}")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i in (1, 0, 4, 2):
            run(i)
    for rep in range(6):
        order = [int(x) for x in rng.permutation(len(calls))]
        for x in calls:
            x[3].fill_(float("nan"))
        g.replay()
        for i in order[:3]:
            run(i)
        g.replay()
        for i in order[3:]:
            run(i)
        for b, x in zip(bits, calls):
            assert np.array_equal(host(x[3]).view(np.uint32), b), f"turn {rep}"
