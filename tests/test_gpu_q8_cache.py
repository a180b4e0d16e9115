"""The Q8_0 cache: rows in and back bit for bit, and every attention form that
reads one against attention in 64 bits over the values it holds."""
import numpy as np
import pytest

import oracle
import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from ramvamp_amd import block as B
from ramvamp_amd import projections as P
from rows_util import attend, check, q8_blocks, q8_values

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e6
GEOMETRIES = [  # n_kv, group, head_dim, positions
    (4, 8, 128, 1), (4, 8, 128, 2), (4, 8, 128, 31), (4, 8, 128, 32), (4, 8, 128, 33), (4, 8, 128, 127),
    (4, 8, 128, 128), (4, 8, 128, 129), (4, 8, 128, 500), (4, 8, 128, 4097), (2, 1, 128, 77), (3, 5, 128, 65),
    (1, 16, 128, 200), (1, 33, 128, 300), (2, 72, 128, 140), (2, 4, 64, 100), (1, 2, 96, 50), (2, 3, 256, 33),
    (1, 1, 512, 9), (2, 2, 32, 40),
]


def rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[:, 5::37] *= 6  # a few large channels
    return x


def cache(rng, n_layers, n_kv, hd, n, cap=None):
    kv = rv.KvCache(n_layers, n_kv, hd, cap or n, "q8_0")
    held = []
    for layer in range(n_layers):
        k, v = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
        if n:
            kv.append_rows(layer, dev(k), dev(v))
        held.append((q8_values(k), q8_values(v)))
    return kv, held


def scale_of(hd):
    return float(np.float32(1.0) / np.sqrt(np.float32(hd)))


def special(kv_dim, rng):
    """Rows with everything a block can hold."""
    r = rows(rng, 12, kv_dim)
    r[0] = 0
    r[1, :3] = [0.0, -0.0, 2.0 ** -149]
    r[1, 3:32] = 0
    r[2, :32] *= 1e-12
    r[3, :32] = np.float32(1e-40)
    r[4, 3] = np.inf
    r[5, 7] = np.nan
    r[6, 31] = -np.inf
    r[7, 0] = 65468.0
    r[8, 0] = 65520.0
    r[9, 0], r[9, 1] = 3e38, -70000.0
    r[10, :32] = np.arange(32, dtype=np.float32) * 0.5 - 7.75  # ties between codes
    r[11, :] = np.float32(np.finfo(np.float16).max)
    return r


@pytest.mark.parametrize("n_kv,hd", [(4, 128), (3, 32), (1, 64), (2, 96), (1, 512)])
@pytest.mark.parametrize("io", ["device", "host"])
def test_rows_are_the_quantizer_s_blocks(n_kv, hd, io):
    torch_cuda()
    say(f"case q8 rows {(n_kv, hd, io)}")
    rng = np.random.default_rng(hd + n_kv)
    kv_dim = n_kv * hd
    K, V = special(kv_dim, rng), special(kv_dim, rng)[::-1].copy()
    kv = rv.KvCache(2, n_kv, hd, K.shape[0] + 3, "q8_0")
    put = dev if io == "device" else (lambda a: a)
    kv.append(1, put(K[0]), put(V[0]))
    kv.append_rows(1, put(K[1:]), put(V[1:]))
    assert kv.len(1) == K.shape[0] and kv.len(0) == 0
    for x, row in ((K, kv.k_row), (V, kv.v_row)):
        codes, scales = q8_blocks(x)
        for t in range(x.shape[0]):
            got = row(1, t)
            d = got[:, :2].copy().view(np.uint16).reshape(-1)
            want = scales[t].view(np.uint16)
            nan = np.isnan(scales[t])
            assert np.array_equal(d[~nan], want[~nan]) and np.all(np.isnan(d[nan].view(np.float16))), t
            assert np.array_equal(got[:, 2:].view(np.int8), codes[t]), t
            # Blocks inside the format's range are quantize_row_q8_0's.
            for b in range(kv_dim // 32):
                blk = x[t, 32 * b:32 * b + 32]
                if np.all(np.isfinite(blk)) and 1e-30 < np.abs(blk).max() < 65000:
                    o = oracle.quantize_row_q8_0(blk)
                    o = np.frombuffer(np.ascontiguousarray(o).tobytes(), np.uint8)
                    assert np.array_equal(o[4:36].view(np.int8), codes[t, b])
                    assert o[:4].view(np.float32)[0] == np.float32(scales[t, b])
    got = kv.read_rows(1, 0, K.shape[0])
    for g, x in zip(got, (K, V)):
        g, w = host(g), q8_values(x)
        assert np.array_equal(np.isnan(g), np.isnan(w))
        assert np.array_equal(g[~np.isnan(w)], w[~np.isnan(w)])


@pytest.mark.parametrize("elem", ["q8_0", "f16", "f32"])
@pytest.mark.parametrize("hd", [128, 32])
def test_read_rows(elem, hd):
    torch = torch_cuda()
    say(f"case read rows {elem} {hd}")
    rng = np.random.default_rng(5)
    n, n_kv = 133, 2
    K, V = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
    kv = rv.KvCache(3, n_kv, hd, n + 1, elem)
    kv.append_rows(2, dev(K), dev(V))
    fix = {"q8_0": q8_values, "f16": lambda x: x.astype(np.float16).astype(np.float32), "f32": lambda x: x}[elem]
    for lo, m in ((0, n), (0, 1), (n - 1, 1), (31, 66), (n, 0)):
        k, v = kv.read_rows(2, lo, m)
        assert np.array_equal(host(k), fix(K[lo:lo + m])) and np.array_equal(host(v), fix(V[lo:lo + m]))
    k = torch.full((4, n_kv * hd), -1.0, device="cuda")
    assert kv.read_rows(2, 3, 4, k=k)[1] is None
    assert np.array_equal(host(k), fix(K[3:7]))
    hv = np.zeros((4, n_kv * hd), np.float32)
    kv.read_rows(2, 3, 4, v=hv)
    assert np.array_equal(hv, fix(V[3:7]))
    for bad in ((0, n + 1), (n, 1), (n + 1, 0)):
        with pytest.raises(rv.KvError) as e:
            kv.read_rows(2, *bad)
        assert e.value.variant == "PositionOutOfRange" and e.value.fields["layer"] == 2
    with pytest.raises(rv.KvError):
        kv.read_rows(3, 0, 1)
    with pytest.raises(ValueError):
        kv.read_rows(2, 0, 3, k=k)


@pytest.mark.parametrize("count", [134, 1 << 40, -1])
def test_read_rows_past_the_capacity_allocates_nothing(count):
    torch_cuda()
    kv = rv.KvCache(1, 2, 128, 133, "q8_0")
    with pytest.raises(rv.KvError) as e:
        kv.read_rows(0, 0, count)
    assert e.value.variant == "PositionOutOfRange"


@pytest.mark.parametrize("n_kv,group,hd,n", GEOMETRIES)
def test_decode(n_kv, group, hd, n):
    torch = torch_cuda()
    say(f"case q8 decode {(n_kv, group, hd, n)}")
    rng = np.random.default_rng(n + hd)
    kv, held = cache(rng, 2, n_kv, hd, n)
    scale = scale_of(hd)
    q = rng.standard_normal(n_kv * group * hd).astype(np.float32)
    for layer in (1, 0):
        k, v = held[layer]
        want, a = attend(q, k, v, n_kv, hd, scale)
        out = torch.full((q.size,), float("nan"), device="cuda")
        rv.decode_attention(dev(q), kv, layer, scale, None, out)
        check(host(out), want, a, np.abs(v).max(), "decode")
    bits = host(out).view(np.uint32)
    again = torch.full_like(out, float("nan"))
    rv.decode_attention_noalloc(dev(q), kv, 0, scale, again)
    assert np.array_equal(host(again).view(np.uint32), bits)
    ho = np.full(q.size, np.nan, np.float32)
    rv.decode_attention_in(q, kv, 0, scale, rv.scratch_len(n_kv * group, n_kv, hd, n), ho)
    assert np.array_equal(ho.view(np.uint32), bits)
    # One kv head's range is that part of the whole.
    part = torch.full((group * hd,), float("nan"), device="cuda")
    rv.decode_attention_kv_range_in(dev(q), kv, 0, scale, range(n_kv - 1, n_kv), 1 << 40, part)
    w = want[(n_kv - 1) * group * hd:]
    check(host(part), w, a, np.abs(held[0][1]).max(), "kv range")


@pytest.mark.parametrize("n,limit", [(300, 1), (300, 40), (300, 128), (300, 257), (700, 699)])
def test_rows_past_the_limit_do_not_count(n, limit):
    torch = torch_cuda()
    say(f"case q8 attention_at {(n, limit)}")
    rng = np.random.default_rng(limit)
    n_kv, group, hd = 2, 8, 128
    kv, held = cache(rng, 1, n_kv, hd, limit, cap=n + 1)
    bad = rows(rng, n - limit, n_kv * hd)
    bad[::2] = np.nan
    bad[1::2] = np.inf
    kv.append_rows(0, dev(bad), dev(bad))
    k, v = held[0]
    q = rng.standard_normal(n_kv * group * hd).astype(np.float32)
    want, a = attend(q, k, v, n_kv, hd, scale_of(hd))
    out = torch.full((q.size,), float("nan"), device="cuda")
    rv.attention_at(dev(q), kv, 0, limit, scale_of(hd), None, out)
    check(host(out), want, a, np.abs(v).max(), "attention_at")
    # Truncated and written again: the stale rows are gone from the short form too.
    kv.truncate(limit)
    rv.decode_attention(dev(q), kv, 0, scale_of(hd), None, out)
    check(host(out), want, a, np.abs(v).max(), "truncated")


def test_extreme_scores():
    """Scores of either sign far past f32's exponent range for 2^x, all equal, and
    a query of zeros, of tiny and of huge values."""
    torch = torch_cuda()
    say("case q8 extreme scores")
    rng = np.random.default_rng(9)
    n_kv, group, hd, n = 1, 8, 128, 200
    k, v = rows(rng, n, hd), rows(rng, n, hd)
    kv = rv.KvCache(1, n_kv, hd, n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    k, v = q8_values(k), q8_values(v)
    q = rng.standard_normal((group, hd)).astype(np.float32)
    q[0] = 0
    q[1] *= 1e-30
    q[2] *= 1e4
    q[3] *= 1e30
    q[4] = -1e30 * np.sign(k[17])
    q[5] *= 1e-42
    q[6] = 30 * k[60]
    out = torch.full((q.size,), float("nan"), device="cuda")
    rv.decode_attention(dev(q.reshape(-1)), kv, 0, scale_of(hd), None, out)
    got = host(out).reshape(group, hd)
    for h in range(group):
        want, a = attend(q[h], k, v, 1, hd, scale_of(hd))
        if a < 1e4:
            check(got[h], want, a, np.abs(v).max(), f"head {h}")
        else:  # the largest score alone decides, where it leads by more than its rounding
            x = np.sort(q[h].astype(np.float64) @ k.astype(np.float64).T * scale_of(hd) * 1.4427)
            assert x[-1] - x[-2] > 40 + a * 37 * 2.0 ** -24
            check(got[h], want, 1.0, np.abs(v).max(), f"head {h}")


@pytest.mark.parametrize("mode", ["exact", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,group,hd,n,start", [
    (4, 8, 128, 1, 0), (4, 8, 128, 2, 0), (4, 8, 128, 33, 0), (2, 8, 128, 64, 5), (4, 8, 128, 77, 901),
    (2, 5, 128, 40, 127), (2, 1, 128, 200, 130), (1, 7, 128, 150, 64), (1, 40, 128, 9, 100), (1, 8, 128, 130, 2000),
    (2, 2, 64, 20, 11), (1, 3, 96, 7, 0),
])
def test_chunk(mode, n_kv, group, hd, n, start):
    torch = torch_cuda()
    say(f"case q8 chunk {(mode, n_kv, group, hd, n, start)}")
    rng = np.random.default_rng(n + start)
    kv, held = cache(rng, 1, n_kv, hd, start + n, cap=start + n + 7)
    k, v = held[0]
    q = rng.standard_normal((n, n_kv * group * hd)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, scale_of(hd), out, mode)
    got = host(out)
    wants = [attend(q[r], k[:start + r + 1], v[:start + r + 1], n_kv, hd, scale_of(hd)) for r in range(n)]
    # (other head sizes have one arithmetic, f32)
    check(got, np.stack([w for w, _ in wants]), max(a for _, a in wants), np.abs(v).max(), "chunk",
          single=mode != "exact" and hd == 128)


def test_a_nan_row_reaches_only_the_rows_that_see_it():
    torch = torch_cuda()
    say("case q8 chunk NaN")
    rng = np.random.default_rng(3)
    n_kv, group, hd, n, start = 2, 8, 128, 90, 50
    k, v = rows(rng, start + n, n_kv * hd), rows(rng, start + n, n_kv * hd)
    v[start + 40, 32:64] = np.nan      # kv head 0, block 1
    v[start + 71, 3] = np.inf          # kv head 0, block 0
    k[start + 60, 128 + 5] = np.nan    # kv head 1
    kv = rv.KvCache(1, n_kv, hd, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    ks, vs = q8_values(k), q8_values(v)
    q = rng.standard_normal((n, n_kv * group * hd)).astype(np.float32)
    out = torch.full(q.shape, 0.0, device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, scale_of(hd), out)
    got = host(out).reshape(n, n_kv, group, hd)
    for r in range(n):
        want, a = attend(q[r], ks[:start + r + 1], vs[:start + r + 1], n_kv, hd, scale_of(hd))
        want = want.reshape(n_kv, group, hd)
        assert np.isnan(want[0, :, 32:64]).all() == (r >= 40) and np.isnan(want[1]).all() == (r >= 60)
        ok = ~np.isnan(want)
        assert np.array_equal(np.isnan(got[r]), ~ok), r
        clean = np.nanmax(np.abs(vs))
        a_k = float(np.max(np.abs(q[r])) * np.nansum(np.abs(ks), 1).max()) * scale_of(hd) * 1.4427
        check(got[r][ok], want[ok], min(a_k, 400.0), clean, f"row {r}")


def _norm_rope64(x, w, hd, pos):
    h = np.asarray(x, np.float64).reshape(-1, hd)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + EPS) * np.asarray(w, np.float64)
    half = hd // 2
    ang = pos * np.power(THETA, -2.0 * np.arange(half) / hd)
    c, s = np.cos(ang), np.sin(ang)
    return np.concatenate([y[:, :half] * c - y[:, half:] * s, y[:, :half] * s + y[:, half:] * c], 1).reshape(-1)


@pytest.mark.parametrize("n_kv,group,hd,n", [(4, 8, 128, 0), (4, 8, 128, 300), (2, 20, 128, 64), (2, 3, 64, 40),
                                            (1, 2, 96, 5)])
def test_step_and_chunk_prologue(n_kv, group, hd, n):
    """The rows a step or a chunk appends are the blocks of what an f32 cache
    holds after the same call, and the output attends them."""
    torch = torch_cuda()
    say(f"case q8 step {(n_kv, group, hd, n)}")
    rng = np.random.default_rng(n + hd)
    kvd, qd, m = n_kv * hd, n_kv * group * hd, 5
    q8, held = cache(rng, 1, n_kv, hd, n, cap=n + m + 1)
    f32 = rv.KvCache(1, n_kv, hd, n + m + 1, "f32")
    if n:
        f32.append_rows(0, dev(held[0][0]), dev(held[0][1]))
    wq, wk = (rng.uniform(0.9, 1.1, hd).astype(np.float32) for _ in range(2))
    q, k, v = (rng.standard_normal((m + 1, d)).astype(np.float32) for d in (qd, kvd, kvd))
    scale = scale_of(hd)
    outs = []
    for kv in (q8, f32):
        one, many = torch.full((qd,), float("nan"), device="cuda"), torch.full((m, qd), float("nan"), device="cuda")
        rv.decode_step(kv, 0, dev(q[0]), dev(k[0]), dev(v[0]), dev(wq), dev(wk), EPS, THETA, n, scale, one)
        rv.prefill_chunk(kv, 0, dev(q[1:]), dev(k[1:]), dev(v[1:]), dev(wq), dev(wk), EPS, THETA, n + 1, scale, many)
        outs.append(np.concatenate([host(one)[None], host(many)]))
        assert kv.len(0) == n + m + 1
    kf, vf = (host(t) for t in f32.read_rows(0, n, m + 1))
    kq, vq = (host(t) for t in q8.read_rows(0, n, m + 1))
    assert np.array_equal(kq, q8_values(kf)) and np.array_equal(vq, q8_values(vf))
    ka, va = np.concatenate([held[0][0], kq]), np.concatenate([held[0][1], vq])
    for r in range(m + 1):
        qr = _norm_rope64(q[r], wq, hd, n + r)
        want, a = attend(qr, ka[:n + r + 1], va[:n + r + 1], n_kv, hd, scale)
        # q itself carries the prologue's five f32 roundings.
        check(outs[0][r], want, a * 2, np.abs(va).max(), f"row {r}")


def test_device_position_step_in_a_graph():
    torch = torch_cuda()
    say("case q8 token graph")
    rng = np.random.default_rng(77)
    n_kv, group, hd, n, cap, layers = 4, 8, 128, 150, 160, 2
    kvd, qd = n_kv * hd, n_kv * group * hd
    seed = rng.integers(1 << 30)
    graph_kv, _ = cache(np.random.default_rng(seed), layers, n_kv, hd, n, cap=cap)
    eager_kv, _ = cache(np.random.default_rng(seed), layers, n_kv, hd, n, cap=cap)
    wq, wk = (dev(rng.uniform(0.9, 1.1, hd)) for _ in range(2))
    scale = scale_of(hd)
    qb, kb, vb = (torch.zeros(layers, d, device="cuda") for d in (qd, kvd, kvd))
    out = torch.zeros(layers, qd, device="cuda")
    pos = torch.tensor([n], dtype=torch.int32, device="cuda")

    def token():
        for layer in range(layers):
            rv.decode_step_dev(graph_kv, layer, qb[layer], kb[layer], vb[layer], wq, wk, EPS, THETA, pos, cap - 2,
                               scale, out[layer])
        rv.position_advance(graph_kv, pos)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        token()  # sizes the buffers
        pos.fill_(n)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            token()
        for t in range(9):
            q, k, v = (rng.standard_normal((layers, d)).astype(np.float32) for d in (qd, kvd, kvd))
            qb.copy_(dev(q)), kb.copy_(dev(k)), vb.copy_(dev(v))
            out.fill_(float("nan"))
            s.synchronize()
            g.replay()
            s.synchronize()
            got = host(out)
            for layer in range(layers):
                want = torch.full((qd,), float("nan"), device="cuda")
                rv.decode_step(eager_kv, layer, dev(q[layer]), dev(k[layer]), dev(v[layer]), wq, wk, EPS, THETA,
                               n + t, scale, want)
                w = host(want)
                # The same rows and query bits; the splits follow the plan's length.
                d = np.abs(got[layer].astype(np.float64) - w)
                assert np.all(np.isfinite(w)) and d.max() <= 2.0 ** -17 * np.abs(w).max(), (t, layer, d.max())
    # Positions 150 .. 158 are written; 159 is past the plan.
    with torch.cuda.stream(s):
        out.fill_(float("nan"))
        g.replay()
        s.synchronize()
        assert np.isnan(host(out)).all()
        with pytest.raises(rv.KvError) as e:
            graph_kv.commit(0, 9)
        assert e.value.variant == "CapacityExceeded"
        for layer in range(layers):
            graph_kv.commit(layer, 9)
            for a, b in zip(graph_kv.read_rows(layer, 0, n + 9), eager_kv.read_rows(layer, 0, n + 9)):
                assert np.array_equal(host(a), host(b))


@pytest.mark.parametrize("n_kv,group,hd", [(2, 1, 128), (2, 20, 128), (2, 40, 128), (1, 72, 128), (2, 5, 64)])
@pytest.mark.parametrize("n,most", [(0, 0), (3, 700), (300, 300), (300, 2500), (1030, 2500)])
def test_device_position_of_every_group(n_kv, group, hd, n, most):
    """What lies between the token's position and the planned one is not read:
    rows of NaN."""
    torch = torch_cuda()
    say(f"case q8 device position {n_kv}x{group}x{hd} at {n} of {most}")
    rng = np.random.default_rng(n + group)
    kvd, qd, cap = n_kv * hd, n_kv * group * hd, 2501
    kvs = [cache(np.random.default_rng(5), 1, n_kv, hd, n, cap=cap)[0] for _ in range(2)]
    if most > n:
        past = torch.full((most - n, kvd), float("nan"), device="cuda")
        kvs[0].append_rows(0, past, past)
    kvs[0].truncate(n)
    q, k, v = (dev(rng.standard_normal(d).astype(np.float32)) for d in (qd, kvd, kvd))
    wq, wk = (dev(rng.uniform(0.9, 1.1, hd).astype(np.float32)) for _ in range(2))
    pos = torch.tensor([n], dtype=torch.int32, device="cuda")
    got, want = (torch.full((qd,), float("nan"), device="cuda") for _ in range(2))
    rv.decode_step_dev(kvs[0], 0, q, k, v, wq, wk, EPS, THETA, pos, most, scale_of(hd), got)
    rv.decode_step(kvs[1], 0, q, k, v, wq, wk, EPS, THETA, n, scale_of(hd), want)
    w = host(want)
    # The same rows and query bits; the splits follow the plan's length.
    d = np.abs(host(got).astype(np.float64) - w)
    assert np.all(np.isfinite(w)) and d.max() <= 2.0 ** -17 * np.abs(w).max(), d.max()


def test_the_workspace_of_a_growing_context_is_not_kept_at_every_size():
    torch = torch_cuda()
    say("case q8 workspace")
    n_kv, group, hd, steps = 4, 8, 128, 200
    kv = rv.KvCache(1, n_kv, hd, 128 * steps, "q8_0")
    kv.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 128)
    x = torch.randn(128, n_kv * hd, device="cuda")
    q = torch.randn(n_kv * group * hd, device="cuda")
    out = torch.empty_like(q)
    before = kv.device_bytes()[0]
    for _ in range(steps):
        kv.append_rows(0, x, x)
        rv.decode_attention(q, kv, 0, scale_of(hd), None, out)
    # The last call's splits, their 16 columns' values, maximum and sum each.
    need = n_kv * steps * 16 * (hd + 2) * 4
    # A buffer is at most twice what its call needed, those before it sum to no more.
    assert kv.device_bytes()[0] - before <= 4 * need


def test_graph_of_decodes_without_a_first_call():
    """rv_kv_new reserves what a decode needs: captured at once, replayed between
    eager calls that use the same workspace."""
    torch = torch_cuda()
    say("case q8 decode graph")
    rng = np.random.default_rng(12)
    n_kv, group, hd, n = 4, 8, 128, 3000
    kv, held = cache(rng, 2, n_kv, hd, n)
    q = [torch.empty(n_kv * group * hd, device="cuda") for _ in range(2)]
    out = [torch.empty_like(q[0]) for _ in range(2)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        for i in range(2):
            rv.decode_attention(q[i], kv, i, scale_of(hd), None, out[i])
    for t in range(4):
        for i in range(2):
            q[i].copy_(dev(rng.standard_normal(q[i].numel())))
            out[i].fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager = torch.full_like(out[i], float("nan"))
            rv.decode_attention(q[i], kv, i, scale_of(hd), None, eager)
            assert np.array_equal(host(eager).view(np.uint32), host(out[i]).view(np.uint32)), (t, i)
    want, a = attend(host(q[1]), *held[1], n_kv, hd, scale_of(hd))
    check(host(out[1]), want, a, np.abs(held[1][1]).max(), "graph")


def test_two_streams_and_a_misaligned_query():
    torch = torch_cuda()
    say("case q8 streams")
    rng = np.random.default_rng(4)
    n_kv, group, hd, n = 2, 8, 128, 400
    kv, held = cache(rng, 1, n_kv, hd, n)
    k, v = held[0]
    buf = torch.zeros(2 * n_kv * group * hd + 3, device="cuda")
    width = n_kv * group * hd
    for off in (1, 3):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            q = buf[off:off + width]
            out = buf[off + width:off + 2 * width] if off == 1 else torch.empty(width + 1, device="cuda")[1:]
            x = rng.standard_normal(width).astype(np.float32)
            q.copy_(torch.from_numpy(x))
            rv.decode_attention(q, kv, 0, scale_of(hd), None, out)
            s.synchronize()
            want, a = attend(x, k, v, n_kv, hd, scale_of(hd))
            check(out.cpu().numpy(), want, a, np.abs(v).max(), f"offset {off}")


def test_split_lengths_agree():
    torch = torch_cuda()
    say("case q8 split lengths")
    rng = np.random.default_rng(41)
    n_kv, group, hd, n = 2, 8, 128, 1100
    kv, held = cache(rng, 1, n_kv, hd, n)
    q = rng.standard_normal(n_kv * group * hd).astype(np.float32)
    want, a = attend(q, *held[0], n_kv, hd, scale_of(hd))
    for length in (0, 1, 128, 200, 512, 1 << 20):
        kv.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, length)
        out = torch.full((q.size,), float("nan"), device="cuda")
        rv.decode_attention(dev(q), kv, 0, scale_of(hd), None, out)
        check(host(out), want, a, np.abs(held[0][1]).max(), f"split {length}")


def block_weights(rng, hidden, n_kv, group, hd):
    torch = torch_cuda()
    qd, kvd = n_kv * group * hd, n_kv * hd

    def q80(rows_, cols):
        b = np.zeros((rows_ * cols // 32, 34), np.uint8)
        b[:, :2] = np.float16(0.003).tobytes()[0], np.float16(0.003).tobytes()[1]
        b[:, 2:] = rng.integers(0, 256, (b.shape[0], 32))
        return torch.from_numpy(b.reshape(-1)).cuda()

    def q6k(rows_, cols):
        b = rng.integers(0, 256, (rows_ * cols // 256, 210)).astype(np.uint8)
        b[:, 192:208] = rng.integers(0, 20, (b.shape[0], 16))
        b[:, 208:210] = np.frombuffer(np.float16(0.0004).tobytes(), np.uint8)
        return torch.from_numpy(b.reshape(-1)).cuda()

    return B.AttnBlockWeights(torch.ones(hidden, device="cuda"), P.Q6_K, q6k(qd, hidden), q80(kvd, hidden), P.Q6_K,
                              q6k(kvd, hidden), torch.ones(hd, device="cuda"), torch.ones(hd, device="cuda"), P.Q6_K,
                              q6k(hidden, qd))


def test_the_block_s_token_graph():
    """rv_attn_block_decode_dev captured once and replayed for every token over a
    Q8_0 cache is rv_attn_block_decode (one split of the positions either way: the
    same bits); a token past the plan leaves its residual as it was."""
    torch = torch_cuda()
    say("case q8 block graph")
    rng = np.random.default_rng(18)
    hidden, n_kv, group, hd, n, cap = 512, 4, 8, 128, 70, 75
    qd = n_kv * group * hd
    w = block_weights(rng, hidden, n_kv, group, hd)
    graph_kv, eager_kv = (cache(np.random.default_rng(2), 1, n_kv, hd, n, cap=cap)[0] for _ in range(2))
    pos = torch.tensor([n], dtype=torch.int32, device="cuda")
    res = torch.zeros(hidden, device="cuda")
    scratch = torch.empty(max(256, B.scratch_bytes(hidden, qd, n_kv * hd)), dtype=torch.uint8, device="cuda")

    def token():
        B.attn_block_decode_dev(graph_kv, 0, res, qd, w, EPS, THETA, pos, cap - 2, scale_of(hd), scratch)
        rv.position_advance(graph_kv, pos)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        token()  # sizes the buffers
        pos.fill_(n)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            token()
        for t in range(cap - 1 - n):
            x = dev(rng.standard_normal(hidden).astype(np.float32))
            res.copy_(x)
            g.replay()
            s.synchronize()
            B.attn_block_decode(eager_kv, 0, x, qd, w, EPS, THETA, n + t, scale_of(hd))
            assert np.array_equal(host(res), host(x)), t
        x = dev(rng.standard_normal(hidden).astype(np.float32))
        res.copy_(x)
        g.replay()
        s.synchronize()
        assert np.array_equal(host(res), host(x))
        with pytest.raises(rv.KvError) as e:
            graph_kv.commit(0, cap - 1 - n)
        assert e.value.variant == "CapacityExceeded"


def test_the_layer_s_attention_block():
    """rv_attn_block_decode and _prefill over a Q8_0 cache are their parts."""
    torch = torch_cuda()
    say("case q8 block")
    rng = np.random.default_rng(8)
    hidden, n_kv, group, hd, n = 512, 4, 8, 128, 70
    qd, kvd = n_kv * group * hd, n_kv * hd

    def q80(rows_, cols):
        b = np.zeros((rows_ * cols // 32, 34), np.uint8)
        b[:, :2] = np.float16(0.003).tobytes()[0], np.float16(0.003).tobytes()[1]
        b[:, 2:] = rng.integers(0, 256, (b.shape[0], 32))
        return torch.from_numpy(b.reshape(-1)).cuda()

    def q6k(rows_, cols):
        b = rng.integers(0, 256, (rows_ * cols // 256, 210)).astype(np.uint8)
        b[:, 192:208] = rng.integers(0, 20, (b.shape[0], 16))
        b[:, 208:210] = np.frombuffer(np.float16(0.0004).tobytes(), np.uint8)
        return torch.from_numpy(b.reshape(-1)).cuda()

    ones = torch.ones(hidden, device="cuda")
    w = B.AttnBlockWeights(ones, P.Q6_K, q6k(qd, hidden), q80(kvd, hidden), P.Q6_K, q6k(kvd, hidden),
                           torch.ones(hd, device="cuda"), torch.ones(hd, device="cuda"), P.Q6_K, q6k(hidden, qd))
    caches = [cache(np.random.default_rng(2), 1, n_kv, hd, n, cap=n + 9)[0] for _ in range(2)]
    x = rng.standard_normal(hidden).astype(np.float32)
    res = dev(x)
    B.attn_block_decode(caches[0], 0, res, qd, w, EPS, THETA, n, scale_of(hd))
    normed = oracle.rmsnorm(x, np.ones(hidden, np.float32), EPS)
    q, k, v, o = (torch.empty(d, device="cuda") for d in (qd, kvd, kvd, hidden))
    P.attn_in_proj(dev(normed), P.Q6_K, w.wq, q, w.wk, k, P.Q6_K, w.wv, v)
    att = torch.empty(qd, device="cuda")
    rv.decode_step(caches[1], 0, q, k, v, w.q_norm, w.k_norm, EPS, THETA, n, scale_of(hd), att)
    P.attn_out_proj(att, P.Q6_K, w.wo, o)
    assert np.array_equal(host(res), x + host(o))
    rows_ = rng.standard_normal((6, hidden)).astype(np.float32)
    res = dev(rows_)
    B.attn_block_prefill(caches[0], 0, res, qd, w, EPS, THETA, n + 1, scale_of(hd))
    normed = np.stack([oracle.rmsnorm(r, np.ones(hidden, np.float32), EPS) for r in rows_])
    q, k, v = (torch.empty(6, d, device="cuda") for d in (qd, kvd, kvd))
    P.attn_in_proj_rows(dev(normed), P.Q6_K, w.wq, q, w.wk, k, P.Q6_K, w.wv, v)
    att, want = torch.empty(6, qd, device="cuda"), dev(rows_)
    rv.prefill_chunk(caches[1], 0, q, k, v, w.q_norm, w.k_norm, EPS, THETA, n + 1, scale_of(hd), att)
    P.attn_out_proj_rows(att, P.Q6_K, w.wo, want)
    assert np.array_equal(host(res), host(want))


def test_bookkeeping_and_refusals():
    torch = torch_cuda()
    say("case q8 bookkeeping")
    kv = rv.KvCache(3, 2, 64, 130, "q8_0")
    assert kv.elem == "q8_0"
    assert rv.KvCache.projected_bytes(3, 2, 64, 130, "q8_0") == 2 * 3 * 130 * 128 * 34 // 32
    now, bound = kv.device_bytes()
    assert now >= 2 * 3 * 256 * 128 * 34 // 32 and bound >= now
    assert rv.KvCache.projected_device_bytes(3, 2, 64, 130, "q8_0") >= bound  # (counts 1 MiB of workspace)
    big = rv.KvCache(2, 2, 128, 130, "q8_0")
    assert rv.KvCache.projected_device_bytes(2, 2, 128, 130, "q8_0") == big.device_bytes()[1]
    x = torch.zeros(130, 128, device="cuda")
    kv.append_rows(0, x, x)
    with pytest.raises(rv.KvError) as e:
        kv.append(0, x[0], x[0])
    assert e.value.variant == "CapacityExceeded"
    for view in (kv.k_layer, kv.v_layer):
        with pytest.raises(rv.DeviceError) as e:
            view(0)
        assert e.value.variant == "Unsupported"
    for hd in (48, 16, 544, 1):
        with pytest.raises(rv.KvError) as e:
            rv.KvCache(1, 2, hd, 8, "q8_0")
        assert e.value.variant == "InvalidDims"
    # One layer's length alone.
    kv.append_rows(2, x[:20], x[:20])
    kv.truncate_layer(0, 7)
    assert [kv.len(i) for i in range(3)] == [7, 0, 20]
    with pytest.raises(rv.KvError) as e:
        kv.truncate_layer(0, 8)
    assert e.value.variant == "TruncateBeyondLength" and e.value.fields == {"requested": 8, "len": 7}
    with pytest.raises(rv.KvError):
        kv.truncate_layer(3, 0)
    out = torch.full((4 * 64,), 5.0, device="cuda")
    with pytest.raises(rv.AttentionError):
        rv.decode_attention(torch.zeros(4 * 64, device="cuda"), kv, 1, 1.0, None, out)
    assert (host(out) == 5.0).all()


@pytest.mark.parametrize("call", ["step", "chunk"])
def test_a_step_refused_for_its_workspace_appends_nothing(call):
    """Under capture a workspace cannot grow; the same call uncaptured then succeeds."""
    torch = torch_cuda()
    say(f"case q8 refused {call}")
    rng = np.random.default_rng(60)
    n_kv, group, hd, n = 2, 72, 128, 5000
    kvd, qd = n_kv * hd, n_kv * group * hd
    m = 1 if call == "step" else 20
    kv, held = cache(rng, 2, n_kv, hd, n, cap=n + m)
    q, k, v = (dev(rng.standard_normal((m, d))) for d in (qd, kvd, kvd))
    w = torch.ones(hd, device="cuda")

    def run(layer, out):
        if call == "step":
            rv.decode_step(kv, layer, q[0], k[0], v[0], w, w, EPS, THETA, n, scale_of(hd), out[0])
        else:
            rv.prefill_chunk(kv, layer, q, k, v, w, w, EPS, THETA, n, scale_of(hd), out)

    first, second = (torch.full((m, qd), float("nan"), device="cuda") for _ in range(2))
    # One split: the query's buffer is there afterwards, no more workspace.
    kv.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 8192)
    run(0, first)
    torch.cuda.synchronize()
    # As many as there can be.
    kv.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 128)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(rv.DeviceError):
            run(1, second)
    assert kv.len(1) == n and np.isnan(host(second)).all()
    run(1, second)
    assert kv.len(1) == n + m
    kk, vv = (host(x) for x in kv.read_rows(1, 0, n + m))
    got = host(second)
    for r in (0, m - 1):
        qr = _norm_rope64(host(q[r]), np.ones(hd), hd, n + r)
        want, a = attend(qr, kk[:n + r + 1], vv[:n + r + 1], n_kv, hd, scale_of(hd))
        check(got[r], want, 2 * a, np.abs(vv).max(), f"row {r}")
