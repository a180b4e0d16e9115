"""Decode for a batch that shares a prefix, against attention in 64 bits over
each sequence's own rows behind the prefix's."""
import numpy as np
import pytest

import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from rows_util import EPS32, LOG2E, attend, check, stored

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e6


def rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[:, 5::37] *= 6
    return x


def scale_of(hd):
    return float(np.float32(1.0) / np.sqrt(np.float32(hd)))


def batch(rng, elem, n_kv, hd, prefix, tails, room=None, junk=0):
    """(prefix cache, tails cache, the values of each); junk: NaN rows behind the
    prefix's, which the batch does not attend."""
    kvd = n_kv * hd
    p = rv.KvCache(2, n_kv, hd, max(prefix + junk, 1), elem)
    pk, pv = rows(rng, prefix, kvd), rows(rng, prefix, kvd)
    if prefix:
        p.append_rows(1, dev(pk), dev(pv))
    if junk:
        bad = np.full((junk, kvd), np.nan, np.float32)
        p.append_rows(1, dev(bad), dev(bad))
    t = rv.KvCache(len(tails) + 3, n_kv, hd, room or max(max(tails), 1), elem)
    own = []
    for i, n in enumerate(tails):
        k, v = rows(rng, n, kvd), rows(rng, n, kvd)
        if n:
            t.append_rows(2 + i, dev(k), dev(v))
        own.append((stored(k, elem), stored(v, elem)))
    bad = np.full((1, kvd), np.nan, np.float32)
    t.append_rows(1, dev(bad), dev(bad))  # a slot beside the batch's
    return p, t, (stored(pk, elem), stored(pv, elem)), own


def expect(q, pre, own, n_kv, hd, check_rows=None):
    outs, a, vmax = [], 0.0, 0.0
    for i in range(q.shape[0]) if check_rows is None else check_rows:
        k, v = np.concatenate([pre[0], own[i][0]]), np.concatenate([pre[1], own[i][1]])
        w, ai = attend(q[i], k, v, n_kv, hd, scale_of(hd))
        outs.append(w)
        a, vmax = max(a, ai), max(vmax, float(np.abs(v).max()))
    return np.stack(outs), a, vmax


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("n_kv,group,hd,prefix,tails", [
    (4, 8, 128, 100, [5]),
    (4, 8, 128, 129, [0, 3]),
    (4, 8, 128, 0, [1, 40, 33]),
    (2, 8, 128, 1, [0, 0, 1, 200, 128, 129]),
    (4, 8, 128, 1000, [7, 0, 31, 32, 33, 127, 300, 2, 64]),
    (2, 1, 128, 300, list(range(40))),
    (2, 5, 128, 77, [4, 9, 1]),
    (1, 40, 128, 60, [10, 0]),
    (1, 16, 128, 2500, [3] * 20),
    (2, 4, 64, 50, [0, 12, 5]),
    (1, 2, 96, 7, [1, 2]),
])
def test_shared_decode(elem, n_kv, group, hd, prefix, tails):
    torch = torch_cuda()
    say(f"case shared {(elem, n_kv, group, hd, prefix, tails)}")
    rng = np.random.default_rng(prefix + len(tails))
    p, t, pre, own = batch(rng, elem, n_kv, hd, prefix, tails, junk=3)
    q = rng.standard_normal((len(tails), n_kv * group * hd)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 1, prefix, t, 2, scale_of(hd), out)
    want, a, vmax = expect(q, pre, own, n_kv, hd)
    got = host(out)
    check(got, want, a, vmax, "shared")
    # Host pointers and a second call: the same bits.
    ho = np.full(q.shape, np.nan, np.float32)
    rv.decode_attention_shared(q, p, 1, prefix, t, 2, scale_of(hd), ho)
    assert np.array_equal(ho.view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("columns", [0, 32, 128, 256])
@pytest.mark.parametrize("case", ["v_1e6", "v_1e-30", "v_1e37", "v_rows_1e-30_to_1e6", "v_later_larger", "v_later_smaller",
                                  "v_zero_then_1e-30", "v_dims_1e-5", "k_rows_1e-25_to_1", "k_1e20_q_1e-20",
                                  "k_1e-20_q_1e20", "k_1e-30", "k_1e-33_q_1e-30"])
def test_f32_planes_of_any_range(case, columns):
    """Finite f32 values far outside f16's range, K's, V's and q's. On top of
    rows_util's bounds, each value is held to 2^-22 of itself or 2^-34 of the
    largest of the rows computed with it, whichever is larger."""
    torch_cuda()
    say(f"case f32 range {case} {columns}")
    rng = np.random.default_rng(len(case))
    n_kv, group, hd, prefix, tails = 2, 8, 128, 700, [0, 3, 70, 130, 31, 64, 1, 5, 9]
    n, kvd = prefix, n_kv * hd
    total = prefix + sum(tails)
    k, v = (rng.standard_normal((total, kvd)) for _ in range(2))
    q = rng.standard_normal((len(tails), n_kv * group * hd))
    decades = rng.uniform(0, 1, (total, 1))
    order = np.arange(total)[:, None]
    if case == "v_1e6":
        v *= 1e6
    elif case == "v_1e-30":
        v *= 1e-30
    elif case == "v_1e37":
        v *= 1e37
    elif case == "v_rows_1e-30_to_1e6":
        v *= 10.0 ** (-30 + 36 * decades)
    elif case == "v_later_larger":
        v *= np.where(order % prefix < 300, 1e-12, 1e4)
    elif case == "v_later_smaller":
        v *= np.where(order % prefix < 300, 1e9, 1e-6)
    elif case == "v_zero_then_1e-30":
        v *= np.where(order % prefix < 400, 0.0, 1e-30)
    elif case == "v_dims_1e-5":
        v[:, ::3] *= 1e-5
    elif case == "k_rows_1e-25_to_1":
        k *= 10.0 ** (-25 + 25 * decades)
    elif case == "k_1e20_q_1e-20":
        k, q = k * 1e20, q * 1e-20
    elif case == "k_1e-20_q_1e20":
        k, q = k * 1e-20, q * 1e20
    elif case == "k_1e-30":
        k *= 1e-30
    elif case == "k_1e-33_q_1e-30":  # the scores' scale itself underflows
        k, q = k * 1e-33, q * 1e-30
    k, v, q = (x.astype(np.float32) for x in (k, v, q))
    p = rv.KvCache(1, n_kv, hd, prefix, "f32")
    p.append_rows(0, dev(k[:n]), dev(v[:n]))
    t = rv.KvCache(len(tails), n_kv, hd, max(tails), "f32")
    for c in (p, t):
        c.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    out = dev(np.full(q.shape, np.nan, np.float32))
    seqs, at = [], n
    for i, m in enumerate(tails):
        if m:
            t.append_rows(i, dev(k[at:at + m]), dev(v[at:at + m]))
        seqs.append((np.concatenate([k[:n], k[at:at + m]]), np.concatenate([v[:n], v[at:at + m]])))
        at += m
    rv.decode_attention_shared(dev(q), p, 0, n, t, 0, scale_of(hd), out)
    got = host(out)
    assert np.all(np.isfinite(got))
    for i, (ki, vi) in enumerate(seqs):
        want, a = attend(q[i], ki, vi, n_kv, hd, scale_of(hd))
        terms, _ = attend(q[i], ki, np.abs(vi), n_kv, hd, scale_of(hd))
        q1 = np.abs(q[i].reshape(-1, hd).astype(np.float64)).sum(-1).max() * scale_of(hd) * LOG2E
        score = 37 * EPS32 * a + 2.0 ** -34 * q1 * np.abs(ki).max()
        prob = np.log(2.0) * score + 2.0 ** -22
        bound = terms * (2 * prob + 2.0 ** -22 + 96 * EPS32) + 2.0 ** -34 * float(np.abs(vi).max())
        err = np.abs(got[i].astype(np.float64) - want)
        assert np.all(err <= bound), (i, float(np.max(err / np.maximum(bound, 1e-300))))


def test_more_sequences_than_one_launch_takes():
    torch = torch_cuda()
    say("case shared 300")
    rng = np.random.default_rng(1)
    n_kv, group, hd, n = 1, 2, 128, 300
    tails = [(i * 7) % 23 for i in range(n)]
    p, t, pre, own = batch(rng, "f16", n_kv, hd, 90, tails)
    q = rng.standard_normal((n, n_kv * group * hd)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 1, 90, t, 2, scale_of(hd), out)
    want, a, vmax = expect(q, pre, own, n_kv, hd)
    check(host(out), want, a, vmax, "300 sequences")
    k, v = rows(rng, n, hd), rows(rng, n, hd)
    t2 = rv.KvCache(n + 2, n_kv, hd, 30, "f16")
    t2.append_each(2, dev(k), dev(v))
    assert [t2.len(i) for i in (0, 1, 2, n + 1)] == [0, 0, 1, 1]
    for i in (0, 255, 256, n - 1):
        assert np.array_equal(host(t2.read_rows(2 + i, 0, 1)[0])[0], stored(k[i], "f16"))


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("hd", [128, 64])
def test_one_row_to_each(elem, hd):
    torch_cuda()
    say(f"case append each {elem} {hd}")
    rng = np.random.default_rng(6)
    n_kv, n = 3, 5
    kv = rv.KvCache(n + 1, n_kv, hd, 4, elem)
    held = [[] for _ in range(n + 1)]
    for step in range(4):
        k, v = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
        if step % 2:
            kv.append_each(1, k, v)
        else:
            kv.append_each(1, dev(k), dev(v))
        for i in range(n):
            held[1 + i].append((k[i], v[i]))
        if step == 1:
            kv.truncate_layer(3, 1)
            held[3] = held[3][:1]
    assert [kv.len(i) for i in range(n + 1)] == [0, 4, 4, 3, 4, 4]
    for i in range(1, n + 1):
        k, v = kv.read_rows(i, 0, len(held[i]))
        assert np.array_equal(host(k), stored(np.stack([a for a, _ in held[i]]), elem))
        assert np.array_equal(host(v), stored(np.stack([b for _, b in held[i]]), elem))
    with pytest.raises(rv.KvError) as e:
        kv.append_each(0, dev(np.zeros((n + 1, n_kv * hd))), dev(np.zeros((n + 1, n_kv * hd))))
    assert e.value.variant == "CapacityExceeded" and e.value.fields == {"layer": 1, "capacity": 4}
    assert kv.len(0) == 0
    with pytest.raises(rv.KvError) as e:
        kv.append_each(4, dev(np.zeros((3, n_kv * hd))), dev(np.zeros((3, n_kv * hd))))
    assert e.value.variant == "LayerOutOfRange"
    with pytest.raises(ValueError):
        kv.append_each(0, np.zeros(5, np.float32), np.zeros(5, np.float32))


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_step_is_each_sequence_s_own(elem):
    """decode_step_shared against decode_step on caches that hold prefix and tail."""
    torch = torch_cuda()
    say(f"case shared step {elem}")
    rng = np.random.default_rng(15)
    n_kv, group, hd, prefix, tails = 2, 8, 128, 70, [0, 3, 17, 1]
    qd, kvd = n_kv * group * hd, n_kv * hd
    p, t, pre, own = batch(rng, elem, n_kv, hd, prefix, tails, room=40)
    wq, wk = (rng.uniform(0.9, 1.1, hd).astype(np.float32) for _ in range(2))
    single = []
    for i in range(len(tails)):
        kv = rv.KvCache(1, n_kv, hd, 200, elem)
        # (the values a cache reads back quantize to themselves but for their
        # scale's last bit, so the whole caches are checked through read_rows)
        kv.append_rows(0, dev(pre[0]), dev(pre[1]))
        if tails[i]:
            kv.append_rows(0, dev(own[i][0]), dev(own[i][1]))
        single.append(kv)
    lens = list(tails)
    for step in range(3):
        q, k, v = (rng.standard_normal((len(tails), d)).astype(np.float32) for d in (qd, kvd, kvd))
        out = torch.full((len(tails), qd), float("nan"), device="cuda")
        rv.decode_step_shared(p, 1, prefix, t, 2, dev(q), dev(k), dev(v), dev(wq), dev(wk), EPS, THETA, scale_of(hd),
                              out)
        got = host(out)
        for i, kv in enumerate(single):
            one = torch.full((qd,), float("nan"), device="cuda")
            rv.decode_step(kv, 0, dev(q[i]), dev(k[i]), dev(v[i]), dev(wq), dev(wk), EPS, THETA, prefix + lens[i],
                           scale_of(hd), one)
            mine = t.read_rows(2 + i, lens[i], 1)
            theirs = kv.read_rows(0, prefix + lens[i], 1)
            for a, b in zip(mine, theirs):
                assert np.array_equal(host(a), host(b)), (step, i)
            if elem != "q8_0":
                w = host(one).astype(np.float64)
                assert np.abs(got[i] - w).max() <= 2.0 ** -16 * np.abs(w).max(), (step, i)
            lens[i] += 1
    assert [t.len(2 + i) for i in range(len(tails))] == lens
    # Host pointers: the same step from numpy arrays.
    q, k, v = (rng.standard_normal((len(tails), d)).astype(np.float32) for d in (qd, kvd, kvd))
    ho = np.full((len(tails), qd), np.nan, np.float32)
    rv.decode_step_shared(p, 1, prefix, t, 2, q, k, v, wq, wk, EPS, THETA, scale_of(hd), ho)
    for i in range(len(tails)):
        t.truncate_layer(2 + i, lens[i])
    out = torch.full((len(tails), qd), float("nan"), device="cuda")
    rv.decode_step_shared(p, 1, prefix, t, 2, dev(q), dev(k), dev(v), dev(wq), dev(wk), EPS, THETA, scale_of(hd), out)
    assert np.array_equal(host(out).view(np.uint32), ho.view(np.uint32))


@pytest.mark.parametrize("elem", ["q8_0", "f16"])
def test_serving_run(elem):
    """A prompt prefilled once, a batch of requests behind it over two layers, one
    of them ending and its slot taken by another: each step's attention against 64
    bits over the rows the caches hold, with the query the step prepared."""
    torch = torch_cuda()
    say(f"case serving run {elem}")
    rng = np.random.default_rng(30)
    layers, n_kv, group, hd, prompt, seqs = 2, 4, 8, 128, 150, 5
    qd, kvd = n_kv * group * hd, n_kv * hd
    pre = rv.KvCache(layers, n_kv, hd, 512, elem)
    tails = rv.KvCache(layers * seqs, n_kv, hd, 16, elem)
    ones = dev(np.ones(hd))
    for layer in range(layers):
        for lo, hi in ((0, 100), (100, prompt)):
            q, k, v = (dev(rng.standard_normal((hi - lo, d))) for d in (qd, kvd, kvd))
            rv.prefill_chunk(pre, layer, q, k, v, ones, ones, EPS, THETA, lo, scale_of(hd), torch.empty_like(q))
    for step in range(6):
        if step == 3:
            for layer in range(layers):
                tails.truncate_layer(layer * seqs + 2, 0)
        for layer in range(layers):
            q, k, v = (rng.standard_normal((seqs, d)).astype(np.float32) for d in (qd, kvd, kvd))
            out = torch.full((seqs, qd), float("nan"), device="cuda")
            rv.decode_step_shared(pre, layer, prompt, tails, layer * seqs, dev(q), dev(k), dev(v), ones, ones, EPS,
                                  THETA, scale_of(hd), out)
            pk, pv = (host(x) for x in pre.read_rows(layer, 0, prompt))
            got = host(out)
            for i in range(seqs):
                n = tails.len(layer * seqs + i)
                assert n == (step - 3 if i == 2 and step >= 3 else step) + 1
                tk, tv = (host(x) for x in tails.read_rows(layer * seqs + i, 0, n))
                h = q[i].astype(np.float64).reshape(-1, hd)
                y = h / np.sqrt((h * h).mean(-1, keepdims=True) + EPS)
                ang = (prompt + n - 1) * np.power(THETA, -2.0 * np.arange(hd // 2) / hd)
                c, s = np.cos(ang), np.sin(ang)
                y = np.concatenate([y[:, :64] * c - y[:, 64:] * s, y[:, :64] * s + y[:, 64:] * c], 1)
                kk, vv = np.concatenate([pk, tk]), np.concatenate([pv, tv])
                want, a = attend(y.reshape(-1), kk, vv, n_kv, hd, scale_of(hd))
                check(got[i], want, 2 * a, np.abs(vv).max(), f"step {step} layer {layer} sequence {i}")


@pytest.mark.parametrize("elem", ["f16", "q8_0"])
def test_captured_and_replayed(elem):
    torch = torch_cuda()
    say(f"case shared graph {elem}")
    rng = np.random.default_rng(21)
    n_kv, group, hd, prefix, tails = 4, 8, 128, 600, [4, 0, 90, 33]
    p, t, pre, own = batch(rng, elem, n_kv, hd, prefix, tails)
    q = torch.zeros(len(tails), n_kv * group * hd, device="cuda")
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        rv.decode_attention_shared(q, p, 1, prefix, t, 2, scale_of(hd), out)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            rv.decode_attention_shared(q, p, 1, prefix, t, 2, scale_of(hd), out)
        for _ in range(4):
            x = rng.standard_normal(tuple(q.shape)).astype(np.float32)
            q.copy_(torch.from_numpy(x))
            out.fill_(float("nan"))
            g.replay()
            s.synchronize()
            got = host(out)
            eager = torch.full_like(out, float("nan"))
            rv.decode_attention_shared(q, p, 1, prefix, t, 2, scale_of(hd), eager)
            assert np.array_equal(host(eager).view(np.uint32), got.view(np.uint32))
            want, a, vmax = expect(x, pre, own, n_kv, hd)
            check(got, want, a, vmax, "replay")


def test_one_cache_for_both():
    """The prefix and the batch's rows as layers of one cache."""
    torch = torch_cuda()
    say("case shared one cache")
    rng = np.random.default_rng(33)
    n_kv, group, hd = 2, 8, 128
    kv = rv.KvCache(4, n_kv, hd, 200, "f16")
    held = []
    for layer, n in enumerate((200, 3, 0, 50)):
        k, v = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
        if n:
            kv.append_rows(layer, dev(k), dev(v))
        held.append((stored(k, "f16"), stored(v, "f16")))
    q = rng.standard_normal((3, n_kv * group * hd)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), kv, 0, 150, kv, 1, scale_of(hd), out)
    want, a, vmax = expect(q, (held[0][0][:150], held[0][1][:150]), held[1:], n_kv, hd)
    check(host(out), want, a, vmax, "one cache")


def test_refusals():
    torch = torch_cuda()
    say("case shared refusals")
    n_kv, hd = 2, 128
    x = torch.zeros(4, n_kv * hd, device="cuda")
    p, t = rv.KvCache(1, n_kv, hd, 8, "f16"), rv.KvCache(3, n_kv, hd, 4, "f16")
    p.append_rows(0, x, x)
    q = torch.zeros(3, 4 * hd, device="cuda")
    out = torch.full_like(q, 7.0)

    def refused(cls, variant, *args, q=q, out=out, prefix=p, tails=t, **fields):
        with pytest.raises(cls) as e:
            rv.decode_attention_shared(q, prefix, args[0], args[1], tails, args[2], 1.0, out)
        assert e.value.variant == variant, e.value
        for k, v in fields.items():
            assert e.value.fields[k] == v, e.value
        assert (host(out) == 7.0).all()

    refused(rv.KvError, "PositionOutOfRange", 0, 5, 0, pos=4, len=4)
    refused(rv.KvError, "LayerOutOfRange", 1, 1, 0, layer=1)
    refused(rv.KvError, "LayerOutOfRange", 0, 1, 1)
    refused(rv.KvError, "LayerOutOfRange", 0, 1, 3)
    refused(rv.AttentionError, "EmptyLayer", 0, 0, 0, layer=0)
    for bad in (rv.KvCache(3, n_kv, hd, 4, "q8_0"), rv.KvCache(3, 1, hd, 4, "f16"), rv.KvCache(3, n_kv, 64, 4, "f16")):
        refused(rv.DeviceError, "Unsupported", 0, 4, 0, tails=bad)
    odd, odd_out = torch.zeros(3, 4 * hd + 1, device="cuda"), torch.full((3, 4 * hd + 1), 7.0, device="cuda")
    refused(rv.AttentionError, "QLenIndivisible", 0, 4, 0, q=odd, out=odd_out)
    three, three_out = torch.zeros(3, 3 * hd, device="cuda"), torch.full((3, 3 * hd), 7.0, device="cuda")
    refused(rv.AttentionError, "GqaGroupMismatch", 0, 4, 0, q=three, out=three_out)
    with pytest.raises(ValueError):
        rv.decode_attention_shared(q, p, 0, 4, t, 0, 1.0, out[:2])
    # No sequence: nothing to do.
    rv.decode_attention_shared(q[:0], p, 0, 4, t, 0, 1.0, out[:0])
    # A full slot refuses the whole step.
    t.append_rows(1, x, x)
    w = torch.ones(hd, device="cuda")
    with pytest.raises(rv.KvError) as e:
        rv.decode_step_shared(p, 0, 4, t, 0, q, x[:3], x[:3], w, w, EPS, THETA, 1.0, out)
    assert e.value.variant == "CapacityExceeded" and e.value.fields["layer"] == 1
    assert [t.len(i) for i in range(3)] == [0, 4, 0] and (host(out) == 7.0).all()
    with pytest.raises(rv.PrimitiveError):
        rv.decode_step_shared(p, 0, 4, t, 0, q, x[:3], x[:3], w[:5], w, EPS, THETA, 1.0, out)
    with pytest.raises(ValueError):
        rv.decode_step_shared(p, 0, 4, t, 0, q, x[:2], x[:2], w, w, EPS, THETA, 1.0, out)


@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("prefix,tails", [(70, [0, 3, 17, 1]), (700, [40, 0, 129, 7, 1])])
def test_step_s_output_is_each_sequence_s_own(elem, prefix, tails):
    """The same float rows given to the batch's caches and to one cache a sequence, so
    that the stored blocks are the same for every element type: decode_step_shared's
    outputs are decode_step's but for the order of the sums, each within
    rows_util.check's bound of the exact ones."""
    torch = torch_cuda()
    say(f"case shared step's output {(elem, prefix, tails)}")
    rng = np.random.default_rng(prefix)
    n_kv, group, hd = 2, 8, 128
    qd, kvd = n_kv * group * hd, n_kv * hd
    ks, vs = rows(rng, prefix, kvd), rows(rng, prefix, kvd)
    own = [(rows(rng, n, kvd), rows(rng, n, kvd)) for n in tails]
    p, t = rv.KvCache(1, n_kv, hd, prefix, elem), rv.KvCache(len(tails), n_kv, hd, max(tails) + 3, elem)
    p.append_rows(0, dev(ks), dev(vs))
    single = []
    for i, (k, v) in enumerate(own):
        kv = rv.KvCache(1, n_kv, hd, prefix + tails[i] + 3, elem)
        kv.append_rows(0, dev(ks), dev(vs))
        if tails[i]:
            t.append_rows(i, dev(k), dev(v))
            kv.append_rows(0, dev(k), dev(v))
        single.append(kv)
    wq, wk = (rng.uniform(0.9, 1.1, hd).astype(np.float32) for _ in range(2))
    for step in range(3):
        q, k, v = (rng.standard_normal((len(tails), d)).astype(np.float32) for d in (qd, kvd, kvd))
        out = torch.full((len(tails), qd), float("nan"), device="cuda")
        rv.decode_step_shared(p, 0, prefix, t, 0, dev(q), dev(k), dev(v), dev(wq), dev(wk), EPS, THETA, scale_of(hd),
                              out)
        got = host(out)
        for i, kv in enumerate(single):
            pos = prefix + tails[i] + step
            one = torch.full((qd,), float("nan"), device="cuda")
            rv.decode_step(kv, 0, dev(q[i]), dev(k[i]), dev(v[i]), dev(wq), dev(wk), EPS, THETA, pos, scale_of(hd), one)
            kk, vv = (host(x) for x in kv.read_rows(0, 0, pos + 1))
            for whole, first, mine in zip((kk, vv), p.read_rows(0, 0, prefix), t.read_rows(i, 0, tails[i] + step + 1)):
                assert np.array_equal(whole, np.concatenate([host(first), host(mine)]))
            h = q[i].astype(np.float64).reshape(-1, hd)
            y = h / np.sqrt((h * h).mean(-1, keepdims=True) + EPS) * wq
            ang = pos * np.power(THETA, -2.0 * np.arange(hd // 2) / hd)
            c, s = np.cos(ang), np.sin(ang)
            y = np.concatenate([y[:, :64] * c - y[:, 64:] * s, y[:, :64] * s + y[:, 64:] * c], 1)
            want, a = attend(y.reshape(-1), kk, vv, n_kv, hd, scale_of(hd))
            # (2 a: the query's own five f32 roundings)
            check(got[i], want, 2 * a, np.abs(vv).max(), f"shared step {step} sequence {i}")
            bound = 2 * np.abs(vv).max() * (2 * (np.log(2.0) * 37 * EPS32 * a + 2.0 ** -22) + 96 * EPS32)
            assert np.abs(got[i].astype(np.float64) - host(one)).max() <= bound, (step, i)


def test_one_prefix_for_the_batches_of_two_threads(monkeypatch):
    """Each thread on a stream of its own: the other's call waits where it would
    bind the prefix to its stream between this one's binding and its call."""
    import threading

    from ramvamp_amd import attention as A

    torch = torch_cuda()
    say("case shared two threads")
    rng = np.random.default_rng(50)
    n_kv, group, hd, prefix = 2, 8, 128, 500
    p = rv.KvCache(1, n_kv, hd, prefix, "f16")
    pk, pv = rows(rng, prefix, n_kv * hd), rows(rng, prefix, n_kv * hd)
    p.append_rows(0, dev(pk), dev(pv))
    torch.cuda.synchronize()
    flags, entered, done, failed = A._flags, threading.Event(), threading.Event(), []

    def batch_of(seqs, seed):
        g = np.random.default_rng(seed)
        t = rv.KvCache(seqs, n_kv, hd, 8, "f16")
        own = [(rows(g, 3, n_kv * hd), rows(g, 3, n_kv * hd)) for _ in range(seqs)]
        for i, (k, v) in enumerate(own):
            t.append_rows(i, dev(k), dev(v))
        q = g.standard_normal((seqs, n_kv * group * hd)).astype(np.float32)
        want = expect(q, (stored(pk, "f16"), stored(pv, "f16")),
                      [(stored(k, "f16"), stored(v, "f16")) for k, v in own], n_kv, hd)
        return t, q, want

    def call(batch):
        t, q, _ = batch
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            d = torch.from_numpy(q).cuda()
            out = torch.full_like(d, float("nan"))
            rv.decode_attention_shared(d, p, 0, prefix, t, 0, scale_of(hd), out)
            s.synchronize()
            return out.cpu().numpy()

    first, second = batch_of(5, 1), batch_of(9, 2)
    torch.cuda.synchronize()
    got = {}

    def other():
        try:
            entered.wait(30)
            got["second"] = call(second)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
        done.set()

    def between(cache, args):
        r = flags(cache, args)
        if cache is first[0]:
            entered.set()
            done.wait(0.5)
        return r

    monkeypatch.setattr(A, "_flags", between)
    th = threading.Thread(target=other)
    th.start()
    got["first"] = call(first)
    th.join(30)
    assert not failed and not th.is_alive()
    for name, b in (("first", first), ("second", second)):
        want, a, vmax = b[2]
        check(got[name], want, a, vmax, name)
