"""What the row attention's sums keep: many small weights behind one that towers
over them, scores so large that their last bits weigh, and a kv head's splits in a
call of its range alone. Scores of the first two are exact: a query has one or two
nonzero values, and SCALE times log2 e is one in f32, so that a weight is 2^score."""
import numpy as np
import pytest

import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from rows_util import EPS32, LOG2E, attend, check, stored

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(np.log(2.0)))
assert np.float32(SCALE) * np.float32(LOG2E) == np.float32(1)


def one_hot(n, heads, hd):
    q = np.zeros((n, heads, hd), np.float32)
    q[:, :, 0] = 1
    return q.reshape(n, heads * hd)


def sink_rows(n, hd, sink, below, elem):
    """One key that scores 0 with value -1, the others ``below`` under it with value
    1 (or what a block holds of them: the values a reader sees come back)."""
    k, v = np.zeros((n, hd), np.float32), np.ones((n, hd), np.float32)
    k[:, 0] = -below
    k[sink, 0] = 0
    v[sink] = -1
    return k, v, stored(k[[sink, sink - 1 if sink else 1]], elem), stored(v[[sink, sink - 1 if sink else 1]], elem)


def sink_output(n, ks, vs):
    w = 2.0 ** float(ks[1, 0])
    return (float(vs[0, 0]) + (n - 1) * w * float(vs[1, 0])) / (1 + (n - 1) * w)


def sink_bound(rows, below):
    """Worst case. The terms of a sum, 16 rows or more each, are either kept or, where
    they are below 2^-24 of it, lost whole: 2^-below a row, at most 2^-28, of the
    rows that one sum takes in before it is put aside. That is of the values' sum
    and of the weights', the values are within 1. The rest is rows_util's: the
    exponentials' 2^-22 twice and 96 roundings."""
    return 2 * rows * min(2.0 ** -below, 2.0 ** -28) + 2 * 2.0 ** -22 + 96 * EPS32


@pytest.mark.parametrize("below", [20, 28, 30, 31, 32])
@pytest.mark.parametrize("sink", [0, 60001])
@pytest.mark.parametrize("columns", [32, 64, 128, 256])
def test_many_small_weights_in_a_chunk(columns, sink, below):
    torch = torch_cuda()
    say(f"case chunk sink {(columns, sink, below)}")
    n, start, heads = 40, 100000, 8
    k, v, ks, vs = sink_rows(start + n, 128, sink, below, "q8_0")
    kv = rv.KvCache(1, 1, 128, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    kv.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    kv.set_tuning(rv.RV_TUNE_PREFILL_KV_SPLIT, 1)
    q = one_hot(n, heads, 128)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, SCALE, out)
    got = host(out).astype(np.float64)
    want = np.array([[sink_output(start + r + 1, ks, vs)] for r in range(n)])
    err = np.abs(got - want).max()
    assert err <= sink_bound(8192 if columns > 32 else 1024, below), err


@pytest.mark.parametrize("below", [20, 28, 31])
@pytest.mark.parametrize("columns", [32, 64, 128, 256])
@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_many_small_weights_in_a_batch(elem, columns, below):
    torch = torch_cuda()
    say(f"case shared sink {(elem, columns, below)}")
    seqs, n, heads = 40, 90000, 8
    k, v, ks, vs = sink_rows(n, 128, 1, below, elem)
    p, t = rv.KvCache(1, 1, 128, n, elem), rv.KvCache(seqs, 1, 128, 1, elem)
    p.append_rows(0, dev(k), dev(v))
    t.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    t.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 1 << 20)
    q = one_hot(seqs, heads, 128)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, n, t, 0, SCALE, out)
    err = np.abs(host(out).astype(np.float64) - sink_output(n, ks, vs)).max()
    assert err <= sink_bound(1024 if columns == 32 else 8192, below), err


@pytest.mark.parametrize("below", [24, 28, 31])
@pytest.mark.parametrize("elem", ["f16", "f32", "q8_0"])
def test_many_small_weights_in_a_tail(elem, below):
    """A long sequence of its own behind a short prefix (few columns, cut short)."""
    torch = torch_cuda()
    say(f"case tail sink {(elem, below)}")
    n, heads = 70000, 8
    k, v, ks, vs = sink_rows(n, 128, 5, below, elem)
    p, t = rv.KvCache(1, 1, 128, 1, elem), rv.KvCache(2, 1, 128, n, elem)
    t.append_rows(0, dev(k), dev(v))
    t.append_rows(1, dev(k[:9]), dev(v[:9]))
    q = one_hot(2, heads, 128)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, 0, t, 0, SCALE, out)
    got = host(out).astype(np.float64)
    for row, m in ((0, n), (1, 9)):
        err = np.abs(got[row] - sink_output(m, ks, vs)).max()
        assert err <= sink_bound(1024, below), (row, err)


@pytest.mark.parametrize("below", [20, 28, 31])
@pytest.mark.parametrize("hd", [128, 64])
def test_many_small_weights_of_one_token(hd, below):
    torch = torch_cuda()
    say(f"case decode sink {(hd, below)}")
    n, heads = 100000, 8
    k, v, ks, vs = sink_rows(n, hd, 3, below, "q8_0")
    kv = rv.KvCache(1, 1, hd, n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    kv.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 1 << 20)
    out = torch.full((heads * hd,), float("nan"), device="cuda")
    rv.decode_attention(dev(one_hot(1, heads, hd)[0]), kv, 0, SCALE, None, out)
    err = np.abs(host(out).astype(np.float64) - sink_output(n, ks, vs)).max()
    assert err <= sink_bound(1024, below), err


@pytest.mark.parametrize("columns", [32, 64, 128, 256])
@pytest.mark.parametrize("nan", [False, True])
@pytest.mark.parametrize("n,start", [(40, 8192 - 20), (40, 3 * 4096 - 17), (70, 2 * 8192 - 40), (33, 4096 - 33)])
def test_columns_that_end_where_sums_are_put_aside(n, start, nan, columns):
    """A chunk in one split, some of whose rows see a few positions past the end of
    a sum and some do not; with a block of NaNs that all see."""
    torch = torch_cuda()
    say(f"case sums put aside {(n, start, nan, columns)}")
    rng = np.random.default_rng(n + start)
    heads = 8
    k, v = (rng.standard_normal((start + n, 128)).astype(np.float32) for _ in range(2))
    if nan:
        v[1000, 70] = np.nan  # block 2
    kv = rv.KvCache(1, 1, 128, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    kv.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    kv.set_tuning(rv.RV_TUNE_PREFILL_KV_SPLIT, 1)
    k, v = stored(k, "q8_0"), stored(v, "q8_0")
    q = (2 * rng.standard_normal((n, heads * 128))).astype(np.float32)
    scale = float(np.float32(128 ** -0.5))
    out = torch.full(q.shape, 0.0, device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, scale, out)
    got = host(out)
    wants = [attend(q[r], k[:start + r + 1], v[:start + r + 1], 1, 128, scale) for r in range(n)]
    want = np.stack([w for w, _ in wants])
    assert np.isnan(want).any() == nan
    check(got, want, max(a for _, a in wants), np.nanmax(np.abs(v)), "chunk")
    ok = ~np.isnan(want)
    a = max(a for _, a in wants)
    rows = 8192 if columns > 32 else 1024
    # four products' roundings and one of the weights' sum for 32 rows, and the joining's
    lim = 2 * np.log(2.0) * 37 * EPS32 * a + 2 * 2.0 ** -22 + (5 * rows / 32 + 32) * EPS32
    terms = np.concatenate([attend(q[r], k[:start + r + 1], np.abs(v[:start + r + 1]), 1, 128, scale)[0] for r in range(n)])
    assert np.all(np.abs(got - want)[ok] <= lim * terms.reshape(want.shape)[ok])


@pytest.mark.parametrize("columns", [32, 128, 256])
@pytest.mark.parametrize("case", ["1e37", "later_larger", "later_smaller", "one_large"])
def test_f32_values_of_any_range_in_long_sums(case, columns):
    """Each sum put aside has a range of its own."""
    torch = torch_cuda()
    say(f"case f32 range in long sums {(case, columns)}")
    rng = np.random.default_rng(len(case))
    seqs, heads, n = 40, 8, 20000
    k, v = (rng.standard_normal((n, 128)) for _ in range(2))
    at = np.arange(n)[:, None]
    v *= {"1e37": 1e37, "later_larger": np.where(at < 9000, 1e-12, 1e25),
          "later_smaller": np.where(at < 9000, 1e30, 1e-6), "one_large": np.where(at == 12345, 1e36, 1.0)}[case]
    k, v = k.astype(np.float32), v.astype(np.float32)
    p, t = rv.KvCache(1, 1, 128, n, "f32"), rv.KvCache(seqs, 1, 128, 1, "f32")
    p.append_rows(0, dev(k), dev(v))
    t.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    t.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 1 << 20)
    q = rng.standard_normal((seqs, heads * 128)).astype(np.float32)
    scale = float(np.float32(128 ** -0.5))
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, n, t, 0, scale, out)
    got = host(out).astype(np.float64)
    assert np.all(np.isfinite(got))
    rows = 8192 if columns > 32 else 1024
    for i in (0, 1, 20, seqs - 1):
        want, a = attend(q[i], k, v, 1, 128, scale)
        terms, _ = attend(q[i], k, np.abs(v), 1, 128, scale)
        q1 = np.abs(q[i].reshape(-1, 128).astype(np.float64)).sum(-1).max() * scale * LOG2E
        score = 37 * EPS32 * a + 2.0 ** -34 * q1 * np.abs(k).max()
        # six products' roundings for 32 rows, and those of the sums' joining
        bound = terms * (2 * (np.log(2.0) * score + 2.0 ** -22) + 2.0 ** -22 + 2 * (6 * rows / 32 + 32) * EPS32)
        bound += 2.0 ** -34 * float(np.abs(v).max())
        err = np.abs(got[i] - want)
        assert np.all(err <= bound), (i, float(np.max(err / bound)))


# (the first key's score, a power of two and the rest: what f16 holds of each)
LARGE = [(2.0 ** 10, 248), (2.0 ** 11, 504), (2.0 ** 12, 1008)]


def large_rows(rng, base, rest, step, sign, elem, n=300):
    """Two keys whose scores are sign * (base * 2^15 + rest) and ``step`` more, the
    larger one four tiles later, so that one wave meets both; the others score far
    below."""
    k, v = np.zeros((n, 128), np.float32), rng.standard_normal((n, 128)).astype(np.float32)
    k[:, 0] = 0 if sign > 0 else -2.0 ** 14
    for row, r in ((0, rest), (128, rest + sign * step)):
        k[row, 0], k[row, 40] = sign * base, sign * r
    ks, vs = stored(k, elem), stored(v, elem)
    assert np.array_equal(ks[[0, 128]], k[[0, 128]])
    w = 2.0 ** -float(step)
    return k, v, (w * vs[0].astype(np.float64) + vs[128]) / (1 + w), np.abs(vs).max()


def large_query(n, heads):
    q = np.zeros((n, heads, 128), np.float32)
    q[:, :, 0], q[:, :, 40] = 2.0 ** 15, 1
    return q.reshape(n, heads * 128)


@pytest.mark.parametrize("columns", [32, 64, 128, 256])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("base,rest", LARGE)
def test_scores_whose_last_bits_weigh(base, rest, sign, columns):
    """At 2^25 .. 2^27 (in log2 units) a score's last bit is 4 .. 16: differences of
    that size are exact and have to stay so."""
    torch = torch_cuda()
    say(f"case large scores {(base, rest, sign, columns)}")
    rng = np.random.default_rng(int(base))
    heads, n = 8, 40
    last = int(base) // 256  # a score's last bit
    for step in (last, 8, 16, 24, 48):
        if step % last or (rest + sign * step) % last:
            continue
        for elem in ("q8_0", "f16", "f32"):
            k, v, want, vmax = large_rows(rng, base, rest, step, sign, elem)
            p, t = rv.KvCache(1, 1, 128, 300 + n, elem), rv.KvCache(n, 1, 128, 1, elem)
            p.append_rows(0, dev(k), dev(v))
            for c, split in ((t, rv.RV_TUNE_DECODE_SPLIT_LEN), (p, rv.RV_TUNE_DECODE_SPLIT_LEN)):
                c.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
                c.set_tuning(split, 1 << 20)
            q = large_query(n, heads)
            out = torch.full(q.shape, float("nan"), device="cuda")
            rv.decode_attention_shared(dev(q), p, 0, 300, t, 0, SCALE, out)
            check(host(out), np.tile(want, (n, heads)), 0.0, vmax, f"shared {elem} {step}")
            if elem != "q8_0":
                continue
            one = torch.full((heads * 128,), float("nan"), device="cuda")
            rv.decode_attention(dev(q[0]), p, 0, SCALE, None, one)
            check(host(one), np.tile(want, heads), 0.0, vmax, f"decode {step}")
            far = np.zeros((n, 128), np.float32)
            far[:, 0] = 0 if sign > 0 else -2.0 ** 14
            p.append_rows(0, dev(far), dev(far))
            p.set_tuning(rv.RV_TUNE_PREFILL_KV_SPLIT, 1)
            rv.attention_at_rows(dev(q), p, 0, 300, SCALE, out)
            check(host(out), np.tile(want, (n, heads)), 0.0, vmax, f"chunk {step}")


@pytest.mark.parametrize("columns", [32, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("base,rest,last", [(2.0 ** 10, 248, 4), (2.0 ** 12, 1008, 16), (2.0 ** 13, 2016, 32)])
def test_large_scores_and_large_values_meet_across_splits(base, rest, last, sign, columns):
    """The same two keys in two splits, the first one's values past 2^60: its partial
    is held in another form than the second one's."""
    torch = torch_cuda()
    say(f"case large scores, values and splits {(base, rest, sign, columns)}")
    rng = np.random.default_rng(int(base) + 1)
    heads, n = 8, 40
    k, v, _, _ = large_rows(rng, base, rest, last, sign, "f32")
    v[:128] *= np.float32(1e30)
    w = 2.0 ** -float(last)
    want = (w * v[0].astype(np.float64) + v[128]) / (1 + w)
    p, t = rv.KvCache(1, 1, 128, 300, "f32"), rv.KvCache(n, 1, 128, 1, "f32")
    p.append_rows(0, dev(k), dev(v))
    t.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    t.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, 128)
    q = large_query(n, heads)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, 300, t, 0, SCALE, out)
    check(host(out), np.tile(want, (n, heads)), 0.0, w * np.abs(v[0]).max(), "splits")


@pytest.mark.parametrize("n_kv,group,n", [(4, 8, 4097), (4, 8, 20000), (8, 4, 9000), (2, 40, 5000), (4, 20, 4500)])
def test_kv_ranges_join_to_the_whole_call_s_bits(n_kv, group, n):
    """A range's splits are the whole call's, so each head's sums are taken in the
    same order (as f16 and f32 caches have it)."""
    torch = torch_cuda()
    say(f"case q8 kv ranges {(n_kv, group, n)}")
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((n, n_kv * 128)).astype(np.float32) for _ in range(2))
    kv = rv.KvCache(1, n_kv, 128, n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    q = dev(rng.standard_normal(n_kv * group * 128))
    scale = float(np.float32(128 ** -0.5))
    whole = torch.full_like(q, float("nan"))
    rv.decode_attention(q, kv, 0, scale, None, whole)
    width = group * 128
    for units in (1, 2, n_kv):
        got = torch.full_like(q, float("nan"))
        for u in range(units):
            heads = range(u * n_kv // units, (u + 1) * n_kv // units)
            rv.decode_attention_kv_range_in(q, kv, 0, scale, heads, 1 << 40,
                                            got[heads.start * width:heads.stop * width])
        assert np.array_equal(host(got).view(np.uint32), host(whole).view(np.uint32)), units
    want, a = attend(host(q), stored(k, "q8_0"), stored(v, "q8_0"), n_kv, 128, scale)
    check(host(whole), want, a, np.abs(v).max() * 1.01, "whole")
