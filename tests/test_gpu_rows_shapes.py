"""Every shape of the row attention's launches (narrow and wide items, whole and
split, folded by the launch or by a second one), forced by the tuning knobs, at
sizes where tiles, splits and column blocks end raggedly."""
import numpy as np
import pytest

import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from rows_util import attend, check, q8_values, stored

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(1.0) / np.sqrt(np.float32(128)))


def rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[:, 5::37] *= 6
    return x


@pytest.mark.parametrize("columns", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("mode", ["exact", "f16"])
@pytest.mark.parametrize("n_kv,group,n,start,split", [
    (1, 8, 70, 500, 0),     # 560 columns, ragged last block
    (2, 5, 53, 129, 1),     # a group that divides no block
    (1, 8, 33, 1300, 3),
    (2, 1, 300, 100, 2),
    (1, 40, 13, 260, 0),    # a row's heads over several blocks
    (1, 8, 2, 900, 8),
])
def test_chunk_shapes(columns, mode, n_kv, group, n, start, split):
    torch = torch_cuda()
    say(f"case chunk shape {(columns, mode, n_kv, group, n, start, split)}")
    rng = np.random.default_rng(n + start)
    k, v = rows(rng, start + n, n_kv * 128), rows(rng, start + n, n_kv * 128)
    kv = rv.KvCache(1, n_kv, 128, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    kv.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    kv.set_tuning(rv.RV_TUNE_PREFILL_KV_SPLIT, split)
    k, v = q8_values(k), q8_values(v)
    q = rng.standard_normal((n, n_kv * group * 128)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, SCALE, out, mode)
    got = host(out)
    look = sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n)))
    wants = [attend(q[r], k[:start + r + 1], v[:start + r + 1], n_kv, 128, SCALE) for r in look]
    check(got[look], np.stack([w for w, _ in wants]), max(a for _, a in wants), np.abs(v).max(), "chunk",
          single=mode != "exact")
    assert np.all(np.isfinite(got))
    again = torch.full(q.shape, float("nan"), device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, SCALE, again, mode)
    assert np.array_equal(host(again).view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("columns", [32, 64, 128, 256])
@pytest.mark.parametrize("split", [1, 4])
def test_nan_rows_in_every_shape(columns, split):
    torch = torch_cuda()
    say(f"case chunk NaN {(columns, split)}")
    rng = np.random.default_rng(columns)
    group, n, start = 8, 150, 200
    k, v = rows(rng, start + n, 128), rows(rng, start + n, 128)
    v[start + 37, 70] = np.nan     # block 2
    v[start + 90, 5] = np.inf      # block 0
    v[start + 91, 6] = -np.inf
    v[start + 128, 127] = np.nan   # block 3
    kv = rv.KvCache(1, 1, 128, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    kv.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    kv.set_tuning(rv.RV_TUNE_PREFILL_KV_SPLIT, split)
    ks, vs = q8_values(k), q8_values(v)
    q = rng.standard_normal((n, group * 128)).astype(np.float32)
    out = torch.full(q.shape, 0.0, device="cuda")
    rv.attention_at_rows(dev(q), kv, 0, start, SCALE, out)
    got = host(out).reshape(n, group, 4, 32)
    first = {2: 37, 0: 90, 3: 128, 1: n}
    for b, at in first.items():
        bad = np.isnan(got[:, :, b]).all(axis=(1, 2))
        assert np.array_equal(bad, np.arange(n) >= at), (b, at)
        assert np.isnan(got[:at, :, b]).sum() == 0
    clean = float(np.nanmax(np.abs(vs)))
    for r in (0, 36, 37, 89, 90, 127, 128, 149):
        want, a = attend(q[r], ks[:start + r + 1], vs[:start + r + 1], 1, 128, SCALE)
        want, g = want.reshape(group, 4, 32), got[r]
        ok = ~np.isnan(want)
        assert np.array_equal(~np.isnan(g), ok)
        check(g[ok], want[ok], a, clean, f"row {r}")


@pytest.mark.parametrize("columns", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("elem", ["q8_0", "f16", "f32"])
@pytest.mark.parametrize("n_kv,group,prefix,seqs,longest,split_len", [
    (1, 8, 700, 9, 200, 0),
    (2, 8, 130, 33, 31, 128),
    (1, 5, 2049, 13, 1, 512),
    (1, 12, 257, 40, 140, 0),
    (1, 24, 300, 4, 60, 0),
])
def test_shared_shapes(columns, elem, n_kv, group, prefix, seqs, longest, split_len):
    torch = torch_cuda()
    say(f"case shared shape {(columns, elem, n_kv, group, prefix, seqs, longest, split_len)}")
    rng = np.random.default_rng(prefix)
    kvd = n_kv * 128
    p = rv.KvCache(1, n_kv, 128, prefix + 1, elem)
    pk, pv = rows(rng, prefix, kvd), rows(rng, prefix, kvd)
    p.append_rows(0, dev(pk), dev(pv))
    bad = np.full((1, kvd), np.nan, np.float32)
    p.append_rows(0, dev(bad), dev(bad))
    lens = [(i * 7919) % (longest + 1) for i in range(seqs)]
    lens[-1] = longest
    t = rv.KvCache(seqs, n_kv, 128, longest + 5, elem)
    own = []
    for i, n in enumerate(lens):
        k, v = rows(rng, n, kvd), rows(rng, n, kvd)
        if n:
            t.append_rows(i, dev(k), dev(v))
        t.append_rows(i, dev(bad), dev(bad))  # written over later: stale, not attended
        t.truncate_layer(i, n)
        own.append((stored(k, elem) if n else k, stored(v, elem) if n else v))
    t.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
    t.set_tuning(rv.RV_TUNE_DECODE_SPLIT_LEN, split_len)
    q = rng.standard_normal((seqs, n_kv * group * 128)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, prefix, t, 0, SCALE, out)
    got = host(out)
    pk, pv = stored(pk, elem), stored(pv, elem)
    look = sorted({0, 1, seqs // 2, seqs - 1})
    outs, a, vmax = [], 0.0, 0.0
    for i in look:
        k, v = np.concatenate([pk, own[i][0]]), np.concatenate([pv, own[i][1]])
        w, ai = attend(q[i], k, v, n_kv, 128, SCALE)
        outs.append(w)
        a, vmax = max(a, ai), max(vmax, float(np.abs(v).max()))
    check(got[look], np.stack(outs), a, vmax, "shared")
    assert np.all(np.isfinite(got))
    again = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), p, 0, prefix, t, 0, SCALE, again)
    assert np.array_equal(host(again).view(np.uint32), got.view(np.uint32))


@pytest.mark.parametrize("n", [129, 1000, 2048, 2049, 4097, 9000])
def test_decode_split_counts(n):
    """Whole, folded in the launch and by a second one, and the same bits whichever
    call came before (the fold's tickets and workspace are left as they were)."""
    torch = torch_cuda()
    say(f"case decode splits {n}")
    rng = np.random.default_rng(n)
    n_kv, group = 2, 8
    k, v = rows(rng, n, n_kv * 128), rows(rng, n, n_kv * 128)
    kv = rv.KvCache(1, n_kv, 128, n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    k, v = q8_values(k), q8_values(v)
    q = rng.standard_normal(n_kv * group * 128).astype(np.float32)
    bits = {}
    for round_ in range(2):
        for limit in (n, n // 2, 100, n - 1):
            out = torch.full((q.size,), float("nan"), device="cuda")
            rv.attention_at(dev(q), kv, 0, limit, SCALE, None, out)
            got = host(out)
            if round_ == 0:
                want, a = attend(q, k[:limit], v[:limit], n_kv, 128, SCALE)
                check(got, want, a, np.abs(v).max(), f"limit {limit}")
                bits[limit] = got.view(np.uint32).copy()
            assert np.array_equal(got.view(np.uint32), bits[limit])


def test_a_large_chunk_and_a_large_batch():
    """The automatic shapes of large calls: a chunk of 1100 rows behind 2500, 64
    sequences of ragged rows behind 5000."""
    torch = torch_cuda()
    say("case large")
    rng = np.random.default_rng(17)
    n_kv, group, n, start = 2, 8, 1100, 2500
    k, v = rows(rng, start + n, n_kv * 128), rows(rng, start + n, n_kv * 128)
    kv = rv.KvCache(1, n_kv, 128, start + n, "q8_0")
    kv.append_rows(0, dev(k), dev(v))
    ks, vs = q8_values(k), q8_values(v)
    q = rng.standard_normal((n, n_kv * group * 128)).astype(np.float32)
    for mode in ("exact", "bf16"):
        out = torch.full(q.shape, float("nan"), device="cuda")
        rv.attention_at_rows(dev(q), kv, 0, start, SCALE, out, mode)
        got = host(out)
        assert np.all(np.isfinite(got))
        look = [0, 17, 512, 1023, 1099]
        wants = [attend(q[r], ks[:start + r + 1], vs[:start + r + 1], n_kv, 128, SCALE) for r in look]
        check(got[look], np.stack([w for w, _ in wants]), max(a for _, a in wants), np.abs(vs).max(), mode,
              single=mode != "exact")
    kv16 = rv.KvCache(1, n_kv, 128, 3600, "f16")
    kv16.append_rows(0, dev(k), dev(v))
    k16, v16 = stored(k, "f16"), stored(v, "f16")
    lens = [(i * 97) % 411 for i in range(64)]
    t = rv.KvCache(64, n_kv, 128, 411, "f16")
    for i, m in enumerate(lens):
        if m:
            t.append_rows(i, dev(k[:m]), dev(v[:m]))
    q = rng.standard_normal((64, n_kv * group * 128)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    rv.decode_attention_shared(dev(q), kv16, 0, 3600, t, 0, SCALE, out)
    got = host(out)
    look = [0, 1, 31, 63]
    wants = [attend(q[i], np.concatenate([k16, k16[:lens[i]]]), np.concatenate([v16, v16[:lens[i]]]), n_kv, 128, SCALE)
             for i in look]
    check(got[look], np.stack([w for w, _ in wants]), max(a for _, a in wants), np.abs(v16).max(), "batch")
    assert np.all(np.isfinite(got))


@pytest.mark.parametrize("elem,row_bytes", [("q8_0", 128), ("f16", 256), ("f32", 512)])
def test_planes_past_4_gib(elem, row_bytes):
    """A layer whose rows pass 2^32 bytes: rows of zeros (score 0, value 0), but
    some thousand around that offset, which carry all but 2^-15 of the weight."""
    torch = torch_cuda()
    say(f"case past 4 GiB {elem}")
    rng = np.random.default_rng(row_bytes)
    mark, group, d = (1 << 32) // row_bytes, 2, 128
    lo, n = mark - 2500, mark + 1777
    kv = rv.KvCache(2, 1, d, n, elem)
    zeros = torch.zeros(1 << 20, d, device="cuda")
    for at in range(0, lo, 1 << 20):
        z = zeros[:min(1 << 20, lo - at)]
        kv.append_rows(1, z, z)
    k, v = rows(rng, n - lo, d), rows(rng, n - lo, d)
    kv.append_rows(1, dev(k), dev(v))
    got_k, got_v = kv.read_rows(1, n - 9, 9)
    ks, vs = stored(k, elem), stored(v, elem)
    assert np.array_equal(host(got_k), ks[-9:]) and np.array_equal(host(got_v), vs[-9:])
    q = (8 * rng.standard_normal((3 if elem == "q8_0" else 20, group * d))).astype(np.float32)

    def want(i, count):  # over the zero rows too, each a term of e^0 below
        x = q[i].reshape(group, d).astype(np.float64) @ ks[:count].astype(np.float64).T * SCALE
        p = np.exp(x - x.max(-1, keepdims=True))
        below = p.sum(-1, keepdims=True) + lo * np.exp(-x.max(-1, keepdims=True))
        a = np.abs(q[i].reshape(group, d)).astype(np.float64) @ np.abs(ks[:count]).T.astype(np.float64)
        assert (lo * np.exp(-x.max(-1)) / below[:, 0]).max() < 2.0 ** -15
        return (p / below @ vs[:count].astype(np.float64)).reshape(-1), a.max() * SCALE * 1.4426950408889634

    vmax = np.abs(vs).max()
    out = torch.full(q.shape, float("nan"), device="cuda")
    if elem == "q8_0":
        rv.decode_attention(dev(q[0]), kv, 1, SCALE, None, out[0])
        w, a = want(0, n - lo)
        check(host(out[0]), w, a, vmax, "decode")
        rv.attention_at_rows(dev(q), kv, 1, n - 3, SCALE, out)
        for i in range(3):
            w, a = want(i, n - lo - 2 + i)
            check(host(out[i]), w, a, vmax, f"chunk row {i}")
    else:
        tails = rv.KvCache(20, 1, d, 1, elem)
        for columns in (32, 128):
            tails.set_tuning(rv.RV_TUNE_ROWS_COLUMNS, columns)
            rv.decode_attention_shared(dev(q), kv, 1, n, tails, 0, SCALE, out)
            for i in (0, 11, 19):
                w, a = want(i, n - lo)
                check(host(out[i]), w, a, vmax, f"sequence {i}")
