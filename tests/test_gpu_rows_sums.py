"""What the row attention's sums keep of scores so large that their last bits
weigh. Scores are exact here: a query has one or two nonzero values, and SCALE
times log2 e is one in f32, so that a weight is 2^score."""
import numpy as np
import pytest

import ramvamp_amd as rv
from gpu_util import dev, host, say, torch_cuda
from rows_util import LOG2E, check, stored

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(np.log(2.0)))
assert np.float32(SCALE) * np.float32(LOG2E) == np.float32(1)


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
