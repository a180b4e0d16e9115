"""What the tests of the Q8_0 cache and of shared-prefix decode share: the
format in numpy, attention in 64 bits, and the bounds its kernels are held to.

The format (a block of 32 values): the bits of quantize_row_q8_0 where its
scale times 127 stays inside f16, the largest such scale and saturated codes
beyond, a NaN scale for a block with an infinity or a NaN; a reader sees
f16(scale * code).
"""
import numpy as np

LOG2E = 1.4426950408889634
EPS32 = 2.0 ** -24  # half a step of f32, relative


def q8_blocks(x):
    """codes int8 [..., blocks, 32], scales f16 [..., blocks] of rows [..., n]."""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        finite = np.isfinite(b).all(-1)
        amax = np.where(finite, np.abs(b).max(-1), 0).astype(np.float32)
        d = (amax / np.float32(127)).astype(np.float32)
        d = np.where(d.astype(np.float16).astype(np.float32) > 515.5, np.float32(515.5), d).astype(np.float32)
        inv = np.where(d >= np.float32(2.0 ** -126), np.float32(1) / d, np.float32(0)).astype(np.float32)
        y = (b * inv[..., None]).astype(np.float32).astype(np.float64)
        codes = np.clip(np.sign(y) * np.floor(np.abs(y) + 0.5), -127, 127)
    codes = np.where(finite[..., None], codes, 0).astype(np.int8)
    scales = np.where(finite, d, np.float32(np.nan)).astype(np.float16)
    return codes, scales


def q8_values(x):
    """The values a reader of a Q8_0 cache sees, float32, x's shape."""
    codes, scales = q8_blocks(x)
    with np.errstate(all="ignore"):
        v = (codes.astype(np.float32) * scales.astype(np.float32)[..., None]).astype(np.float16)
    return v.astype(np.float32).reshape(np.shape(x))


def stored(x, elem):
    x = np.asarray(x, np.float32)
    if elem == "q8_0":
        return q8_values(x)
    return x.astype(np.float16).astype(np.float32) if elem == "f16" else x


def attend(q, k, v, n_kv, hd, scale):
    """One query row over the rows given, f64: (out [n_q * hd], A), A the largest
    sum_d |q'_d k_d| over heads and rows (q' = q * scale * log2 e): what a
    score's rounding errors are relative to."""
    q = np.asarray(q, np.float64).reshape(-1, hd)
    k = np.asarray(k, np.float64).reshape(-1, n_kv, hd)
    v = np.asarray(v, np.float64).reshape(-1, n_kv, hd)
    g = q.shape[0] // n_kv
    s = float(np.float32(scale))
    out, a = np.empty_like(q), 0.0
    with np.errstate(all="ignore"):
        for j in range(n_kv):
            qs = q[j * g:(j + 1) * g]
            x = qs @ k[:, j].T * s
            a = max(a, float(np.max(np.abs(qs) @ np.abs(k[:, j]).T)) * abs(s) * LOG2E)
            p = np.exp(x - x.max(-1, keepdims=True))
            out[j * g:(j + 1) * g] = (p / p.sum(-1, keepdims=True)) @ v[:, j]
    return out.reshape(-1), a


def check(got, want, a, vmax, what, single=False):
    """Holds f32 outputs to the kernels' arithmetic.

    Elementwise, worst case. A score, in log2 units, is off by at most A times:
    2^-24 for q's scaling, 2^-22 for its hi + lo split, and one rounding of
    2^-24 for each of at most 32 f32 additions on the way of a sum over a head's
    (padded) dims: 37 * 2^-24 A. A probability is then off by ln 2 times that,
    plus 2^-22 for the exponential's and the split's own. An output, a quotient
    of two sums of them, is off by twice that of the largest |v|, plus the sums'
    own roundings: at most 2 * 48 at 2^-24, since a sum is taken 16 rows at a
    time within a split and over few splits, its terms shrinking the further off
    the later partial is rescaled. In 2-norm the roundings, independent, add as
    squares: 2^-17 of the output's own norm where the outputs are not smaller
    than the values they average by more than 1/64.
    single: q and p carry one f16 rounding of 2^-12 each in place of the splits."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaNs differ"
    ok = ~np.isnan(want)
    got, want = got[ok], want[ok]
    if not got.size:
        return
    assert np.all(np.isfinite(got)), f"{what}: non-finite"
    score = a * (2.0 ** -12 + 33 * EPS32 if single else 37 * EPS32)
    prob = np.log(2.0) * score + (2.0 ** -12 if single else 0.0) + 2.0 ** -22
    bound = vmax * (2 * prob + 96 * EPS32)
    err = float(np.max(np.abs(got - want)))
    assert err <= bound, f"{what}: max |err| {err:.3e} > {bound:.3e}"
    norm, rms = float(np.linalg.norm(want)), float(np.sqrt(np.mean(want ** 2)))
    if rms * 64 >= vmax:
        rel = float(np.linalg.norm(got - want)) / norm
        lim = max(2.0 ** -17, 4 * EPS32 * a) if not single else 2.0 ** -7
        assert rel <= lim, f"{what}: 2-norm error {rel:.3e} > {lim:.3e}"
