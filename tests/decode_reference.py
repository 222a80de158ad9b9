"""Plain numpy forms, in 64 bits, of the decoder operators (include/wkf_decode.h), and how far a kernel that keeps its
sums in f32 and rounds its result once may be from them.

U is the relative error of one rounding, half a step: 2^-24 for f32, 2^-11 for f16."""
import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -11
U = {np.dtype(np.float32): U32, np.dtype(np.float16): U16}
TINY = {np.dtype(np.float32): 2.0 ** -149, np.dtype(np.float16): 2.0 ** -25}  # half a step of the subnormals, or more


def close(got, want, dtype, slack, what=""):
    """|got - want| <= the result's own rounding + `slack` (an array or a number), NaN and infinities in the same places."""
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN at {np.argwhere(np.isnan(got) != np.isnan(want))[:4].tolist()}"
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    u = U[np.dtype(dtype)]
    allowed = u * np.abs(want) + TINY[np.dtype(dtype)] + slack * np.ones(want.shape)
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)) - allowed, -1)
    at = np.unravel_index(int(off.argmax()), off.shape) if off.size else ()
    assert not off.size or off.max() <= 0, f"{what}: at {at} got {got[at]!r}, want {want[at]!r}, allowed {allowed[at]:.3g}"


# ---- 4-bit products ------------------------------------------------------------------------------

def q4_weights(rng, k, n, group, zeros, scale_dtype):
    groups = -(-k // group)
    codes = rng.integers(0, 16, (k, n)).astype(np.uint8)
    scales = (rng.uniform(0.5, 1.5, (groups, n)) * 0.02).astype(scale_dtype)
    z = rng.integers(0, 16, (groups, n)).astype(np.uint8) if zeros else None
    return codes, scales, z


def q4_dense(codes, scales, zeros, group):
    k = codes.shape[0]
    g = np.arange(k) // group
    z = 8.0 if zeros is None else zeros[g].astype(np.float64)
    return (codes.astype(np.float64) - z) * scales[g].astype(np.float64)


def q4_slack(x, w, rounded_weights=False):
    """What f32 sums of k products may lose: each of about k roundings is off by U32 of a partial sum that is at most a few
    times s = sqrt(sum (x w)^2), independently: 8 sqrt(k) U32 s is far out in that distribution, and the sums of codes before
    the scale are larger than the products by up to 16 / |code - zero| on average under 3 (3 * 8 = 24).  Products with many
    rows may round each weight to f16 first (U16 each, independent: 6 U16 s)."""
    x, w = np.abs(np.asarray(x, dtype=np.float64)), np.abs(w)
    s = np.sqrt(np.square(x) @ np.square(w))
    return s * (24 * np.sqrt(x.shape[-1]) * U32 + (6 * U16 if rounded_weights else 0))


# ---- norm and rotation ----------------------------------------------------------------------------

def norm_rope(x, weight, cos, sin, eps, positions):
    """x [batch, heads, seq, dim] (or rank 3); cos, sin [positions, dim / 2] or [positions, dim]."""
    four = x.ndim == 4
    x = np.asarray(x, dtype=np.float64)
    x = x if four else x[None]
    y = x / np.sqrt(np.mean(np.square(x), -1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    half = x.shape[-1] // 2
    out = np.empty_like(y)
    for b in range(x.shape[0]):
        rows = slice(positions[b], positions[b] + x.shape[2])
        c, s = (np.asarray(t, dtype=np.float64)[rows] for t in (cos, sin))
        if c.shape[1] == half:
            c, s = np.concatenate([c, c], -1), np.concatenate([s, s], -1)
        lo, hi = y[b, ..., :half], y[b, ..., half:]
        out[b] = np.concatenate([lo * c[:, :half] - hi * s[:, :half], hi * c[:, half:] + lo * s[:, half:]], -1)
    return out if four else out[0]


def norm_rope_slack(x, weight, eps):
    """The norm: dim / 2 + 8 roundings of a sum of squares (halved by the root), a division, three products and a sum:
    under (dim / 4 + 12) U32 of the larger of the two terms, each at most |y| of its half."""
    x = np.asarray(x, dtype=np.float64)
    y = np.abs(x / np.sqrt(np.mean(np.square(x), -1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64))
    half = x.shape[-1] // 2
    both = y[..., :half] + y[..., half:]
    return (x.shape[-1] / 4 + 12) * U32 * np.concatenate([both, both], -1)


# ---- the cache ---------------------------------------------------------------------------------------

def stored(x, block):
    """[tokens, dim] as the 8-bit cache holds it: codes and the scale of each block."""
    x = np.asarray(x, dtype=np.float64)
    codes, scales = np.zeros(x.shape), np.zeros(-(-x.shape[0] // block), dtype=np.float32)
    for i in range(scales.size):
        part = x[i * block:(i + 1) * block]
        finite = np.where(np.isfinite(part), np.abs(part), 0)
        scales[i] = np.float32(finite.max() if finite.size else 0) / np.float32(127)
        if scales[i] > 0:
            with np.errstate(invalid="ignore"):
                codes[i * block:(i + 1) * block] = np.nan_to_num(np.clip(np.rint(part / np.float64(scales[i])), -127, 127), nan=0.0)
    return codes, scales


def values(x, block):
    codes, scales = stored(x, block)
    return codes * scales.astype(np.float64)[np.arange(x.shape[0]) // block][:, None]


def attend(q, k, v, scale, causal, length, count):
    """One sequence: q [heads, S, dim], k and v [kv_heads, length, dim] as the cache holds them.  Returns the output and what a
    kernel may be off by."""
    q = np.asarray(q, dtype=np.float64)
    heads, rows, dim = q.shape
    out, slack = np.zeros(q.shape), np.zeros(q.shape)
    share = heads // max(1, k.shape[0])
    last = np.minimum(np.arange(count) + (length - count + 1 if causal else length), length)  # tokens a row sees
    seen = np.arange(length)[None, :] < last[:, None]
    for h in range(heads if count and length else 0):
        kk, vv = k[h // share], v[h // share]
        with np.errstate(invalid="ignore", over="ignore"):
            x = np.where(seen, q[h, :count] @ kk.T * scale, -np.inf)
            size = np.where(seen, np.abs(q[h, :count]) @ np.abs(kk).T * scale, 0)
            p = np.where(seen, np.exp(x - x.max(1, keepdims=True)), 0)
            total = p.sum(1, keepdims=True)
            out[h, :count] = p @ vv / total
            # a score: dim + 4 roundings of partial sums no larger than `size`, and the rounding of the exponent; a weight: that,
            # twice (the row's largest score too), its own rounding and two of the exponential; sums of n weights and n products.
            # What lies below 2^-126 of the largest weight is below f32's normals, and may count as zero: so may the parts
            # of a weight that is taken in three, so 3 2^-126 times the largest value, for each token.
            d = (dim + 4) * U32 * size.max(1) + 4 * U32 * np.maximum(1.0, np.abs(np.where(seen, x, 0)).max(1))
            slack[h, :count] = (2 * d + (last + 16) * U32)[:, None] * (p @ np.abs(vv)) / total * 2 + (3 * 2.0 ** -126 * last * np.abs(vv).max())[:, None]
    return out, slack


def f16_weights_slack(q, k, v, scale, causal, length, count):
    """What rounding each softmax weight to f16, before it meets the values, may add: U16 of every term, and for weights so
    small that they are subnormal at least 2^-37 of the largest (a kernel gives its largest weight 2^12 or more, the step of
    f16 subnormals is 2^-24, half of it 2^-25) times the largest value, for each token."""
    a, _ = attend(q, k, np.abs(v), scale, causal, length, count)
    return U16 * a + length * 2.0 ** -37 * (np.abs(v).max() if v.size else 0.0)


def two_part_weights_slack(q, k, v, scale, causal, length, count):
    """What softmax weights in two parts of f16 may add.  The first part is off by half a step, which f32 holds exactly; the second
    is that, off by half a step of its own: U16^2 = 4 U32 of the weight.  Below f16's normal numbers: as in f16_weights_slack."""
    a, _ = attend(q, k, np.abs(v), scale, causal, length, count)
    return U16 * U16 * a + length * 2.0 ** -37 * (np.abs(v).max() if v.size else 0.0)
