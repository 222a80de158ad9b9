"""The decoder operators on the GPU against their plain forms in 64 bits (tests/decode_reference.py): sizes and masks
where they can go wrong, strided inputs, both element types, and a run of them together."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import decode_reference as ref
from helpers import load_package

pytestmark = pytest.mark.gpu

F16, F32 = np.float16, np.float32
DTYPES = pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])


def leaf(dev, x):
    return load_package().Tensor.new(dev, x)


def computed(*tensors):
    """Values of lazy tensors; on a plan-only device their kernels are compiled and the test stops here."""
    if tensors[0].device.is_planner:
        for t in tensors:
            t.materialize()
        pytest.skip("plan-only device: kernels compiled, nothing computed")
    got = [t.to_numpy() for t in tensors]
    return got[0] if len(got) == 1 else got


def rng_of(*key):
    return np.random.default_rng([abs(hash(str(k))) % (1 << 31) if isinstance(k, str) else int(k) for k in key])


# ---- results that stay on the device ---------------------------------------------------------------

def test_materialize_into_writes_the_outputs(gpu):
    w, rng = load_package(), rng_of(1)
    x, y = rng.standard_normal((3, 70)).astype(F32), rng.standard_normal((3, 70)).astype(F32)
    a, b = leaf(gpu, x), leaf(gpu, y)
    out, swapped, col = w.Tensor.zeros(gpu, (3, 70)), w.Tensor.zeros(gpu, (70, 3)), w.Tensor.zeros(gpu, (3,))
    first = a + b
    w.materialize_into([first, first.transpose(0, 1), a.sum(1)], [out, swapped, col])
    # outputs that are leaves of the graphs: both sides are computed from what the leaves held before
    w.materialize_into([b, a * 2.0], [a, b])
    got = computed(out, swapped, col, a, b)
    assert np.array_equal(got[0], x + y) and np.array_equal(got[1], (x + y).T)
    ref.close(got[2], x.astype(np.float64).sum(1), F32, 70 * ref.U32 * np.abs(x).sum(1).astype(np.float64))
    assert np.array_equal(got[3], y) and np.array_equal(got[4], x * 2)


def test_materialize_into_swaps_leaves_and_views_of_them(gpu):
    w, rng = load_package(), rng_of(2)
    x, y = rng.standard_normal((5, 5)).astype(F16), rng.standard_normal((5, 5)).astype(F16)
    a, b = leaf(gpu, x), leaf(gpu, y)
    w.materialize_into([b, a], [a, b])
    w.materialize_into([a.transpose(0, 1)], [a])
    got = computed(a, b)
    assert np.array_equal(got[0], y.T) and np.array_equal(got[1], x)


def test_an_output_below_a_decoder_operator(gpu):
    """The output is a leaf of the operator's own graph: it is written after the operator has read it."""
    w, rng = load_package(), rng_of(3)
    x = rng.standard_normal((4, 6, 64)).astype(F32)
    tables = [rng.standard_normal((6, 32)).astype(F32) for _ in range(2)]
    g = rng.standard_normal(64).astype(F32)
    t, (c, s), gw = leaf(gpu, x), [leaf(gpu, v) for v in tables], leaf(gpu, g)
    w.materialize_into([t.norm_rope(gw, c, s, 1e-5)], [t])
    ref.close(computed(t), ref.norm_rope(x, g, *tables, 1e-5, [0]), F32, ref.norm_rope_slack(x, g, 1e-5))


# ---- products with 4-bit weights ---------------------------------------------------------------------

Q4_CASES = [  # m, k, n, group, zeros, scale dtype
    (1, 32, 16, 32, False, F16), (1, 1, 1, 32, True, F16), (3, 37, 5, 32, True, F32), (1, 4096, 64, 128, False, F16),
    (2, 130, 17, 64, True, F16), (16, 256, 48, 96, False, F32), (17, 384, 33, 128, True, F16), (5, 1000, 100, 1024, False, F16),
    (40, 512, 80, 64, True, F16), (65, 640, 130, 32, False, F16), (128, 256, 256, 128, True, F16), (300, 200, 264, 64, True, F32),
    (513, 1024, 272, 128, False, F16), (24, 200, 40, 64, False, F16), (20, 136, 4200, 32, True, F16), (33, 264, 48, 128, True, F32), (600, 96, 2000, 32, True, F16),
    (300, 160, 2000, 64, False, F16), (1100, 130, 2000, 128, True, F16), (800, 203, 144, 96, True, F32), (768, 64, 64, 32, False, F16), (7, 1290, 1037, 64, True, F16),
]


def q4_rounds_weights(dtype, m):
    """Products of this many f16 rows may round each weight to f16 (tests/decode_reference.py: q4_slack)."""
    return dtype == F16 and m >= 768


@DTYPES
@pytest.mark.parametrize("case", Q4_CASES, ids=lambda c: "x".join(str(v) if not isinstance(v, type) else v.__name__ for v in c))
def test_mat_mul_q4(gpu, case, dtype):
    w, (m, k, n, group, zeros, sdt) = load_package(), case
    rng = rng_of(10, m, k, n, group)
    codes, scales, z = ref.q4_weights(rng, k, n, group, zeros, sdt)
    x = rng.standard_normal((m, k)).astype(dtype)
    got = computed(leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, group)))
    dense = ref.q4_dense(codes, scales, z, group)
    assert got.dtype == dtype
    ref.close(got, x.astype(np.float64) @ dense, dtype, ref.q4_slack(x, dense, q4_rounds_weights(dtype, m)), str(case))


Q4_PATHS = [  # dtype, m, k, n, group, zeros, scale dtype, what the kernel's signature has
    (F16, 16, 200, 70, 32, True, F16, "q4_mat_mul|gfx950|f16|sf16|zeros|step1|w8|pf2|mt1"), (F16, 24, 264, 300, 64, False, F32, "|mt2"), (F32, 24, 264, 300, 64, False, F32, "|mt2"),
    (F16, 33, 296, 200, 128, True, F16, "|2x1x4x4"), (F16, 300, 160, 2000, 64, False, F16, "|2x2x4x4"), (F16, 600, 1031, 2000, 96, True, F32, "|4x2x4x2"),
    (F16, 1100, 130, 2000, 128, True, F16, "|4x2x8x1"), (F16, 600, 203, 7000, 32, True, F16, "|4x4x8x1"),
    (F16, 1100, 130, 7700, 128, True, F16, "q4_dense"), (F16, 800, 72, 11001, 32, False, F32, "q4_dense"),
    (F32, 33, 296, 200, 128, True, F16, "|2x1x4x2"), (F32, 300, 1031, 2000, 96, True, F32, "|2x1x8x2"), (F32, 600, 203, 2000, 64, False, F16, "|2x2x8x1"),
]


@pytest.mark.parametrize("case", Q4_PATHS, ids=lambda c: f"{c[0].__name__}-{c[1]}x{c[2]}x{c[3]}")
def test_mat_mul_q4_by_every_kernel(gpu, case):
    """A dense x and one whose rows start anywhere, a result of its own and one written where it is wanted, infinities and
    NaN that stay in their rows."""
    w, (dtype, m, k, n, group, zeros, sdt, kernel) = load_package(), case
    rng = rng_of(17, m, k, n, group)
    codes, scales, z = ref.q4_weights(rng, k, n, group, zeros, sdt)
    weights, dense = w.Q4Weights(gpu, codes, scales, z, group), ref.q4_dense(codes, scales, z, group)
    x = rng.standard_normal((m, k)).astype(dtype)
    odd = {1: np.nan, 5: np.inf, m - 1: -np.inf}
    for row, v in odd.items():
        x[row, row % k] = v
    flat = np.concatenate([np.zeros(3, dtype), x.reshape(-1)])
    first, second = leaf(gpu, x).mat_mul_q4(weights), leaf(gpu, flat).narrow(0, 3, m * k).reshape([m, k]).mat_mul_q4(weights)
    out = w.Tensor.zeros(gpu, (m, n), w.F16 if dtype == F16 else w.F32)
    first.materialize()
    assert any(kernel in i.signature for i in first.kernels()), [i.signature for i in first.kernels()]
    w.materialize_into([second], [out])
    got, placed = computed(first, out)
    finite = np.where(np.isfinite(x), x, 0).astype(np.float64)
    want = finite @ dense
    for row in odd:
        with np.errstate(invalid="ignore"):
            want[row] = (x[row].astype(np.float64)[:, None] * dense).sum(0)
    slack = ref.q4_slack(finite, dense, q4_rounds_weights(dtype, m))
    ref.close(got, want, dtype, slack)
    ref.close(placed, want, dtype, slack)


@DTYPES
def test_mat_mul_q4_of_views_batches_and_expressions(gpu, dtype):
    w, rng = load_package(), rng_of(11)
    codes, scales, z = ref.q4_weights(rng, 96, 40, 32, True, F16)
    weights, dense = w.Q4Weights(gpu, codes, scales, z, 32), ref.q4_dense(codes, scales, z, 32)
    x = rng.standard_normal((96, 7)).astype(dtype)
    big = rng.standard_normal((3, 5, 200)).astype(dtype)
    t, b = leaf(gpu, x), leaf(gpu, big)
    got = computed(t.transpose(0, 1).mat_mul_q4(weights), b.narrow(2, 51, 96).mat_mul_q4(weights), (t.transpose(0, 1) * 2.0).mat_mul_q4(weights) + 1.0,
                   b.narrow(2, 0, 96).narrow(0, 1, 1).narrow(1, 2, 1).mat_mul_q4(weights))
    for g, a in ((got[0], x.T), (got[1], big[..., 51:147]), (got[3], big[1:2, 2:3, :96])):
        ref.close(g, a.astype(np.float64) @ dense, dtype, ref.q4_slack(a, dense))
    twice = (x.T * dtype(2)).astype(np.float64)
    y = twice @ dense  # the product is rounded to dtype before 1 is added
    ref.close(got[2], y + 1, dtype, ref.q4_slack(twice, dense) + ref.U[np.dtype(dtype)] * np.abs(y))


def test_mat_mul_q4_keeps_infinities_and_nan_in_their_rows(gpu):
    w, rng = load_package(), rng_of(12)
    codes, scales, z = ref.q4_weights(rng, 64, 20, 32, False, F16)
    codes[codes == 8] = 9  # no weight is zero: infinity times a weight is infinity
    for dtype, m in ((F16, 6), (F32, 6), (F16, 70), (F32, 70), (F16, 800)):
        x = rng.standard_normal((m, 64)).astype(dtype)
        x[1, 3], x[3, 60], x[4, 0], x[4, 1] = np.inf, np.nan, np.inf, -np.inf
        dense = ref.q4_dense(codes, scales, z, 32)
        with np.errstate(invalid="ignore"):
            want = (x.astype(np.float64)[:, :, None] * dense).sum(1)
        finite = np.where(np.isfinite(x), x, 0)
        ref.close(computed(leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, 32))), want, dtype, ref.q4_slack(finite, dense, q4_rounds_weights(dtype, m)))


@DTYPES
def test_mat_mul_q4_of_rows_that_do_not_start_on_16_bytes(gpu, dtype):
    """A dense view whose first element is off the alignment that tiles are read with."""
    w, rng = load_package(), rng_of(14)
    codes, scales, z = ref.q4_weights(rng, 72, 40, 32, True, F16)
    weights, dense = w.Q4Weights(gpu, codes, scales, z, 32), ref.q4_dense(codes, scales, z, 32)
    for rows in (5, 50, 800):
        x = rng.standard_normal(rows * 72 + 3).astype(dtype)
        got = computed(leaf(gpu, x).narrow(0, 3, rows * 72).reshape([rows, 72]).mat_mul_q4(weights))
        ref.close(got, x[3:].reshape(rows, 72).astype(np.float64) @ dense, dtype, ref.q4_slack(x[3:].reshape(rows, 72), dense, q4_rounds_weights(dtype, rows)))


def test_mat_mul_q4_with_scales_that_are_not_finite(gpu):
    """An infinite or NaN scale stays in its column, and in the rows that it belongs to: zeros behind K do not meet it."""
    w, rng = load_package(), rng_of(15)
    codes, scales, z = ref.q4_weights(rng, 40, 20, 32, False, F16)
    codes[codes == 8] = 7
    scales[1, 3], scales[0, 5], scales[1, 19] = np.inf, np.nan, np.inf
    for dtype, m in ((F16, 6), (F32, 6), (F16, 40), (F32, 40)):
        x = np.abs(rng.standard_normal((m, 40))).astype(dtype) + dtype(0.5)
        codes[32:, 3] = 9  # one sign: the sum is an infinity, not a NaN
        codes[32:, 19] = 2
        dense = ref.q4_dense(codes, scales, z, 32)
        finite = np.where(np.isfinite(dense), dense, 0)
        with np.errstate(invalid="ignore"):
            want = (x.astype(np.float64)[:, :, None] * dense).sum(1)
        ref.close(computed(leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, 32))), want, dtype, ref.q4_slack(x, finite))


@pytest.mark.parametrize("scale", [2e4, 1e-7, 3e-5], ids=str)
def test_mat_mul_q4_of_weights_beyond_f16(gpu, scale):
    """Weights that f16 could not hold, or not with all its bits, meet many rows of f16."""
    w, rng = load_package(), rng_of(16)
    codes, scales, z = ref.q4_weights(rng, 96, 11008, 32, True, F32)
    scales = (scales * F32(scale / 0.02)).astype(F32)
    x = (rng.standard_normal((800, 96)) * min(1.0, 1e-3 / scale)).astype(F16)
    dense = ref.q4_dense(codes, scales, z, 32)
    y = leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, 32))
    y.materialize()
    assert not any("q4_dense" in i.signature for i in y.kernels())
    ref.close(computed(y), x.astype(np.float64) @ dense, F16, ref.q4_slack(x, dense))


Q4_LARGE = [(1, 200, 70, 32, True, "q4_mat_mul"), (7, 384, 40, 128, False, "q4_mat_mul"), (24, 200, 300, 64, True, "|mt2"), (33, 296, 200, 128, True, "|2x1x4x2"),
            (300, 330, 2000, 96, False, "|2x1x8x2"), (600, 203, 2000, 32, True, "|2x2x8x1")]


@pytest.mark.parametrize("case", Q4_LARGE, ids=lambda c: "x".join(str(v) for v in c[:4]))
def test_mat_mul_q4_of_the_largest_numbers(gpu, case):
    """Rows near f32's largest number and scales far below 1: x times codes leaves f32, the product with the weights does not.
    Rows of an ordinary size beside them, and one with an infinity, are what they are alone."""
    w, (m, k, n, group, zeros, kernel) = load_package(), case
    rng = rng_of(18, m, k, n, group)
    codes, scales, z = ref.q4_weights(rng, k, n, group, zeros, F32)
    scales = (scales * F32(2.0 ** -8)).astype(F32)
    x = rng.choice([-1.0, 1.0], (m, k)) * rng.uniform(0.5, 1, (m, k)) * 3.4e38
    x[2::3] /= 1e38
    x = x.astype(F32)
    if m > 1:
        x[1] = np.abs(x[1])  # every product of a column of one sign has it
        x[m - 1, 5] = np.inf
    dense = ref.q4_dense(codes, scales, z, group)
    y = leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, group))
    y.materialize()
    assert any(kernel in i.signature for i in y.kernels()), [i.signature for i in y.kernels()]
    finite = np.where(np.isfinite(x), x, 0).astype(np.float64)
    want = finite @ dense
    assert np.abs(want).max() < 3e38
    if m > 1:
        with np.errstate(invalid="ignore"):
            want[m - 1] = (x[m - 1].astype(np.float64)[:, None] * dense).sum(0)
    ref.close(computed(y), want, F32, ref.q4_slack(finite, dense), str(case))


def test_mat_mul_q4_of_a_square_matrix_and_rows_behind_the_first_element(gpu):
    """A copy of x has the product's shape here; the weights are written out."""
    w, rng = load_package(), rng_of(19)
    n, m = 6656, 1300
    codes, scales, z = ref.q4_weights(rng, n, n, 128, True, F16)
    flat = rng.standard_normal(m * n + 8).astype(F16)
    t, out = leaf(gpu, flat), w.Tensor.zeros(gpu, (m, n), w.F16)
    y = t.narrow(0, 8, m * n).reshape([m, n]).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, 128))
    w.materialize_into([y], [out])
    assert "q4_dense" in [i.kind for i in y.kernels()]
    got, alone, x = *computed(out, y), flat[8:].reshape(m, n)
    rows = np.r_[0:4, 700:704, m - 4:m]
    dense = ref.q4_dense(codes, scales, z, 128)
    ref.close(got[rows], x[rows].astype(np.float64) @ dense, F16, ref.q4_slack(x[rows], dense, True))
    assert np.array_equal(got, alone) and np.array_equal(computed(t), flat)


def test_mat_mul_q4_without_rows(gpu):
    w = load_package()
    codes, scales, z = ref.q4_weights(rng_of(13), 64, 20, 32, False, F16)
    x = leaf(gpu, np.zeros((0, 64), F16))
    assert computed(x.mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, 32))).shape == (0, 20)


# ---- the norm of a head and its rotation ----------------------------------------------------------------

@DTYPES
@pytest.mark.parametrize("shape", [(1, 1, 1, 2), (2, 3, 1, 128), (1, 4, 37, 64), (3, 5, 2, 80), (1, 2, 3, 6), (2, 1, 9, 256), (1, 3, 5, 1024), (70, 2, 1, 96), (300, 1, 1, 8)], ids=str)
def test_norm_rope(gpu, shape, dtype):
    rng = rng_of(20, *shape)
    x = (rng.standard_normal(shape) * 3).astype(dtype)
    batch, _, seq, dim = shape
    positions = [int(p) for p in rng.integers(0, 50, batch)]
    weight = (1 + 0.2 * rng.standard_normal(dim)).astype(dtype)
    got, want = [], []
    for width, table in ((dim // 2, F32), (dim, dtype)):
        angle = rng.uniform(-3, 3, (50 + seq, width))
        c, s = np.cos(angle).astype(table), np.sin(angle).astype(table)
        got.append(leaf(gpu, x).norm_rope(leaf(gpu, weight), leaf(gpu, c), leaf(gpu, s), 1e-5, positions))
        want.append(ref.norm_rope(x, weight, c, s, 1e-5, positions))
    for g, t in zip(computed(*got), want):
        assert g.dtype == dtype
        ref.close(g, t, dtype, ref.norm_rope_slack(x, weight, 1e-5))


@DTYPES
def test_norm_rope_of_a_projection_in_one_launch(gpu, dtype):
    """q and k are strided views of one projection [batch, seq, heads, dim]; both are computed by one kernel."""
    w, rng = load_package(), rng_of(21)
    batch, seq, heads, kv, dim = 3, 5, 8, 2, 72
    x = rng.standard_normal((batch, seq, heads + kv, dim)).astype(dtype)
    angle = rng.uniform(-3, 3, (40, dim // 2))
    c, s = np.cos(angle).astype(F32), np.sin(angle).astype(F32)
    gq, gk = (rng.uniform(0.5, 1.5, dim).astype(F32) for _ in range(2))
    positions = [7, 0, 35]
    t, tc, ts = leaf(gpu, x), leaf(gpu, c), leaf(gpu, s)
    views = [t.narrow(2, 0, heads).transpose(1, 2), t.narrow(2, heads, kv).transpose(1, 2)]
    nodes = [v.norm_rope(leaf(gpu, g), tc, ts, 1e-6, positions) for v, g in zip(views, (gq, gk))]
    outs = [w.Tensor.zeros(gpu, n.shape(), w.F16 if dtype == F16 else w.F32) for n in nodes]
    w.materialize_into(nodes, outs)
    assert [k.kind for k in nodes[0].kernels()] == ["norm_rope"]
    got = computed(*outs, *nodes)
    for i, (part, g) in enumerate(((x[:, :, :heads], gq), (x[:, :, heads:], gk))):
        part = part.transpose(0, 2, 1, 3)
        ref.close(got[i], ref.norm_rope(part, g, c, s, 1e-6, positions), dtype, ref.norm_rope_slack(part, g, 1e-6))
        assert np.array_equal(got[i], got[2 + i])  # alone: the same values


def test_norm_rope_of_a_norm_rope_beside_it(gpu):
    """A root that is computed from another one with the same tables is a launch of its own, after it."""
    w, rng = load_package(), rng_of(23)
    x = rng.standard_normal((2, 7, 64)).astype(F32)
    c, s = (rng.standard_normal((7, 32)).astype(F32) for _ in range(2))
    g = np.ones(64, F32)
    tg, tc, ts = (leaf(gpu, v) for v in (g, c, s))
    once = leaf(gpu, x).norm_rope(tg, tc, ts, 1e-5)
    twice = once.norm_rope(tg, tc, ts, 1e-5)
    outs = [w.Tensor.zeros(gpu, x.shape) for _ in range(2)]
    w.materialize_into([twice, once], outs)
    assert [k.kind for k in twice.kernels()] == ["norm_rope"] * 2
    got = computed(*outs)
    first = ref.norm_rope(x, g, c, s, 1e-5, [0])
    ref.close(got[1], first, F32, ref.norm_rope_slack(x, g, 1e-5))
    ref.close(got[0], ref.norm_rope(got[1], g, c, s, 1e-5, [0]), F32, ref.norm_rope_slack(got[1], g, 1e-5))


def test_norm_rope_of_columns_zeros_and_infinities(gpu):
    rng = rng_of(22)
    x = rng.standard_normal((2, 64, 6)).astype(F32)  # the last dimension of the view is not dense
    x[0, :, 1] = 0
    x[1, 5, 2], x[1, 7, 3] = np.nan, 1e30
    c, s = (rng.standard_normal((6, 32)).astype(F32) for _ in range(2))
    weight = np.ones(64, F32)
    got = computed(leaf(gpu, x).transpose(1, 2).norm_rope(leaf(gpu, weight), leaf(gpu, c), leaf(gpu, s), 1e-5))
    want = ref.norm_rope(x.transpose(0, 2, 1), weight, c, s, 1e-5, [0])
    rows = np.ones((2, 6), bool)
    rows[1, 3] = False  # 1e30 squared leaves f32: the norm is infinite and the row zero
    assert np.all(got[1, 3] == 0) and np.all(got[0, 1] == 0) and np.all(np.isnan(got[1, 2]))
    ref.close(got[rows], want[rows], F32, ref.norm_rope_slack(x.transpose(0, 2, 1), weight, 1e-5)[rows])


# ---- the cache ----------------------------------------------------------------------------------------------

def filled(gpu, rng, dtype, lengths, heads, dim, block, capacity=None, spread=True):
    """A cache and what it holds, per sequence [heads, length, dim] in 64 bits."""
    w = load_package()
    longest = max(1, max(lengths))
    k, v = (rng.standard_normal((len(lengths), heads, longest, dim)).astype(dtype) for _ in range(2))
    if spread:  # blocks of very different magnitudes
        k *= dtype(2) ** rng.integers(-1, 2, (len(lengths), heads, longest, 1)).astype(dtype)
        v *= (dtype(2) ** rng.integers(-8, 4, (len(lengths), heads, -(-longest // block), 1))).astype(dtype).repeat(block, 2)[:, :, :longest]
    cache = w.KvCache(gpu, len(lengths), heads, dim, capacity or longest, block)
    cache.append(leaf(gpu, k), leaf(gpu, v), lengths)
    held = [[np.stack([ref.values(x[b, h, :n], block) for h in range(heads)]) for x in (k, v)] for b, n in enumerate(lengths)]
    return cache, held, (k, v)


@DTYPES
@pytest.mark.parametrize("dim,block,lengths", [(64, 32, [1]), (128, 64, [64, 0, 65]), (80, 32, [31, 33, 100]), (1, 32, [5]), (256, 128, [300, 129]), (100, 128, [127]), (66, 64, [200])], ids=str)
def test_append_stores_what_the_definition_says(gpu, dim, block, lengths, dtype):
    cache, held, _ = filled(gpu, rng_of(30, dim, block, *lengths), dtype, lengths, 2, dim, block)
    n = max(lengths)
    got32, got16, tail = computed(cache.values(0, n), cache.values(0, n, load_package().F16), cache.values(n - 1, 1))
    for b, pair in enumerate(held):
        for i in range(2):
            want = np.zeros((2, n, dim))
            want[:, :lengths[b]] = pair[i]
            assert np.array_equal(got32[i, b], want.astype(F32)), (b, i)  # a code times a scale, rounded once: the same bits
            with np.errstate(over="ignore"):
                assert np.array_equal(got16[i, b], want.astype(F32).astype(F16)), (b, i)
            assert np.array_equal(tail[i, b], want[:, n - 1:].astype(F32))


@DTYPES
@pytest.mark.parametrize("dim", [1, 66, 80, 100, 128, 255])
def test_values_of_windows(gpu, dim, dtype):
    """Windows that start and end anywhere, over the ends of sequences, are cut from the whole."""
    w, rng = load_package(), rng_of(31, dim)
    cache, held, _ = filled(gpu, rng, dtype, [75, 0, 131], 3, dim, 32, capacity=140)
    windows = [(0, 140), (1, 1), (2, 5), (3, 70), (74, 2), (129, 9), (130, 1), (137, 3), (5, 0)]
    got = computed(*[cache.values(at, n, w.F16 if dtype == F16 else w.F32) for at, n in windows])
    want = np.zeros((2, 3, 3, 140, dim))
    for b in range(3):
        for kv in range(2):
            want[kv, b, :, :held[b][kv].shape[1]] = held[b][kv]
    for g, (at, n) in zip(got, windows):
        assert g.shape == (2, 3, 3, n, dim) and np.array_equal(g, want[:, :, :, at:at + n].astype(F32).astype(dtype))


@DTYPES
def test_append_in_pieces_gives_the_cache_of_one_append(gpu, dtype):
    """Tokens one at a time, in pieces that end inside a block, on its border and across several, by sequences of their own pace."""
    w, rng = load_package(), rng_of(31)
    heads, dim, block, total = 3, 72, 32, 203
    k, v = (rng.standard_normal((2, heads, total, dim)).astype(dtype) * dtype(3) for _ in range(2))
    whole, pieces = (w.KvCache(gpu, 2, heads, dim, 256, block) for _ in range(2))
    whole.append(leaf(gpu, k), leaf(gpu, v), [total, total - 10])
    at = [0, 0]
    for step in [(1, 1), (1, 0), (30, 31), (0, 1), (33, 64), (3, 65), (128, 1), (1, 0), (6, 30)]:
        n = max(step)
        kk, vv = (np.full((2, heads, n, dim), 7777, dtype) for _ in range(2))  # rows behind a count are not read as tokens
        for b in range(2):
            kk[b, :, :step[b]], vv[b, :, :step[b]] = k[b, :, at[b]:at[b] + step[b]], v[b, :, at[b]:at[b] + step[b]]
            at[b] += step[b]
        pieces.append(leaf(gpu, kk), leaf(gpu, vv), step)
    assert at == [total, total - 10] and pieces.lengths() == whole.lengths() == at
    a, b = computed(whole.values(), pieces.values())
    assert a.shape == (2, 2, heads, total, dim) and np.array_equal(a, b)


def test_append_of_special_values(gpu):
    """Zeros, infinities, NaN, subnormals, and quotients on the border of two codes."""
    w = load_package()
    x = np.zeros((1, 6, 64, 64), F32)
    x[0, 1, :32] = 1.0
    x[0, 1, 0, 0], x[0, 1, 1, 1], x[0, 1, 2, 2] = np.inf, -np.inf, np.nan
    x[0, 2, :, 0] = np.inf                                             # nothing finite but zeros
    x[0, 3] = (np.arange(64 * 64).reshape(64, 64) - 2000) * 2.0 ** -149  # subnormals
    x[0, 4] = (np.arange(64 * 64).reshape(64, 64) % 255 - 127) * 0.5    # halves of the scale: borders
    x[0, 4, 0, 0] = 127.0
    x[0, 4, 32, 0] = -127.0
    x[0, 5] = np.float32(3.4e38) * (np.arange(64 * 64).reshape(64, 64) % 3 - 1)
    cache = w.KvCache(gpu, 1, 6, 64, 64, 32)
    t = leaf(gpu, x)
    cache.append(t, t)
    got = computed(cache.values())
    for h in range(6):
        want = ref.values(x[0, h], 32).astype(F32)
        for i in range(2):
            if h == 3:  # scale = amax / 127 rounded to a subnormal: products of subnormals are exact in f32
                assert np.array_equal(got[i, 0, h], want), h
            else:
                assert np.array_equal(got[i, 0, h], want), h


def test_append_takes_views_and_expressions(gpu):
    w, rng = load_package(), rng_of(33)
    x = rng.standard_normal((2, 9, 6, 64)).astype(F16)  # [batch, tokens, k heads and v heads, dim]
    t = leaf(gpu, x)
    cache = w.KvCache(gpu, 2, 3, 64, 20, 32)
    cache.append(t.narrow(2, 0, 3).transpose(1, 2), t.narrow(2, 3, 3).transpose(1, 2) * 2.0)
    one = w.KvCache(gpu, 1, 3, 64, 20, 32)
    one.append(t.narrow(0, 1, 1).reshape([9, 6, 64]).transpose(0, 1).narrow(0, 0, 3), t.narrow(0, 1, 1).reshape([9, 6, 64]).transpose(0, 1).narrow(0, 3, 3))
    got, alone = computed(cache.values(), one.values())
    for b in range(2):
        for h in range(3):
            assert np.array_equal(got[0, b, h], ref.values(x[b, :, h], 32).astype(F32))
            assert np.array_equal(got[1, b, h], ref.values(x[b, :, 3 + h] * F16(2), 32).astype(F32))
            if b == 1:
                assert np.array_equal(alone[0, 0, h], got[0, b, h]) and np.array_equal(alone[1, 0, h] * 2, got[1, b, h])


def test_reset_forgets_one_sequence_or_all(gpu):
    w, rng = load_package(), rng_of(34)
    x = leaf(gpu, rng.standard_normal((2, 1, 40, 64)).astype(F32))
    cache = w.KvCache(gpu, 2, 1, 64, 64, 32)
    cache.append(x, x)
    before = cache.values(0, 40)
    cache.reset(0)
    assert cache.lengths() == [0, 40]
    with pytest.raises(w.WkfError, match="appended to or reset"):
        before.materialize()
    cache.append(x, x, [40, 0])
    again = cache.values(0, 40)
    first = computed(again)
    cache.reset()
    assert cache.lengths() == [0, 0]
    cache.append(x, x)
    assert np.array_equal(computed(cache.values(0, 40)), first)


# ---- attention over the cache ------------------------------------------------------------------------------------

def check_attend(gpu, dtype, lengths, heads, kv, dim, block, rows, causal=True, counts=None, scale=None, seed=0, **more):
    rng = rng_of(40, seed, dim, block, rows, *lengths)
    cache, held, _ = filled(gpu, rng, dtype, lengths, kv, dim, block, **more)
    q = rng.standard_normal((len(lengths), heads, rows, dim)).astype(dtype)
    counts = [min(rows, n) for n in lengths] if counts is None else counts
    scale = dim ** -0.5 if scale is None else scale
    got = computed(leaf(gpu, q).attend(cache, scale, causal, counts))
    assert got.dtype == dtype and got.shape == q.shape
    for b, n in enumerate(lengths):
        want, slack = ref.attend(q[b], *held[b], np.float32(scale).astype(np.float64), causal, n, counts[b])
        if dtype == F16:
            slack = slack + ref.f16_weights_slack(q[b], *held[b], np.float32(scale).astype(np.float64), causal, n, counts[b])
        ref.close(got[b], want, dtype, slack, f"sequence {b}")


ATTEND_CASES = [  # lengths, heads, kv heads, dim, block, rows
    ([1], 1, 1, 64, 32, 1), ([5, 0, 33], 4, 2, 128, 32, 1), ([1000], 32, 8, 128, 64, 1), ([31, 32, 65], 6, 6, 80, 32, 3),
    ([130, 7], 8, 1, 256, 128, 2), ([257], 3, 1, 20, 64, 1), ([64, 200, 0, 1], 24, 1, 96, 64, 1), ([700], 40, 1, 64, 128, 1),
    ([300], 4, 2, 64, 64, 300), ([190, 33], 6, 2, 128, 32, 40), ([129, 0, 128], 2, 1, 72, 128, 129), ([90], 16, 1, 192, 32, 17),
    ([500], 1, 1, 1, 32, 9), ([2100], 2, 1, 64, 32, 1), ([40, 77], 8, 2, 130, 64, 6),
]


@DTYPES
@pytest.mark.parametrize("case", ATTEND_CASES, ids=str)
def test_attend(gpu, case, dtype):
    lengths, heads, kv, dim, block, rows = case
    check_attend(gpu, dtype, lengths, heads, kv, dim, block, rows)


# enough tiles of 128 rows for every compute unit
PROMPT_CASES = [([150, 0, 129, 200], 32, 32, 64, 64, 129), ([100, 37, 300, 1, 128, 0], 48, 16, 72, 32, 100), ([141, 140, 0, 270, 64, 33], 32, 16, 128, 128, 140),
                ([70, 90, 0, 5, 65, 64, 71, 200], 32, 32, 200, 32, 70), ([260] * 4, 32, 32, 128, 64, 256), ([400, 260], 64, 64, 16, 32, 200)]


@DTYPES
@pytest.mark.parametrize("case", PROMPT_CASES, ids=str)
def test_attend_with_many_rows(gpu, case, dtype):
    lengths, heads, kv, dim, block, rows = case
    check_attend(gpu, dtype, lengths, heads, kv, dim, block, rows)


@DTYPES
def test_attend_with_many_rows_in_other_ways(gpu, dtype):
    check_attend(gpu, dtype, [150, 0, 190, 65], 64, 64, 64, 32, 70, causal=False)
    check_attend(gpu, dtype, [150, 0, 190, 65], 64, 64, 64, 32, 70, counts=[70, 0, 33, 1])
    check_attend(gpu, dtype, [150, 0, 190, 65], 128, 64, 64, 64, 100, counts=[64, 0, 100, 65], causal=False)
    for scale in (0.0, 4.0):
        check_attend(gpu, dtype, [150, 10, 190, 65], 64, 64, 64, 64, 70, scale=scale)


@DTYPES
@pytest.mark.parametrize("rows", [1, 3, 30, 70])
def test_attend_to_the_whole_sequence(gpu, rows, dtype):
    check_attend(gpu, dtype, [150, 71, 0], 4, 2, 64, 64, rows, causal=False)


@DTYPES
def test_attend_with_counts_leaves_zeros_behind_them(gpu, dtype):
    check_attend(gpu, dtype, [100, 40, 9, 64], 4, 4, 64, 32, 5, counts=[5, 0, 2, 1])
    check_attend(gpu, dtype, [100, 140], 4, 2, 128, 64, 90, counts=[90, 33])


@DTYPES
@pytest.mark.parametrize("scale", [0.0, 4.0])
def test_attend_with_flat_and_sharp_weights(gpu, scale, dtype):
    check_attend(gpu, dtype, [333], 4, 2, 64, 32, 1, scale=scale)
    check_attend(gpu, dtype, [333], 4, 2, 64, 32, 50, scale=scale)


@DTYPES
def test_attend_takes_views_of_q(gpu, dtype):
    rng = rng_of(41)
    cache, held, _ = filled(gpu, rng, dtype, [50, 61], 2, 64, 32)
    x = rng.standard_normal((2, 3, 10, 64)).astype(dtype)  # [batch, tokens, heads and more, dim]
    y = rng.standard_normal((2, 4, 64, 3)).astype(dtype)   # the last dimension of the view is not dense
    got = computed(leaf(gpu, x).narrow(2, 1, 4).transpose(1, 2).attend(cache), leaf(gpu, y).transpose(2, 3).attend(cache))
    for g, q in zip(got, (x[:, :, 1:5].transpose(0, 2, 1, 3), y.transpose(0, 1, 3, 2))):
        for b, n in enumerate((50, 61)):
            want, slack = ref.attend(q[b], *held[b], np.float32(0.125).astype(np.float64), True, n, 3)
            if dtype == F16:
                slack = slack + ref.f16_weights_slack(q[b], *held[b], 0.125, True, n, 3)
            ref.close(g[b], want, dtype, slack)


@DTYPES
@pytest.mark.parametrize("rows,kv", [(4, 1), (40, 1), (70, 256)])
def test_attend_keeps_nan_and_infinities_of_q_in_their_rows(gpu, rows, kv, dtype):
    rng = rng_of(42, rows)
    cache, held, _ = filled(gpu, rng, dtype, [100], kv, 64, 32)
    q = rng.standard_normal((2 * kv, rows, 64)).astype(dtype)
    clean = computed(leaf(gpu, q).attend(cache))
    q[0, 1, 5], q[1, 2, 0] = np.nan, np.inf
    got = computed(leaf(gpu, q).attend(cache))
    assert np.all(np.isnan(got[0, 1])) and np.all(np.isnan(got[1, 2]))
    rest = np.ones((2 * kv, rows), bool)
    rest[0, 1] = rest[1, 2] = False
    assert np.array_equal(got[rest], clean[rest])


@DTYPES
@pytest.mark.parametrize("rows,kv", [(1, 2), (60, 2), (70, 256)])
def test_attend_over_zero_blocks_and_what_lies_behind_the_end(gpu, rows, kv, dtype):
    """Blocks of zeros (scale 0) among others; infinities and NaN in tokens that a reset has forgotten."""
    w, rng = load_package(), rng_of(43, rows)
    k, v = (rng.standard_normal((1, kv, 160, 64)).astype(dtype) for _ in range(2))
    v[:, :, 32:64] = 0
    k[:, :, 64:96] = 0
    v[:, 1] = 0  # a head without any values
    cache = w.KvCache(gpu, 1, kv, 64, 320, 32)
    cache.append(leaf(gpu, np.full((1, kv, 320, 64), np.inf, dtype)), leaf(gpu, np.full((1, kv, 320, 64), np.nan, dtype)))
    cache.reset()
    cache.append(leaf(gpu, k), leaf(gpu, v))
    held = [np.stack([ref.values(x[0, h], 32) for h in range(kv)]) for x in (k, v)]
    q = rng.standard_normal((1, 2 * kv, rows, 64)).astype(dtype)
    got = computed(leaf(gpu, q).attend(cache))
    want, slack = ref.attend(q[0], *held, 0.125, True, 160, rows)
    if dtype == F16:
        slack = slack + ref.f16_weights_slack(q[0], *held, 0.125, True, 160, rows)
    ref.close(got[0], want, dtype, slack)
    assert np.all(got[0, 2:4] == 0)


@pytest.mark.parametrize("scale", [0.0, 0.125])
def test_attend_with_many_rows_before_a_block_of_zero_keys_and_large_values(gpu, scale):
    """Rows that end before a block are not touched by its scales, also where those scales make every score 0."""
    w, rng = load_package(), rng_of(45)
    cache = w.KvCache(gpu, 4, 16, 64, 64, 32)
    k, v = (rng.standard_normal((4, 16, 64, 64)).astype(F32) for _ in range(2))
    k[:, :, 32:] = 0
    v[:, :, 32:] *= F32(1e9)  # f16 holds no result of the rows that see them
    cache.append(leaf(gpu, k), leaf(gpu, v))
    q = rng.standard_normal((4, 128, 64, 64)).astype(F16)
    out = leaf(gpu, q).attend(cache, scale)
    got, held = computed(out, cache.values(0, 32, w.F32))
    assert [i.kind for i in out.kernels()] == ["attend_prompt"]
    for b in range(4):
        case = (q[b, :, :32], held[0, b].astype(np.float64), held[1, b].astype(np.float64), scale, True, 32, 32)
        want, slack = ref.attend(*case)
        ref.close(got[b, :, :32], want, F16, slack + ref.f16_weights_slack(*case), f"sequence {b}")


@DTYPES
def test_attend_in_a_cache_of_more_than_32_bits_of_bytes(gpu, dtype):
    """The last head's keys and all values lie behind 4 GiB; one sequence of a few is long, the others short."""
    check_attend(gpu, dtype, [3000, 1, 64], 3, 3, 128, 64, 1, capacity=5 << 20)
    check_attend(gpu, dtype, [200, 130, 70], 3, 3, 128, 64, 70, capacity=5 << 20)


def test_attend_over_many_short_sequences_and_a_long_one(gpu):
    check_attend(gpu, F16, [4000] + [3, 40, 0, 17] * 30, 8, 8, 64, 32, 1)


def test_the_operators_under_the_reference_s_own_fusion(gpu):
    """Nothing is shared or joined there; the values are the same."""
    w, rng = load_package(), rng_of(46)
    codes, scales, z = ref.q4_weights(rng, 128, 256, 32, True, F16)
    weights = w.Q4Weights(gpu, codes, scales, z, 32)
    x = leaf(gpu, rng.standard_normal((800, 128)).astype(F16))
    c, s = (leaf(gpu, rng.standard_normal((800, 32)).astype(F32)) for _ in range(2))
    g = leaf(gpu, np.ones(64, F32))
    got = []
    for mode in (w.FUSION_TREE, w.FUSION_REFERENCE):
        gpu.set_fusion(mode)
        try:
            cache = w.KvCache(gpu, 1, 2, 64, 800, 32)
            y = x.mat_mul_q4(weights)
            q, k = (y.narrow(1, at, n * 64).reshape([800, n, 64]).transpose(0, 1).norm_rope(g, c, s, 1e-5) for at, n in ((0, 2), (128, 2)))
            cache.append(k, y.narrow(1, 128, 128).reshape([800, 2, 64]).transpose(0, 1))
            lazy = [q, k, q.attend(cache, 0.125), cache.values(0, 800, w.F16)]
            outs = [w.Tensor.zeros(gpu, t.shape(), w.F16) for t in lazy]
            w.materialize_into(lazy, outs)
            got += outs
        finally:
            gpu.set_fusion(w.FUSION_TREE)
    values = computed(*got)
    for i in range(4):
        assert np.array_equal(values[i], values[4 + i])


def test_attend_of_an_empty_cache_and_of_no_rows(gpu):
    w = load_package()
    cache = w.KvCache(gpu, 2, 2, 64, 64, 32)
    q = leaf(gpu, np.ones((2, 4, 3, 64), F16))
    none = leaf(gpu, np.ones((2, 4, 0, 64), F16))
    got = computed(q.attend(cache, counts=[0, 0]), none.attend(cache))
    assert np.all(got[0] == 0) and got[1].shape == (2, 4, 0, 64)


def test_attend_gives_the_same_bits_every_time(gpu):
    rng = rng_of(44)
    for kv, lengths, rows in ((2, [5000, 1200], 1), (2, [5000, 1200], 64), (64, [300, 200], 200)):
        cache, _, _ = filled(gpu, rng, F16, lengths, kv, 128, 64)
        t = leaf(gpu, rng.standard_normal((2, 4 * kv, rows, 128)).astype(F16)).attend(cache)
        first = computed(t)
        for _ in range(3):
            assert np.array_equal(computed(t), first)


# ---- attention of sequences with different numbers of rows -----------------------------------------------------------

def check_attend_by(kernel, gpu, dtype, lengths, counts, heads, kv, dim, block, rows=None, causal=True, scale=None, seed=0):
    """As check_attend, by a kernel of this name; rows of q behind a count are NaN, and their results zeros."""
    rows = max(counts) if rows is None else rows
    rng = rng_of(60, seed, dim, block, rows, *lengths)
    cache, held, _ = filled(gpu, rng, dtype, lengths, kv, dim, block)
    q = rng.standard_normal((len(lengths), heads, rows, dim)).astype(dtype)
    for b, n in enumerate(counts):
        q[b, :, n:] = np.nan
    scale = np.float32(dim ** -0.5 if scale is None else scale).astype(np.float64)
    t = leaf(gpu, q).attend(cache, scale, causal, counts)
    t.materialize()
    assert [i.kind for i in t.kernels()] == [kernel], [(i.kind, i.detail) for i in t.kernels()]
    got = computed(t)
    for b, n in enumerate(lengths):
        case = (q[b, :, :counts[b]], *held[b], scale, causal, n, counts[b])
        want, slack = ref.attend(*case)
        if dtype == F16:
            slack = slack + ref.f16_weights_slack(*case)
        ref.close(got[b, :, :counts[b]], want, dtype, slack, f"sequence {b}")
        assert np.all(got[b, :, counts[b]:] == 0), f"sequence {b}"
    return t, got


MIXED_CASES = [  # lengths, counts, heads, kv heads, dim, block, rows
    ([3000, 2500, 40, 700], [200, 1, 1, 3], 8, 2, 64, 32, 200), ([5000, 131, 64, 5000], [1, 130, 0, 1], 16, 4, 128, 64, 131),
    ([4000, 3900, 4000], [0, 2, 0], 4, 2, 80, 128, 33), ([4000, 3000, 100], [1, 0, 0], 4, 1, 20, 32, 9), ([0, 3000, 0, 2000], [0, 17, 0, 16], 2, 2, 256, 64, 18),
    ([900] * 9 + [6000], [1] * 9 + [50], 6, 3, 96, 64, 50), ([2000, 1], [5, 1], 12, 2, 64, 32, 100),
]


@DTYPES
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", MIXED_CASES, ids=str)
def test_attend_of_a_chunk_beside_single_tokens(gpu, case, causal, dtype):
    lengths, counts, heads, kv, dim, block, rows = case
    t, got = check_attend_by("attend_rows", gpu, dtype, lengths, counts, heads, kv, dim, block, rows, causal)
    for _ in range(3):
        assert np.array_equal(computed(t), got)


# so many rows of like sequences that tiles of 128 fill the chip
FULL_CASES = [([150, 0, 129, 200], [129, 0, 129, 129], 96, 96, 64, 64), ([100, 37, 300, 1, 128, 0], [100, 37, 100, 1, 100, 0], 165, 55, 72, 32),
              ([141, 140, 0, 270, 64, 33], [140, 140, 0, 140, 64, 33], 96, 48, 128, 128), ([260] * 4, [256] * 4, 32, 32, 128, 64), ([400, 260], [200, 200], 128, 64, 16, 32)]


@DTYPES
@pytest.mark.parametrize("case", FULL_CASES, ids=str)
def test_attend_with_full_tiles(gpu, case, dtype):
    check_attend_by("attend_prompt", gpu, dtype, *case)


@pytest.mark.parametrize("dtype,lengths,counts,heads,kv,dim,block", [(F32, [70, 66, 0, 5, 65, 64, 71, 74], [70, 66, 0, 5, 65, 64, 70, 70], 96, 48, 200, 32), (F32, [70, 66, 0, 70], [70, 66, 0, 70], 160, 80, 255, 32),
                                                                     (F32, [300, 280], [140, 140], 112, 56, 130, 64), (F16, [300, 280], [140, 140], 112, 56, 130, 64),
                                                                     (F16, [128, 128, 127, 128], [128, 128, 0, 127], 344, 86, 200, 32)], ids=str)
def test_attend_with_full_tiles_of_large_heads(gpu, dtype, lengths, counts, heads, kv, dim, block):
    check_attend_by("attend_prompt", gpu, dtype, lengths, counts, heads, kv, dim, block)


@DTYPES
def test_attend_with_full_tiles_in_other_ways(gpu, dtype):
    check_attend_by("attend_prompt", gpu, dtype, [150, 0, 190, 65], [70, 0, 70, 65], 216, 216, 64, 32, causal=False)
    check_attend_by("attend_prompt", gpu, dtype, [150, 0, 190, 65], [70, 0, 70, 33], 216, 216, 64, 32)
    check_attend_by("attend_prompt", gpu, dtype, [150, 0, 190, 65], [64, 0, 100, 65], 192, 96, 64, 64, causal=False)
    for scale in (0.0, 4.0):
        check_attend_by("attend_prompt", gpu, dtype, [150, 10, 190, 65], [70, 10, 70, 65], 216, 216, 64, 64, scale=scale)


# ---- without roundings to f16 on the way -----------------------------------------------------------------------------------

@pytest.mark.parametrize("kernel,lengths,counts,heads,kv,dim,block,exact", [
    ("attend_rows", [1000, 0, 33], [1, 0, 1], 32, 8, 128, 64, False), ("attend_rows", [3000], [3], 5, 1, 64, 32, False), ("attend_rows", [700, 130], [2, 2], 16, 2, 256, 128, False),
    ("attend_rows", [300, 4000], [40, 1], 4, 2, 80, 32, True), ("attend_rows", [333], [50], 40, 1, 20, 64, True),
    ("attend_prompt", [150, 0, 129, 200], [129, 0, 129, 129], 96, 96, 64, 64, True), ("attend_prompt", [260] * 4, [256] * 4, 32, 32, 128, 64, True),
    ("attend_prompt", [128, 128, 127, 128], [128, 128, 0, 127], 344, 86, 200, 32, True)], ids=str)
def test_attend_in_f16_with_weights_of_22_bits(gpu, kernel, lengths, counts, heads, kv, dim, block, exact):
    """One tile of rows a key head, and any number of them under exact math."""
    rng = rng_of(62, dim, *lengths)
    cache, held, _ = filled(gpu, rng, F16, lengths, kv, dim, block)
    q = rng.standard_normal((len(lengths), heads, max(counts), dim)).astype(F16)
    scale = np.float32(dim ** -0.5).astype(np.float64)
    t = leaf(gpu, q).attend(cache, scale, True, counts)
    gpu.set_exact_math(exact)
    try:
        t.materialize()
        assert [i.kind for i in t.kernels()] == [kernel]
        got = computed(t)
    finally:
        gpu.set_exact_math(False)
    for b, n in enumerate(lengths):
        case = (q[b], *held[b], scale, True, n, counts[b])
        want, slack = ref.attend(*case)
        ref.close(got[b], want, F16, slack + ref.two_part_weights_slack(*case), f"sequence {b}")


@pytest.mark.parametrize("lengths,rows,exact", [([1000], 1, False), ([3000, 700], 2, False), ([700, 650], 60, True)], ids=str)
def test_attend_in_f16_errs_by_the_rounding_of_its_result(gpu, lengths, rows, exact):
    """In the 2-norm.  A rounding is spread evenly over half a step to both sides: its square is step^2 / 12 on average.  The
    step is 2^-10 of the power of two below the value, and the square of that power over the value's is on average (1 - 1/4) /
    (2 ln 2) where significands are spread as 1 / m: 2.07e-4 of the result.  Ten thousand values come within 1 % of that, 10 % are
    allowed; one more rounding of each weight makes it 2.6e-4 and more."""
    w, rng = load_package(), rng_of(64, rows, *lengths)
    cache, held, _ = filled(gpu, rng, F16, lengths, 8, 128, 64, spread=False)
    q = rng.standard_normal((len(lengths), 32, rows, 128)).astype(F16)
    gpu.set_exact_math(exact)
    try:
        got = computed(leaf(gpu, q).attend(cache)).astype(np.float64)
    finally:
        gpu.set_exact_math(False)
    scale = np.float32(128 ** -0.5).astype(np.float64)
    want = np.stack([ref.attend(q[b], *held[b], scale, True, n, rows)[0] for b, n in enumerate(lengths)])
    normal = np.abs(want) >= 2.0 ** -14
    off = np.sqrt(np.square(got - want)[normal].sum() / np.square(want)[normal].sum())
    assert off < 1.1 * 2.0 ** -10 * np.sqrt(0.75 / (2 * np.log(2)) / 12), off


Q4_MANY = [(1100, 130, 7700, 128, True, F16), (800, 72, 11001, 32, False, F32), (1100, 130, 2000, 128, True, F16), (768, 64, 64, 32, False, F16), (800, 264, 300, 96, True, F32)]


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("case", Q4_MANY, ids=lambda c: "x".join(str(v) for v in c[:4]))
def test_mat_mul_q4_rounds_weights_only_where_it_writes_them_out(gpu, case, exact):
    w, (m, k, n, group, zeros, sdt) = load_package(), case
    rng = rng_of(63, m, k, n, group)
    codes, scales, z = ref.q4_weights(rng, k, n, group, zeros, sdt)
    x = rng.standard_normal((m, k)).astype(F16)
    y = leaf(gpu, x).mat_mul_q4(w.Q4Weights(gpu, codes, scales, z, group))
    gpu.set_exact_math(exact)
    try:
        y.materialize()
        written = "q4_dense" in [i.kind for i in y.kernels()]
        got = computed(y)
    finally:
        gpu.set_exact_math(False)
    assert written == (n > 7000 and not exact)
    dense = ref.q4_dense(codes, scales, z, group)
    ref.close(got, x.astype(np.float64) @ dense, F16, ref.q4_slack(x, dense, written), str(case))


# ---- together ---------------------------------------------------------------------------------------------------

@DTYPES
def test_a_block_serves_a_prompt_and_then_tokens(gpu, dtype):
    """Project with 4-bit weights, normalise and rotate, store, attend, project: a prompt of two lengths, then one token of
    each sequence at a time, every step against the same steps in 64 bits on the step's own inputs, through outputs that
    stay on the device."""
    w, rng = load_package(), rng_of(50)
    hidden, heads, kv, dim, block, batch = 96, 4, 2, 64, 32, 2
    width = (heads + 2 * kv) * dim
    code = w.F16 if dtype == F16 else w.F32
    into = ref.q4_weights(rng, hidden, width, 32, True, F16)
    back = ref.q4_weights(rng, heads * dim, hidden, 64, False, F16)
    w_in, w_out = w.Q4Weights(gpu, *into, 32), w.Q4Weights(gpu, *back, 64)
    gq, gk = (rng.uniform(0.5, 1.5, dim).astype(dtype) for _ in range(2))
    angle = np.arange(80)[:, None] * 10000.0 ** (-np.arange(dim // 2) / (dim // 2))
    c, s = np.cos(angle).astype(F32), np.sin(angle).astype(F32)
    tgq, tgk, tc, ts = (leaf(gpu, v) for v in (gq, gk, c, s))
    cache = w.KvCache(gpu, batch, kv, dim, 80, block)
    past = [[np.zeros((kv, 0, dim)) for _ in range(2)] for _ in range(batch)]
    lengths = [0, 0]
    for counts in ([40, 23], [1, 1], [1, 1], [2, 0], [1, 1]):
        n = max(counts)
        x = rng.standard_normal((batch * n, hidden)).astype(dtype)
        qkv = w.Tensor.zeros(gpu, (batch * n, width), code)
        w.materialize_into([leaf(gpu, x).mat_mul_q4(w_in)], [qkv])
        parts = qkv.reshape([batch, n, heads + 2 * kv, dim])
        view = lambda at, count: parts.narrow(2, at, count).transpose(1, 2)  # noqa: E731
        turned = [view(0, heads).norm_rope(tgq, tc, ts, 1e-6, lengths), view(heads, kv).norm_rope(tgk, tc, ts, 1e-6, lengths)]
        q, k = w.materialize_into(turned, [w.Tensor.zeros(gpu, t.shape(), code) for t in turned])
        cache.append(k, view(heads + kv, kv), counts)
        o = w.Tensor.zeros(gpu, (batch, heads, n, dim), code)
        w.materialize_into([q.attend(cache, counts=counts)], [o])
        y = o.transpose(1, 2).reshape([batch * n, heads * dim]).mat_mul_q4(w_out)
        if gpu.is_planner:
            y.materialize()
            lengths = [a + b for a, b in zip(lengths, counts)]
            continue
        h_qkv, h_q, h_k, h_o, h_y = (t.to_numpy() for t in (qkv, q, k, o, y))
        dense = ref.q4_dense(*into, 32)
        ref.close(h_qkv, x.astype(np.float64) @ dense, dtype, ref.q4_slack(x, dense))
        split = h_qkv.reshape(batch, n, heads + 2 * kv, dim).transpose(0, 2, 1, 3)
        for got, part, g in ((h_q, split[:, :heads], gq), (h_k, split[:, heads:heads + kv], gk)):
            ref.close(got, ref.norm_rope(part, g, c, s, 1e-6, lengths), dtype, ref.norm_rope_slack(part, g, 1e-6))
        for b in range(batch):
            lengths[b] += counts[b]
            for i, new in enumerate((h_k[b], split[b, heads + kv:])):
                past[b][i] = np.concatenate([past[b][i], new[:, :counts[b]].astype(np.float64)], 1)
            held = [np.stack([ref.values(t, block) for t in p]) for p in past[b]]
            want, slack = ref.attend(h_q[b], *held, 0.125, True, lengths[b], counts[b])
            if dtype == F16:
                slack = slack + ref.f16_weights_slack(h_q[b], *held, 0.125, True, lengths[b], counts[b])
            ref.close(h_o[b], want, dtype, slack)
        rows = h_o.transpose(0, 2, 1, 3).reshape(batch * n, heads * dim)
        dense = ref.q4_dense(*back, 64)
        ref.close(h_y, rows.astype(np.float64) @ dense, dtype, ref.q4_slack(rows, dense))
    if gpu.is_planner:
        pytest.skip("plan-only device: kernels compiled, nothing computed")
    assert cache.lengths() == lengths


def test_two_threads_at_once(gpu):
    """Two programs on one device, weights shared, a cache each, and one cache that both read: the values of one after the other."""
    w, rng = load_package(), rng_of(47)
    codes, scales, z = ref.q4_weights(rng, 256, 256, 64, True, F16)
    weights = w.Q4Weights(gpu, codes, scales, z, 64)
    x = rng.standard_normal((2, 20, 256)).astype(F16)
    common = w.KvCache(gpu, 1, 2, 64, 3000, 64)
    k = rng.standard_normal((1, 2, 3000, 64)).astype(F16)
    common.append(leaf(gpu, k), leaf(gpu, k))

    def program(i):
        cache, out, seen = w.KvCache(gpu, 1, 2, 64, 400, 32), w.Tensor.zeros(gpu, (1, 4, 20, 64), w.F16), []
        t = leaf(gpu, x[i])
        for _ in range(12):
            y = t.mat_mul_q4(weights)
            heads = y.reshape([20, 4, 64]).transpose(0, 1).reshape([1, 4, 20, 64])
            cache.append(heads.narrow(1, 0, 2), heads.narrow(1, 2, 2))
            w.materialize_into([heads.attend(cache) + heads.attend(common)], [out])
            seen.append(None if gpu.is_planner else out.to_numpy())
        return seen

    alone = [program(0), program(1)]
    if gpu.is_planner:
        pytest.skip("plan-only device: kernels compiled, nothing computed")
    with ThreadPoolExecutor(2) as pool:
        both = list(pool.map(program, range(2)))
    for one, other in zip(alone, both):
        assert all(np.array_equal(a, b) for a, b in zip(one, other))
        assert np.isfinite(one[-1]).all() and not np.array_equal(one[0], one[-1])


def test_views_of_device_memory(gpu):
    """Another library's view of a tensor that holds data reads what a later call left there."""
    w = load_package()
    t = w.Tensor.zeros(gpu, (3, 4), w.F16)
    if gpu.is_planner:
        pytest.skip("plan-only device: no device memory")
    face = t.__cuda_array_interface__
    assert face["shape"] == (3, 4) and face["typestr"] == "<f2" and face["data"] == (t.device_ptr(), False) and face["strides"] is None
    assert not hasattr(t + 1.0, "__cuda_array_interface__")
    assert np.array_equal(t.to_numpy(), np.zeros((3, 4), F16))
    w.materialize_into([t + 1.0], [t])
    assert np.array_equal(t.to_numpy(), np.ones((3, 4), F16)) and t.__cuda_array_interface__["data"] == face["data"]
