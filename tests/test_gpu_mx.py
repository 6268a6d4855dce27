"""Block-scaled tensors on a B200, through the C ABI, against the 64-bit implementations of mx_reference.

Quantisation and restoration are exact: every byte and value is compared for equality.  For the products, S is the
sum of the magnitudes of a result's terms: each step of the tensor cores (32 or more products) may lose one unit of
2^-23 of the running sum, which never exceeds S."""
import numpy as np
import pytest

import mx_reference as ref
from helpers import run_image
from synaptik_b200 import native, nn, program
from synaptik_b200.program import F32, GraphBuilder

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16"]
ACTIVATIONS = ["relu", "tanh", "sigmoid", "silu", "gelu_tanh", "gelu"]


@pytest.fixture(scope="module")
def ctx():
    c = native.Context(0)
    yield c
    c.close()


def mixed(rng, *shape):
    """Values whose magnitude varies from block to block, with exact zeros and a few far above the rest."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-12, 12, shape[:-1] + (1,)))
    x *= np.where(rng.random(shape) < 0.02, 50.0, 1.0)
    return np.where(rng.random(shape) < 0.1, 0.0, x).astype(np.float32)


def special_blocks():
    """One block each of what quantisation treats apart."""
    f = np.float32
    rows = [np.zeros(32), -np.zeros(32), np.full(32, 6.0), np.full(32, 448.0), np.full(32, np.nextafter(f(6), f(7))), np.full(32, np.nextafter(f(448), f(449))),
            np.linspace(-6, 6, 32), np.linspace(-448, 448, 32), np.linspace(0, 2.0 ** -130, 32), np.full(32, 2.0 ** -149), np.full(32, np.finfo(f).max),
            np.full(32, np.finfo(f).tiny), np.concatenate([[np.inf], np.ones(31)]), np.concatenate([np.ones(31), [np.nan]]), np.concatenate([[-np.inf], np.zeros(31)]),
            # halfway between neighbouring elements, both formats: ties go to the even code
            np.concatenate([[6.0], np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, -2.5], 4)[:31]]),
            np.concatenate([[448.0], np.tile([17.0, 19.0, 21.0, 232.0, 2.0 ** -10, 3 * 2.0 ** -10, -17.0], 5)[:31]])]
    return np.array(rows, dtype=np.float32).reshape(1, -1)


def quantized(ctx, kind, fmt, fed, shape, strides=None, permute=None):
    g = GraphBuilder()
    x = g.feed(ref.STORAGE[kind], shape, strides)
    if permute:
        x = g.permute(x, permute)
    held = g.mx_quantize(x, fmt)
    g.publish(held.codes)
    g.publish(held.scales)
    return run_image(ctx, g, [fed])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 128), (2, 129), (64, 784), (33, 785), (1, 4096), (300, 256), (5000, 40), (17,), (2, 3, 100), (2, 3, 5, 36), (0, 64)])
def test_quantize_is_exact(ctx, kind, fmt, shape):
    rng = np.random.default_rng(len(shape) * 1000 + shape[-1])
    fed, exact = ref.stored(kind, mixed(rng, *shape) if shape != (0, 64) else np.zeros(shape))
    codes, scales = quantized(ctx, kind, fmt, fed, shape)
    want_codes, want_scales = ref.quantize(exact, fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_quantize_special_blocks(ctx, kind, fmt):
    fed, exact = ref.stored(kind, special_blocks())
    codes, scales = quantized(ctx, kind, fmt, fed, fed.shape)
    want_codes, want_scales = ref.quantize(exact, fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)


@pytest.mark.parametrize("kind", KINDS)
def test_quantize_strided_views(ctx, kind):
    rng = np.random.default_rng(5)
    fed, exact = ref.stored(kind, mixed(rng, 50, 70))
    # rows of 64 out of rows of 70; the transpose; every second row and column through strides; a rank-3 PERMUTE
    for shape, strides, permute, view in [((50, 64), (70, 1), None, exact[:, :64]), ((50, 70), None, (1, 0), exact.T),
                                          ((25, 35), (140, 2), None, exact[::2, ::2]), ((5, 10, 70), None, (1, 0, 2), exact.reshape(5, 10, 70).transpose(1, 0, 2)),
                                          ((5, 10, 70), None, (2, 1, 0), exact.reshape(5, 10, 70).transpose(2, 1, 0))]:
        codes, scales = quantized(ctx, kind, "mx8", fed.reshape(shape) if strides is None else fed, shape, strides, permute)
        want_codes, want_scales = ref.quantize(view, "mx8")
        assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)


def random_held(rng, fmt, shape):
    """Any bytes a block-scaled tensor may hold (no NaN codes), padding zero."""
    features = shape[-1]
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-6, 6, shape[:-1] + (1,)))
    return ref.quantize(x.astype(np.float32), fmt)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (64, 128), (33, 785), (2, 3, 40), (1000, 48), (0, 5)])
def test_restore_is_exact(ctx, kind, fmt, shape):
    rng = np.random.default_rng(shape[-1])
    codes = rng.integers(0, 256, shape[:-1] + (program.mx_code_bytes(fmt, shape[-1]),)).astype(np.uint8)
    scales = rng.integers(0, 256, shape[:-1] + (program.mx_scale_bytes(shape[-1]),)).astype(np.uint8)
    g = GraphBuilder()
    held = g.mx_feed(fmt, shape)
    g.publish(g.mx_restore(held, ref.STORAGE[kind]))
    got, = run_image(ctx, g, [codes, scales])
    with np.errstate(over="ignore", invalid="ignore"):
        want = ref.values(codes, scales, fmt, shape[-1])
        want = program.to_storage(kind, want.astype(np.float32))      # exact in FLOAT32 apart from overflow, then one rounding
    assert np.array_equal(ref.read(kind, got), ref.read(kind, want), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("shape", [(1, 1), (1023, 129), (64, 256), (2, 3, 40), (0, 32)])
def test_activation_gradient(ctx, kind, act, shape):
    """The functions' errors (exp 2 units, division 2, erfc 4, their arguments' roundings times slopes below 1.2) stay
    below 40 units of 2^-24 of the upstream gradient; then one rounding to the storage type."""
    rng = np.random.default_rng(shape[-1])
    codes, scales = ref.quantize(rng.standard_normal(shape).astype(np.float32) * 3, "mx8")
    fed, up = ref.stored(kind, rng.standard_normal(shape))
    g = GraphBuilder()
    held, u = g.mx_feed("mx8", shape), g.feed(ref.STORAGE[kind], shape)
    g.publish(g.mx_activation_gradient(act, held, u))
    got, = run_image(ctx, g, [codes, scales, fed])
    want = up * ref.slope(act, ref.values(codes, scales, "mx8", shape[-1]))
    bound = 40 * 2.0 ** -24 * np.abs(up) + ref.EPS[kind] / 2 * np.abs(want) + (2.0 ** -25 if kind == "f16" else 0)
    assert (np.abs(ref.read(kind, got) - want) <= bound).all()


@pytest.mark.parametrize("act", ACTIVATIONS)
def test_activation_gradient_special_values(ctx, act):
    """Blocks of NaN give NaN; values far out have slope 0 or 1; a closed ReLU gate gives 0 for an infinite upstream."""
    x = np.zeros((5, 32), dtype=np.float32)
    x[0, 3] = np.nan
    x[1], x[2], x[3], x[4] = 1e30, -1e30, 3.4e38, -3.4e38
    codes, scales = ref.quantize(x, "mx8")
    up = np.ones((5, 32), dtype=np.float32)
    if act == "relu":
        up[2] = np.inf
    g = GraphBuilder()
    held, u = g.mx_feed("mx8", x.shape), g.feed(F32, x.shape)
    g.publish(g.mx_activation_gradient(act, held, u))
    got, = run_image(ctx, g, [codes, scales, up])
    open_slope = 0.0 if act in ("tanh", "sigmoid") else 1.0
    assert np.isnan(got[0]).all()
    assert (got[1] == open_slope).all() and (got[2] == 0).all() and (got[3] == open_slope).all() and (got[4] == 0).all()


def test_activation_gradient_is_the_derivative(ctx):
    """Against central differences of the activation in 64 bits: h^2 / 6 * |act'''| <= 1e-8 * 2, the difference quotient
    rounds at 1e-16 / 1e-4."""
    z = np.linspace(-6, 6, 352, dtype=np.float32).reshape(11, 32)
    codes, scales = ref.quantize(z, "mx8")
    held = ref.values(codes, scales, "mx8", 32)
    for act in ACTIVATIONS[1:]:
        g = GraphBuilder()
        mx, u = g.mx_feed("mx8", z.shape), g.feed(F32, z.shape)
        g.publish(g.mx_activation_gradient(act, mx, u))
        got, = run_image(ctx, g, [codes, scales, np.ones_like(z)])
        h = 1e-4
        difference = (ref.activate(act, held + h) - ref.activate(act, held - h)) / (2 * h)
        assert np.abs(got - difference).max() <= 40 * 2.0 ** -24 + 2e-8


def linear(ctx, kind, x, w, bias, act):
    """x, w: (codes, scales) with their feature count; returns float64 results."""
    g = GraphBuilder()
    xm, wm = g.mx_feed("mx4", x[2]), g.mx_feed("mx4", w[2])
    feeds = [x[0], x[1], w[0], w[1]]
    b = None
    if bias is not None:
        b = g.feed(ref.STORAGE[kind], bias.shape)
        feeds.append(bias)
    g.publish(g.mx_linear(xm, wm, b, act, ref.STORAGE[kind]))
    got, = run_image(ctx, g, feeds)
    return ref.read(kind, got)


def check_linear(ctx, kind, lead, k, n, act=None, bias=True, seed=0):
    rng = np.random.default_rng(seed + k * 7 + n)
    x = (*random_held(rng, "mx4", lead + (k,)), lead + (k,))
    w = (*random_held(rng, "mx4", (n, k)), (n, k))
    xv, wv = ref.values(x[0], x[1], "mx4", k), ref.values(w[0], w[1], "mx4", k)
    fed, b = ref.stored(kind, rng.standard_normal(n)) if bias else (None, 0.0)
    z = xv @ wv.T + b
    s = np.abs(xv) @ np.abs(wv).T + np.abs(b)
    want = ref.activate(act, z)
    got = linear(ctx, kind, x, w, fed, act)
    # the activations' slopes stay below 1.2; their own errors below 40 units of 2^-24 of |z| + 1
    bound = 1.2 * (k / 32 + 4) * 2.0 ** -23 * s + 40 * 2.0 ** -24 * (np.abs(z) + 1 if act not in (None, "relu") else 0) + ref.EPS[kind] / 2 * np.abs(want) * 1.01
    if kind == "f16":
        bound = bound + 2.0 ** -24
        got, want = np.where(np.abs(want) > 65504, 0, got), np.where(np.abs(want) > 65504, 0, want)
    assert got.shape == want.shape
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 32, 8), (1, 784, 4096), (1, 4096, 1000), (2, 33, 5), (3, 100, 17), (5, 256, 130), (8, 129, 64), (9, 512, 300),
                                   (16, 785, 96), (17, 640, 257), (31, 1024, 96), (33, 64, 128), (64, 300, 200), (100, 4095, 100), (127, 96, 511), (128, 256, 256),
                                   (129, 288, 255), (200, 784, 1000), (257, 1000, 384), (500, 32, 10)])
def test_linear(ctx, kind, m, k, n):
    check_linear(ctx, kind, (m,), k, n)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("kind,m", [("f32", 3), ("bf16", 130), ("f16", 300)])
def test_linear_activations(ctx, kind, m, act):
    check_linear(ctx, kind, (m,), 320, 272, act)


@pytest.mark.parametrize("kind", KINDS)
def test_linear_without_bias_and_over_leading_dimensions(ctx, kind):
    check_linear(ctx, kind, (4,), 96, 40, "relu", bias=False)
    check_linear(ctx, kind, (3, 50), 130, 144, bias=False)
    check_linear(ctx, kind, (2, 2, 70), 64, 48)


def test_linear_no_rows(ctx):
    check_linear(ctx, "f32", (0,), 64, 16)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_special_values(ctx, m):
    """A block of NaN reaches exactly the results that read it; an infinite bias its column; scales far apart."""
    rng = np.random.default_rng(m)
    k, n = 200, 140
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[m // 2, 70] = np.nan
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[9, 199] = np.inf
    w[11] *= 2.0 ** 60
    w[12] *= 2.0 ** -100
    xq, wq = ref.quantize(x, "mx4"), ref.quantize(w, "mx4")
    bias = np.zeros(n, dtype=np.float32)
    bias[20] = -np.inf
    got = linear(ctx, "f32", (*xq, x.shape), (*wq, w.shape), bias, None)
    xv, wv = ref.values(*xq, "mx4", k), ref.values(*wq, "mx4", k)
    want = xv @ wv.T + bias
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(got[m // 2]).all() and np.isnan(got[:, 9]).all()
    good = np.isfinite(want)
    s = np.abs(xv) @ np.abs(wv).T
    assert (np.abs(got[good] - want[good]) <= 12 * 2.0 ** -23 * s[good]).all()
    assert np.array_equal(got[~good & ~np.isnan(want)], want[~good & ~np.isnan(want)])


@pytest.mark.parametrize("m", [3, 200, 3000])
@pytest.mark.parametrize("k", [32, 96, 288, 800])
def test_linear_ignores_what_pads_the_scales(ctx, m, k):
    """Bytes of a row of scales past its last block, NaN among them, do not reach the result."""
    rng = np.random.default_rng(m + k)
    n = 1000
    x, w = (*random_held(rng, "mx4", (m, k)), (m, k)), (*random_held(rng, "mx4", (n, k)), (n, k))
    want = linear(ctx, "f32", x, w, None, None)
    for held in (x, w):
        held[1][:, k // 32:] = 255
    assert np.array_equal(linear(ctx, "f32", x, w, None, None), want)


@pytest.mark.parametrize("kind,m,k,n", [("f32", 700, 512, 600), ("bf16", 1500, 2048, 4096), ("f16", 4100, 800, 1016)])
def test_linear_many_tiles(ctx, kind, m, k, n):
    check_linear(ctx, kind, (m,), k, n, "relu")


def weight_gradient(ctx, kind, held, shape, fed, n):
    g = GraphBuilder()
    mx, u = g.mx_feed("mx8", shape), g.feed(ref.STORAGE[kind], shape[:-1] + (n,))
    g.publish(g.mx_weight_gradient(mx, u))
    got, = run_image(ctx, g, [held[0], held[1], fed])
    return got.astype(np.float64)


def check_weight_gradient(ctx, kind, lead, k, n, seed=0):
    rng = np.random.default_rng(seed + k * 11 + n)
    held = random_held(rng, "mx8", lead + (k,))
    fed, up = ref.stored(kind, rng.standard_normal(lead + (n,)) * 0.01)
    x = ref.values(*held, "mx8", k).reshape(-1, k)
    up = up.reshape(-1, n)
    want, s = up.T @ x, np.abs(up).T @ np.abs(x)
    got = weight_gradient(ctx, kind, held, lead + (k,), fed, n)
    # at most three products and one addition per 16 rows, each losing up to 2^-23 of the running sum
    rows = x.shape[0]
    bound = (rows / 16 * 4 + 4) * 2.0 ** -23 * s + 2.0 ** -149
    assert got.shape == want.shape
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    if rows:        # errors of independent signs: far below the bound on the whole
        assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want) + 1e-30


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 32, 16), (2, 5, 3), (15, 33, 7), (16, 64, 128), (17, 100, 130), (63, 129, 65), (64, 256, 256), (65, 257, 255),
                                      (128, 784, 10), (200, 32, 1000), (300, 784, 136), (1024, 32, 128), (1000, 96, 1), (777, 300, 264)])
def test_weight_gradient(ctx, kind, rows, k, n):
    check_weight_gradient(ctx, kind, (rows,), k, n)


@pytest.mark.parametrize("kind", KINDS)
def test_weight_gradient_over_leading_dimensions(ctx, kind):
    check_weight_gradient(ctx, kind, (3, 41), 70, 40)


@pytest.mark.parametrize("kind,rows,k,n", [("f32", 5000, 520, 512), ("bf16", 9000, 784, 512), ("f16", 3000, 1024, 1000), ("f32", 20, 2500, 3300),
                                           ("bf16", 70, 4097, 2600), ("f16", 130, 3300, 2049), ("f32", 700, 1500, 4000)])
def test_weight_gradient_long(ctx, kind, rows, k, n):
    check_weight_gradient(ctx, kind, (rows,), k, n)


def test_weight_gradient_without_rows_is_zero(ctx):
    got = weight_gradient(ctx, "f32", (np.zeros((0, 64), np.uint8), np.zeros((0, 4), np.uint8)), (0, 40), np.zeros((0, 8), np.float32), 8)
    assert np.array_equal(got, np.zeros((8, 40)))


@pytest.mark.parametrize("kind", KINDS)
def test_weight_gradient_special_values(ctx, kind):
    """An infinite gradient gives infinities where the checkpoint is not zero and NaN where it is; a NaN block its columns."""
    rng = np.random.default_rng(2)
    rows, k, n = 150, 96, 40
    x = np.abs(rng.standard_normal((rows, k))).astype(np.float32) + 0.5
    x[7, 40] = np.nan
    x[100, 3] = 0
    up = rng.standard_normal((rows, n)).astype(np.float32)
    up[100, 5], up[101, 6], up[102, 8] = np.inf, np.nan, -np.inf
    held = ref.quantize(x, "mx8")
    fed, upv = ref.stored(kind, up)
    got = weight_gradient(ctx, kind, held, (rows, k), fed, n)
    xv = ref.values(*held, "mx8", k)
    with np.errstate(invalid="ignore"):
        want = np.stack([(upv[:, j:j + 1] * xv).sum(0) for j in range(n)])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    infinite = np.isinf(want)
    assert infinite.any() and np.array_equal(got[infinite], want[infinite])


def test_weight_gradient_is_the_derivative(ctx):
    """dL/dW of L = sum(G * (X W^T)) against differences along random directions: L is linear in W, so the
    difference quotient is exact up to rounding."""
    rng = np.random.default_rng(4)
    rows, k, n = 90, 70, 30
    held = random_held(rng, "mx8", (rows, k))
    up = rng.standard_normal((rows, n)).astype(np.float32)
    got = weight_gradient(ctx, "f32", held, (rows, k), up, n)
    x = ref.values(*held, "mx8", k)
    for _ in range(5):
        d = rng.standard_normal((n, k))
        loss = lambda w: float((up.astype(np.float64) * (x @ w.T)).sum())       # noqa: E731
        assert abs((loss(d) - loss(-d)) / 2 - (got * d).sum()) <= 1e-5 * np.abs(got * d).sum()


def test_same_bits_every_time(ctx):
    """No order of additions depends on the run."""
    rng = np.random.default_rng(9)
    held = random_held(rng, "mx8", (3000, 200))
    up = rng.standard_normal((3000, 150)).astype(np.float32)
    first = weight_gradient(ctx, "f32", held, (3000, 200), up, 150)
    x, w = (*random_held(rng, "mx4", (9, 2000)), (9, 2000)), (*random_held(rng, "mx4", (700, 2000)), (700, 2000))
    product = linear(ctx, "f32", x, w, None, None)
    for _ in range(3):
        assert np.array_equal(first, weight_gradient(ctx, "f32", held, (3000, 200), up, 150))
        assert np.array_equal(product, linear(ctx, "f32", x, w, None, None))


@pytest.mark.parametrize("m", [40, 300, 2600])
@pytest.mark.parametrize("order", ["weights fed", "weights first", "x first"])
def test_quantised_operands_are_complete_before_the_product(ctx, order, m):
    """Runs in a row whose inputs alternate: no product reads what an earlier run, or only part of this one, has written.
    Codes and scales are exact and no sum depends on the run, so the results are those of a product of fed codes."""
    k, n = 288, 2100
    rng = np.random.default_rng(m)
    xs = [mixed(rng, m, k) for _ in range(2)]
    ws = [mixed(rng, n, k) for _ in range(2)]
    held = [[(*ref.quantize(v.astype(np.float64), "mx4"), v.shape) for v in (x, w)] for x, w in zip(xs, ws)]
    want = [linear(ctx, "f32", x, w, None, "relu") for x, w in held]
    g = GraphBuilder()
    x = g.feed(F32, (m, k))
    if order == "weights fed":
        w = g.mx_feed("mx4", (n, k))
        q = g.mx_quantize(x, "mx4")
    else:
        w = g.feed(F32, (n, k))
        if order == "weights first":
            w = g.mx_quantize(w, "mx4")
            q = g.mx_quantize(x, "mx4")
        else:
            q = g.mx_quantize(x, "mx4")
            w = g.mx_quantize(w, "mx4")
    g.publish(g.mx_linear(q, w, None, "relu", F32))
    ex = native.Executable(ctx, g.build())
    feeds = [[ctx.upload(xs[i]), *([ctx.upload(held[i][1][0]), ctx.upload(held[i][1][1])] if order == "weights fed" else [ctx.upload(ws[i])])] for i in range(2)]
    outs = [ctx.buffer(4 * m * n) for _ in range(8)]
    try:
        for run, out in enumerate(outs):
            ex.enqueue(feeds[run % 2], [out])
        ex.finish()
        for run, out in enumerate(outs):
            assert np.array_equal(out.download(np.float32, (m, n)), want[run % 2].astype(np.float32)), run
    finally:
        ex.close()
        for b in outs + feeds[0] + feeds[1]:
            b.close()


@pytest.mark.parametrize("m", [40, 2600])
@pytest.mark.parametrize("view", ["contiguous", "permute", "expand"])
def test_a_view_of_the_quantised_input_as_weight_is_complete_before_the_product(ctx, view, m):
    """x . x^T whose weight is a view of what the launch in front makes, in runs in a row whose inputs alternate."""
    k = 288
    rng = np.random.default_rng(m)
    xs = [mixed(rng, m, k) for _ in range(2)]
    held = [(*ref.quantize(v.astype(np.float64), "mx4"), v.shape) for v in xs]
    want = [linear(ctx, "f32", h, h, None, "relu").astype(np.float32) for h in held]
    g = GraphBuilder()
    q = g.mx_quantize(g.feed(F32, (m, k)), "mx4")
    make = {"contiguous": g.contiguous, "permute": lambda v: g.permute(v, (0, 1)), "expand": lambda v: g.expand(v, v.shape)}[view]
    g.publish(g.mx_linear(q, program.MxValue("mx4", (m, k), make(q.codes), make(q.scales)), None, "relu", F32))
    ex = native.Executable(ctx, g.build())
    feeds = [ctx.upload(x) for x in xs]
    outs = [ctx.buffer(4 * m * m) for _ in range(8)]
    try:
        for run, out in enumerate(outs):
            ex.enqueue([feeds[run % 2]], [out])
        ex.finish()
        for run, out in enumerate(outs):
            assert np.array_equal(out.download(np.float32, (m, m)), want[run % 2]), run
    finally:
        ex.close()
        for b in outs + feeds:
            b.close()


@pytest.mark.parametrize("kind,rows,k,n", [("f32", 2600, 520, 512), ("bf16", 4000, 300, 512), ("f16", 3000, 784, 200)])
def test_sums_of_slices_are_complete_before_they_are_added(ctx, kind, rows, k, n):
    """Weight gradients cut into slices of the rows, in runs in a row whose gradients alternate: each run has the bits of
    a run by itself."""
    rng = np.random.default_rng(rows)
    held = random_held(rng, "mx8", (rows, k))
    fed = [ref.stored(kind, rng.standard_normal((rows, n)))[0] for _ in range(2)]
    want = [weight_gradient(ctx, kind, held, (rows, k), f, n).astype(np.float32) for f in fed]
    assert not np.array_equal(want[0], want[1])
    g = GraphBuilder()
    g.publish(g.mx_weight_gradient(g.mx_feed("mx8", (rows, k)), g.feed(ref.STORAGE[kind], (rows, n))))
    ex = native.Executable(ctx, g.build())
    kept, feeds = [ctx.upload(held[0]), ctx.upload(held[1])], [ctx.upload(f) for f in fed]
    outs = [ctx.buffer(4 * n * k) for _ in range(8)]
    try:
        for run, out in enumerate(outs):
            ex.enqueue(kept + [feeds[run % 2]], [out])
        ex.finish()
        assert ex.launch_count() == 3       # pieces, product, sums of the slices
        for run, out in enumerate(outs):
            assert np.array_equal(out.download(np.float32, (n, k)), want[run % 2]), run
    finally:
        ex.close()
        for b in outs + feeds + kept:
            b.close()


@pytest.mark.parametrize("order", [(32, 128), (128, 32), (160, 256)])
def test_products_that_share_scales_take_as_many_as_they_have_blocks(ctx, order):
    """One tensor of scales serves codes of other widths, as long as they fill the same row of scales: each product reads
    the blocks it has, whatever the one before it read."""
    m, n = 3000, 1000                   # enough tiles for scales in tiles
    rng = np.random.default_rng(order[0])
    wide = max(order)
    w_codes, w_scales = random_held(rng, "mx4", (n, wide))
    w_scales[::7, wide // 32 - 1] = 255         # NaN for the wide product, nothing to the narrow one
    xs = {k: random_held(rng, "mx4", (m, k)) for k in order}
    g = GraphBuilder()
    scales = g.feed(program.U8, w_scales.shape)
    feeds, want = [w_scales], []
    for k in order:
        x = g.mx_feed("mx4", (m, k))
        codes = g.feed(program.U8, (n, k // 2))
        g.publish(g.mx_linear(x, program.MxValue("mx4", (n, k), codes, scales)))
        feeds += [*xs[k], w_codes[:, :k // 2]]
        padded = w_scales.copy()
        padded[:, k // 32:] = 0
        want.append(linear(ctx, "f32", (*xs[k], (m, k)), (np.ascontiguousarray(w_codes[:, :k // 2]), padded, (n, k)), None, None))
    for got, expected in zip(run_image(ctx, g, feeds), want):
        assert np.array_equal(got, expected.astype(np.float32), equal_nan=True)


def keep_nonzero(x, codes, fmt):
    """Codes in which what is not zero takes at least the smallest element of its sign; blocks of NaN stay as they are."""
    b = ref.blocked(x)
    tiny = ((b != 0) & np.isfinite(b).all(-1, keepdims=True)).reshape(x.shape[:-1] + (-1,))
    negative = np.signbit(b).reshape(tiny.shape)
    if fmt == "mx8":
        return np.where(tiny & (codes & 127 == 0), np.where(negative, 129, 1), codes).astype(np.uint8)
    each = np.stack((codes & 15, codes >> 4), -1).reshape(tiny.shape)
    each = np.where(tiny & (each & 7 == 0), np.where(negative, 9, 1), each).astype(np.uint8)
    return each[..., 0::2] | (each[..., 1::2] << 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (64, 784), (33, 785), (300, 256)])
def test_quantize_keeps_what_is_not_zero(ctx, kind, fmt, shape):
    rng = np.random.default_rng(shape[-1])
    x = mixed(rng, *shape) * np.exp2(rng.integers(-40, 1, shape))       # most of a block far below its largest
    x[..., ::5] = 0
    x[..., 1::7] *= -1
    fed, exact = ref.stored(kind, x)
    g = GraphBuilder()
    held = g.mx_quantize(g.feed(ref.STORAGE[kind], shape), fmt, keep_nonzero=True)
    g.publish(held.codes)
    g.publish(held.scales)
    codes, scales = run_image(ctx, g, [fed])
    want_codes, want_scales = ref.quantize(exact, fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, keep_nonzero(exact, want_codes, fmt))
    back = ref.values(codes, scales, fmt, shape[-1])        # blocks with an infinity (large FLOAT16 values) are NaN
    assert np.array_equal(np.sign(back[~np.isnan(back)]), np.sign(exact[~np.isnan(back)]))


def test_quantize_keeps_special_blocks(ctx):
    """Zeros of both signs, blocks of NaN, numbers that vanish under their block's scale in FLOAT32."""
    x = special_blocks().reshape(-1, 32)
    x = np.concatenate([x, [np.concatenate([[f], np.full(31, -2.0 ** -149)]) for f in (3e38, 1.0, 2.0 ** -149)]]).astype(np.float32)
    g = GraphBuilder()
    held = g.mx_quantize(g.feed(F32, x.shape), "mx8", keep_nonzero=True)
    g.publish(held.codes)
    g.publish(held.scales)
    codes, scales = run_image(ctx, g, [x])
    want_codes, want_scales = ref.quantize(x, "mx8")
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, keep_nonzero(x.astype(np.float64), want_codes, "mx8"))


@pytest.mark.parametrize("k", [4096, 4128, 8192, 1 << 20])
def test_linear_long_contractions_of_one_sign(ctx, k):
    """Terms that are all positive: tensor memory truncates, so the error of a sum kept there grows with the contraction.
    At most 64 steps of the tensor cores, each losing up to one unit of 2^-23 of the running sum, lie between two additions
    in FP32 registers, and those (one per 4096 terms, and one per slice) lose half a unit each."""
    rng = np.random.default_rng(k)
    m, n = 3, 8
    held = []
    for rows in (m, n):
        codes, scales = random_held(rng, "mx4", (rows, k))
        # scales from 2^-10 to 1 in every row: with equal ones the sums would be whole numbers of small units, and exact
        held.append((codes & 0x77, (scales != 0) * rng.integers(117, 128, scales.shape).astype(np.uint8), (rows, k)))
    xv, wv = (ref.values(*h[:2], "mx4", k) for h in held)
    want = xv @ wv.T
    got = linear(ctx, "f32", *held, None, None)
    bound = (64 + (k / 4096 + 8) / 2) * 2.0 ** -23
    assert (np.abs(got - want) <= bound * want).all(), float((np.abs(got - want) / want).max() * 2 ** 23)


@pytest.mark.parametrize("form", [0, 1])
def test_both_forms_of_the_product_at_every_size(form):
    """The products above again, in a process that takes one-SM tiles (0) or two-SM tiles (1) whatever the size: single rows on two-SM
    tiles, rows of results that are not whole 16 bytes, every activation, more tiles than SMs on one-SM tiles."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, SYNAPTIK_CUDA_MX_PAIR=str(form))
    ran = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-k",
                          "(linear or product or same_bits or share_scales) and not every_size"], env=env, capture_output=True, text=True, timeout=600)
    assert ran.returncode == 0, ran.stdout[-3000:]


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("kind", KINDS)
def test_linear_activations_on_many_rows(ctx, kind, act):
    """More tiles than SMs, and rows of 16-bit results that are not whole 16 bytes."""
    check_linear(ctx, kind, (2100,), 64, 1100, act)


@pytest.mark.parametrize("act", ACTIVATIONS[1:])
def test_activation_gradient_of_every_held_value(ctx, act):
    """All codes under all scales.  In units of 2^-24: an exponential of -x is off by 4 + 2.35 x of itself, and by x per unit of
    its argument's rounding (none for x = |z| or 2 |z|, 1 for z^2 / 2, 4 for the tanh form's u); the divisions, polynomials and
    the other roundings by 24 of the sum of the slope's terms.  Below 2^-125 results leave the normal numbers."""
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(8, 32), (255, 1))
    codes[(codes & 127) == 127] = 0
    scales = np.zeros((8 * 255, 4), dtype=np.uint8)
    scales[:, 0] = np.repeat(np.arange(255), 8)
    z = ref.values(codes, scales, "mx8", 32)
    g = GraphBuilder()
    held, u = g.mx_feed("mx8", z.shape), g.feed(F32, z.shape)
    g.publish(g.mx_activation_gradient(act, held, u))
    got, = run_image(ctx, g, [codes, scales, np.ones(z.shape, dtype=np.float32)])
    want = ref.slope(act, z)
    a = np.minimum(np.abs(z), 120)
    zc = np.clip(z, -120, 120)
    u = np.abs(2 * ref.C * (zc + 0.044715 * zc ** 3))
    near = lambda x: np.exp(-x) / (1 + np.exp(-x)) ** 2         # noqa: E731
    x, roundings, terms = {"tanh": (2 * a, 0, want), "sigmoid": (a, 0, want), "silu": (a, 0, ref.sigmoid(zc) + a * near(a)),
                           "gelu_tanh": (u, 4, ref.sigmoid(np.copysign(u, zc)) + a * near(u) * 2 * ref.C * (1 + 3 * 0.044715 * a * a)),
                           "gelu": (a * a / 2, 1, ref.slope("gelu", zc) + 2 * a * np.exp(-a * a / 2) / np.sqrt(2 * np.pi))}[act]
    bound = 2.0 ** -24 * (4 + (2.35 + roundings) * x + 24) * np.abs(terms) + 2.0 ** -125
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    assert np.abs(got - want).max() <= 6 * 2.0 ** -24


@pytest.mark.parametrize("x_byte,w_byte", [(0, 227), (254, 0), (227, 0), (1, 200), (254, 20), (127, 127)])
def test_linear_scales_at_the_ends_of_their_range(ctx, x_byte, w_byte):
    """The least and the largest power of two as a scale, against one that brings the result back into range."""
    rng = np.random.default_rng(x_byte)
    m, n, k = 150, 140, 160
    held = []
    for rows, byte in ((m, x_byte), (n, w_byte)):
        codes, scales = random_held(rng, "mx4", (rows, k))
        held.append((codes, np.where(np.arange(scales.shape[1]) < k // 32, byte, 0).astype(np.uint8) + np.zeros_like(scales), (rows, k)))
    got = linear(ctx, "f32", *held, None, None)
    xv, wv = (ref.values(*h[:2], "mx4", k) for h in held)
    want, s = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    assert (np.abs(got - want) <= (k / 32 + 4) * 2.0 ** -23 * s + 2.0 ** -149).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_quantize_broadcast_views(ctx, kind, fmt):
    """EXPAND along rows, along columns and of a scalar: strides of zero."""
    rng = np.random.default_rng(3)
    for source, shape in [((1, 96), (50, 96)), ((50, 1), (50, 96)), ((1, 1), (7, 70)), ((3, 1, 40), (3, 9, 40)), ((3, 9, 1), (3, 9, 33)), ((), (5, 64))]:
        fed, exact = ref.stored(kind, mixed(rng, *source) if source else np.float32(2.7).reshape(()))
        g = GraphBuilder()
        held = g.mx_quantize(g.expand(g.feed(ref.STORAGE[kind], source), shape), fmt)
        g.publish(held.codes)
        g.publish(held.scales)
        codes, scales = run_image(ctx, g, [fed])
        want_codes, want_scales = ref.quantize(np.broadcast_to(exact, shape), fmt)
        assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes), (source, shape)


@pytest.mark.parametrize("exponent", [-100, -112, -118, -126, -140])
def test_weight_gradient_of_tiny_gradients(ctx, exponent):
    """What lies below 2^-133 in an element of a FLOAT32 gradient is lost, and nothing else."""
    rng = np.random.default_rng(-exponent)
    rows, k, n = 300, 300, 264
    held = ref.quantize((rng.standard_normal((rows, k)) * 2.0 ** 30).astype(np.float32), "mx8")
    up = np.ldexp(rng.standard_normal((rows, n)), exponent).astype(np.float32)
    x = ref.values(*held, "mx8", k)
    up64 = up.astype(np.float64)
    want, s = up64.T @ x, np.abs(up64).T @ np.abs(x)
    got = weight_gradient(ctx, "f32", held, (rows, k), up, n)
    bound = (rows / 16 * 4 + 4) * 2.0 ** -23 * s + 2.0 ** -133 * np.abs(x).sum(0) + 2.0 ** -149
    assert (np.abs(got - want) <= bound).all()
