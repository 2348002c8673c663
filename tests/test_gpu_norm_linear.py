"""group_norm and fully_connected with activation / residual on the GPU against their definitions in 64 bits.

Tolerances. u = 2^-24 (fp32), h = half a step of the result's type: 2^-8 (BF16) or u (fp32), relative to the value.

group_norm, z = (x - mean) rstd: a partial sum takes at most L = 1024 values one after the other (more are joined as trees), so that
the mean is off by (L + 16) u A, A = max |x| of the group, or of |x - first value| plus two roundings of the mean itself; the variance by
2 (L + 16) u relative. With rstd this gives |dz| <= (L + 16) u A rstd + (L + 16) u |z|, then gamma and beta with a rounding each.
linear: K products summed in any order, each partial sum rounded or cut to 24 bits: K 2 u S, S = sum |x w| + |bias|.
The activations' slopes are at most 1.13; their own errors at most 2.5e-5 max(|v|, 1) (BF16) or 1e-6 max(|v|, 1) (fp32: 3.1e-7 of the
tail's polynomial, and products and exponentials of a few u).
"""
import numpy as np
import pytest

import oracle as O
from oracle import graph_runner
from tpu_compiler_b200 import graphs

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def M():
    from tpu_compiler_b200 import module
    return module


def cast(v, dtype):
    return O.bf16_round(np.asarray(v, np.float32)) if dtype == "BF16" else np.asarray(v, np.float32)


def dims(shape):
    return ",".join(str(int(d)) for d in shape)


def own_error(v, dtype):
    return (2.5e-5 if dtype == "BF16" else 1e-6) * np.maximum(np.abs(v), 1.0)


def assert_close(got, want, tol, what=""):
    got = got.astype(np.float64)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g of the tolerance, first at %s: got %r want %r" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / tol), np.unravel_index(np.flatnonzero(bad)[0], bad.shape),
        got[bad][:4], want[bad][:4])


def norm_want(x, groups, gamma, beta, eps, act, dtype):
    """(value in 64 bits, tolerance)"""
    n, c = x.shape[0], (x.shape[1] if x.ndim > 1 else 1)
    t = x.astype(np.float64).reshape(n, groups, -1)
    big = np.abs(t).max(2, keepdims=True)
    rstd = 1.0 / np.sqrt(t.var(2, keepdims=True) + float(np.float32(eps)))
    z = (t - t.mean(2, keepdims=True)) * rstd
    dz = (1040 * U * (big * rstd + np.abs(z))).reshape(n, c, -1)
    z = z.reshape(n, c, -1)
    ga = (np.ones(c) if gamma is None else gamma.astype(np.float64))[None, :, None]
    be = (np.zeros(c) if beta is None else beta.astype(np.float64))[None, :, None]
    v = z * ga + be
    y = O.activation64(v, act)
    h = 2.0 ** -8 if dtype == "BF16" else U
    tol = h * np.abs(y) + 1.13 * (dz * np.abs(ga) + 3 * U * (np.abs(z * ga) + np.abs(be))) + own_error(v, dtype)
    return y.reshape(x.shape), tol.reshape(x.shape)


def run_norm(M, x, groups, gamma, beta, eps=1e-5, act="none", dtype="BF16", options=(), form=None):
    w, ins = {}, ["x"]
    for name, v in (("ga", gamma), ("be", beta)):
        ins.append("-" if v is None else name)
        if v is not None:
            w[name] = v
    m = M(0)
    for k, v in options:
        m.set_option(k, v)
    m.load_text("input name=x shape=%s dtype=%s\ngroup_norm name=y in=%s shape=%s dtype=%s groups=%d variance_epsilon=%g activation=%s\n" % (
        dims(x.shape), dtype, ",".join(ins), dims(x.shape), dtype, groups, eps, act), w)
    if form is not None:
        form.update(m.op_form("y"))
    m.set_tensor("x", x)
    m.invoke()
    got = m.get_tensor("y")
    m.close()
    return got


NORM_CASES = [
    # shape, groups: rows
    ((1, 1), 1), ((1, 16), 1), ((3, 33), 1), ((3, 33), 11), ((5, 1024), 1), ((2, 8192), 1), ((300, 100), 1), ((257, 48), 3),
    ((7, 1280), 32), ((2, 20000), 1), ((2049, 24), 1), ((4, 640), 640), ((7,), 1), ((3, 4099), 1), ((1000, 520), 2),
    # images
    ((2, 320, 16, 16), 32), ((1, 64, 1, 1), 4), ((2, 33, 5, 7), 11), ((1, 34, 9, 9), 2), ((3, 6, 1, 5), 6), ((2, 1280, 8, 8), 32),
    ((1, 128, 96, 97), 32), ((1, 17, 64, 64), 1), ((5, 8, 3, 3), 8), ((2, 96, 31, 33), 1), ((1, 640, 33, 1), 32), ((1, 2048, 7, 7), 32),
    ((1, 40, 130, 300), 4), ((9, 24, 40, 40), 24), ((1, 4100, 3, 3), 4), ((1, 1025, 6, 5), 1), ((2, 50, 20), 10),
]


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("k", range(len(NORM_CASES)))
def test_group_norm(M, k, dtype):
    shape, groups = NORM_CASES[k]
    rng = np.random.default_rng(100 + k)
    c = shape[1] if len(shape) > 1 else 1
    per = [1, c] + [1] * (len(shape) - 2) if len(shape) > 1 else [1]
    x = cast(rng.normal(0, 1, shape) * np.exp(0.5 * rng.normal(0, 1, c)).reshape(per) + rng.normal(0, 1, c).reshape(per), dtype)
    gamma, beta = rng.normal(1, 0.3, c).astype(np.float32), rng.normal(0, 0.3, c).astype(np.float32)
    act = ACTS[k % 5]
    want, tol = norm_want(x, groups, gamma, beta, 1e-5, act, dtype)
    assert_close(run_norm(M, x, groups, gamma, beta, act=act, dtype=dtype), want, tol, "%s %d %s %s" % (shape, groups, act, dtype))


NORM_FORMS = ["rows_warp", "rows_block", "slab", "streamed", "strided"]


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("form,shape,groups", [(f, s, g) for s, g, forms in [
    ((37, 200), 1, "rows_warp rows_block slab streamed strided"), ((37, 203), 1, "rows_warp rows_block slab streamed strided"),
    ((5, 640), 16, "rows_warp rows_block slab streamed strided"), ((130, 1000), 1, "rows_warp rows_block slab streamed strided"),
    ((3, 6001), 1, "rows_block strided"), ((2, 33, 5, 7), 11, "slab streamed strided"), ((2, 64, 40, 41), 8, "slab streamed strided"),
    ((2, 40, 40, 41), 4, "slab streamed strided"), ((1, 17, 30, 100), 1, "slab streamed strided"), ((3, 96, 3, 1), 96, "slab streamed strided"),
    ((1, 512, 60, 77), 32, "slab streamed strided"), ((4, 2048, 2, 2), 32, "slab streamed strided"), ((1, 64, 200, 203), 2, "streamed strided"),
    ((1, 4100, 3, 3), 4, "strided")] for f in forms.split()])
def test_group_norm_forms(M, form, shape, groups, dtype):
    """Every form on every tensor that it can take, whatever the rule by size would choose."""
    rng = np.random.default_rng(30)
    per = [1, shape[1]] + [1] * (len(shape) - 2)
    x = cast(rng.normal(0, 1, shape) * np.exp(rng.normal(0, 0.5, per)) + rng.normal(0, 1, per), dtype)
    gamma, beta = rng.normal(1, 0.3, shape[1]).astype(np.float32), rng.normal(0, 0.3, shape[1]).astype(np.float32)
    want, tol = norm_want(x, groups, gamma, beta, 1e-5, "silu", dtype)
    took = {}
    options = [("norm_form", 1 + NORM_FORMS.index(form))]
    got = run_norm(M, x, groups, gamma, beta, act="silu", dtype=dtype, options=options, form=took)
    assert took["form"] == form
    assert_close(got, want, tol)
    assert np.array_equal(got, run_norm(M, x, groups, gamma, beta, act="silu", dtype=dtype, options=options))
    hard = cast(rng.normal(0, 1, shape) + 500.0, dtype)  # a mean far from zero
    want, tol = norm_want(hard, groups, None, None, 1e-5, "none", dtype)
    assert_close(run_norm(M, hard, groups, None, None, dtype=dtype, options=options), want, tol)


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("form,shape,groups", [
    ("slab", (1, 320, 96, 100), 32), ("slab", (1, 96, 70, 111), 8), ("slab", (2, 64, 90, 90), 2), ("slab", (150, 64, 20, 20), 32),  # most of shared memory
    ("slab", (2, 1500, 9, 9), 1),  # wide groups
    ("streamed", (1, 512, 40, 60), 512), ("streamed", (1, 2048, 20, 21), 2048), ("streamed", (1, 2100, 20, 21), 300),  # many groups per row
    ("strided", (1, 524400, 2, 1), 8)])  # more channels than the others divide
def test_group_norm_at_its_limits(M, form, shape, groups, dtype):
    rng = np.random.default_rng(31)
    x = cast(rng.normal(0, 1, shape) + rng.normal(0, 1, (1, shape[1], 1, 1)), dtype)
    gamma, beta = rng.normal(1, 0.3, shape[1]).astype(np.float32), rng.normal(0, 0.3, shape[1]).astype(np.float32)
    want, tol = norm_want(x, groups, gamma, beta, 1e-5, "gelu", dtype)
    took = {}
    options = [("norm_form", 0 if form == "strided" else 1 + NORM_FORMS.index(form))]
    assert_close(run_norm(M, x, groups, gamma, beta, act="gelu", dtype=dtype, options=options, form=took), want, tol)
    assert took["form"] == form


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((6, 256), 1), ((2, 64, 6, 6), 4)])
def test_group_norm_activations_far_out(M, shape, groups, act, dtype):
    """Pre-activations from -40 to 40: tails without cancellation, nothing overflows."""
    rng = np.random.default_rng(5)
    x = cast(rng.normal(0, 1, shape), dtype)
    gamma, beta = rng.uniform(-15, 15, shape[1]).astype(np.float32), rng.uniform(-5, 5, shape[1]).astype(np.float32)
    want, tol = norm_want(x, groups, gamma, beta, 1e-5, act, dtype)
    assert_close(run_norm(M, x, groups, gamma, beta, act=act, dtype=dtype), want, tol)


@pytest.mark.parametrize("shape,groups", [((4, 512), 1), ((1, 64, 40, 41), 4), ((2, 40, 24, 24), 4), ((1, 16, 300, 400), 2)])
@pytest.mark.parametrize("kind", ["constant", "mean", "outlier", "channel means", "first outlier"])
def test_group_norm_hard_statistics(M, shape, groups, kind):
    """A variance of zero, means thousands of times the spread, one value far from all others (the first of the tensor, too)."""
    rng = np.random.default_rng(11)
    x = rng.normal(0, 1, shape)
    if kind == "constant":
        x = np.full(shape, 3.25)
    elif kind == "mean":
        x = x + 4000.0
    elif kind == "channel means":
        x = x + rng.normal(0, 1000, (1, shape[1]) + (1,) * (len(shape) - 2))
    elif kind == "outlier":
        x.reshape(-1)[x.size // 3] = 1e5
    else:
        x.reshape(shape[0], groups, -1)[:, :, 0] = -1e5
    for dtype in ("FP32", "BF16"):
        xc = cast(x, dtype)
        want, tol = norm_want(xc, groups, None, None, 1e-5, "none", dtype)
        assert_close(run_norm(M, xc, groups, None, None, dtype=dtype), want, tol, kind + " " + dtype)


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("shape,groups", [((3, 96), 3), ((3, 96), 1), ((2, 48, 5, 5), 6), ((1, 64, 70, 70), 4)])
def test_group_norm_keeps_groups_apart(M, shape, groups, dtype):
    """NaN and infinity in one group reach no other group."""
    rng = np.random.default_rng(12)
    x = cast(rng.normal(0, 1, shape), dtype)
    clean = run_norm(M, x, groups, None, None, act="silu", dtype=dtype)
    poisoned = x.copy()
    p = poisoned.reshape(shape[0], groups, -1)
    p[0, 0, 1] = np.nan
    p[-1, -1, -1] = np.inf
    got = run_norm(M, poisoned, groups, None, None, act="silu", dtype=dtype).reshape(shape[0], groups, -1)
    clean = clean.reshape(shape[0], groups, -1)
    other = np.ones((shape[0], groups), bool)
    other[0, 0] = other[-1, -1] = False
    assert np.array_equal(got[other], clean[other])
    assert np.isnan(got[0, 0]).all() and np.isnan(got[-1, -1]).all()  # inf - inf in the second


def test_group_norm_result_does_not_depend_on_the_batch(M):
    rng = np.random.default_rng(13)
    for shape, groups in (((64, 320, 8, 8), 32), ((5, 64, 33, 35), 8), ((300, 768), 1)):
        x = cast(rng.normal(0, 1, shape), "BF16")
        y = run_norm(M, x, groups, None, None)
        one, tol = norm_want(x[3:4], groups, None, None, 1e-5, "none", "BF16")
        assert_close(y[3:4], one, tol)
        assert np.array_equal(y, run_norm(M, x, groups, None, None))  # and is the same every time


def linear_want(x, w, bias, act, res, dtype):
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    v = x64 @ w64.T + b
    s = np.abs(x64) @ np.abs(w64).T + np.abs(b)
    y = O.activation64(v, act)
    tol = 1.13 * 2 * U * (x.shape[1] + 2) * s + own_error(v, dtype)
    if res is not None:
        y = y + res.astype(np.float64)
        tol = tol + U * np.abs(y)
    return y, tol + (2.0 ** -8 if dtype == "BF16" else U) * np.abs(y)


def run_linear(M, x, w, bias, act=None, res=None, dtype="BF16", options=(), form=None):
    m, n = x.shape[0], w.shape[0]
    text = "input name=x shape=%s dtype=%s\n" % (dims(x.shape), dtype)
    weights = {"f": w.reshape(n, -1)}
    if bias is not None:
        weights["b"] = bias
    if res is not None:
        text += "input name=r shape=%d,%d dtype=%s\n" % (m, n, dtype)
    text += "fully_connected name=y in=x,f,%s,-,-,-,-,%s shape=%d,%d dtype=%s%s\n" % (
        "-" if bias is None else "b", "-" if res is None else "r", m, n, dtype, "" if act is None else " activation=" + act)
    mod = M(0)
    for k, v in options:
        mod.set_option(k, v)
    mod.load_text(text, weights)
    if form is not None:
        form.update(mod.op_form("y"))
    mod.set_tensor("x", x)
    if res is not None:
        mod.set_tensor("r", res)
    mod.invoke()
    got = mod.get_tensor("y")
    mod.close()
    return got


LINEAR_CASES = [
    # m, k, n
    (1, 1, 1), (1, 16, 16), (2, 17, 15), (3, 33, 100), (1, 1000, 300), (1, 4096, 512), (17, 1000, 130), (64, 64, 64), (128, 256, 128),
    (129, 130, 257), (127, 1024, 48), (33, 5000, 40), (300, 96, 1000), (256, 512, 256), (1025, 200, 72), (7, 64, 5000), (515, 700, 530),
    (2048, 64, 16), (1, 8192, 33), (90, 2048, 2048), (2304, 320, 776), (4, 40, 16384),
]


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("k", range(len(LINEAR_CASES)))
def test_linear(M, k, dtype):
    m, kk, n = LINEAR_CASES[k]
    rng = np.random.default_rng(200 + k)
    x, w = cast(rng.normal(0, 1, (m, kk)), dtype), cast(rng.normal(0, kk ** -0.5, (n, kk)), dtype)
    bias = rng.normal(0, 0.3, n).astype(np.float32) if k % 4 != 3 else None
    res = cast(rng.normal(0, 1, (m, n)), dtype) if k % 2 else None
    act = ACTS[k % 5]
    want, tol = linear_want(x, w, bias, act, res, dtype)
    assert_close(run_linear(M, x, w, bias, act, res, dtype), want, tol, "%s %s %s" % (LINEAR_CASES[k], act, dtype))


@pytest.mark.parametrize("tiles", [1016, 1032, 1064, 1128, 1256, 2016, 2064, 3048, 4112, 4256, 5080, 7128, 8016, 8128, 8256, 10064, 10128, 10192, 10256])
@pytest.mark.parametrize("m,k,n", [(1, 600, 300), (33, 1000, 130), (200, 520, 272), (300, 4160, 530), (515, 64, 1040)])
def test_linear_tensor_core_forms(M, m, k, n, tiles):
    """Every form of the tensor-core kernels on every size, whatever the rule by size would take."""
    rng = np.random.default_rng(m + n)
    x, w = cast(rng.normal(0, 1, (m, k)), "BF16"), cast(rng.normal(0, k ** -0.5, (n, k)), "BF16")
    bias, res = rng.normal(0, 0.3, n).astype(np.float32), cast(rng.normal(0, 1, (m, n)), "BF16")
    want, tol = linear_want(x, w, bias, "silu", res, "BF16")
    form = {}
    got = run_linear(M, x, w, bias, "silu", res, options=[("linear_tiles", tiles)], form=form)
    pair = tiles >= 10000
    assert form == {"tiles": "pair" if pair else "cluster", "channels": tiles % 1000, "split_k": 1 if pair else min(tiles // 1000, (k + 63) // 64)}
    assert_close(got, want, tol)
    assert np.array_equal(got, run_linear(M, x, w, bias, "silu", res, options=[("linear_tiles", tiles)]))


@pytest.mark.parametrize("rows", [8, 16, 24, 32, 40, 48, 56])
@pytest.mark.parametrize("split", [1, 2, 3, 8])
@pytest.mark.parametrize("m,k,n", [(1, 600, 300), (77, 333, 130), (200, 20, 71)])
def test_linear_fp32_forms(M, m, k, n, split, rows):
    rng = np.random.default_rng(m + n)
    x, w = cast(rng.normal(0, 1, (m, k)), "FP32"), cast(rng.normal(0, k ** -0.5, (n, k)), "FP32")
    bias, res = rng.normal(0, 0.3, n).astype(np.float32), cast(rng.normal(0, 1, (m, n)), "FP32")
    want, tol = linear_want(x, w, bias, "gelu_tanh", res, "FP32")
    form, options = {}, [("linear_tiles", 1000 * split + rows)]
    got = run_linear(M, x, w, bias, "gelu_tanh", res, "FP32", options=options, form=form)
    assert form == {"tiles": "direct", "rows": rows, "split_k": min(split, (k + 15) // 16)}
    assert_close(got, want, tol)
    assert np.array_equal(got, run_linear(M, x, w, bias, "gelu_tanh", res, "FP32", options=options))


@pytest.mark.parametrize("tiles", [1128, 4064, 10064])
def test_linear_bounded_wait_runs_out(M, tiles):
    """A hand-over that never comes: the launch ends with a status, the interpreter stays usable."""
    from tpu_compiler_b200 import TpucbError
    rng = np.random.default_rng(19)
    m, k, n = 700, 512, 2048  # 96 tiles of a pair: some do the third, which needs an accumulator back
    n = 8192 if tiles >= 10000 else n
    x, w = cast(rng.normal(0, 1, (m, k)), "BF16"), cast(rng.normal(0, k ** -0.5, (n, k)), "BF16")
    text = "input name=x shape=%d,%d dtype=BF16\nfully_connected name=y in=x,f shape=%d,%d dtype=BF16 activation=relu\n" % (m, k, m, n)
    mod = M(0)
    mod.set_option("linear_tiles", tiles)
    for rounds in (4, 0):
        mod.set_option("selftest_lost_arrival", rounds)
        mod.load_text(text, {"f": w})
        mod.set_tensor("x", x)
        if rounds:
            for _ in range(2):
                with pytest.raises(TpucbError, match="bounded wait"):
                    mod.invoke()
        else:
            mod.invoke()
    want, tol = linear_want(x, w, None, "relu", None, "BF16")
    assert_close(mod.get_tensor("y"), want, tol)
    mod.close()


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(3, 40), (200, 144)])
def test_linear_activations_far_out(M, m, n, act, dtype):
    rng = np.random.default_rng(15)
    x, w = cast(rng.normal(0, 1, (m, 64)), dtype), cast(rng.normal(0, 1.5, (n, 64)), dtype)
    bias, res = rng.uniform(-10, 10, n).astype(np.float32), cast(rng.normal(0, 1, (m, n)), dtype)
    want, tol = linear_want(x, w, bias, act, res, dtype)
    assert_close(run_linear(M, x, w, bias, act, res, dtype), want, tol)


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
def test_linear_of_an_image_and_forms_of_the_line(M, dtype):
    """Rows that are images (K runs over channels, then pixels, as the filter's), do_relu with a residual, no bias, the input as residual."""
    rng = np.random.default_rng(16)
    x, w = cast(rng.normal(0, 1, (5, 19, 3, 4)), dtype), cast(rng.normal(0, 0.1, (30, 228)), dtype)
    want, tol = linear_want(x.reshape(5, 228), w, None, "gelu", None, dtype)
    assert_close(run_linear(M, x, w, None, "gelu", None, dtype), want, tol)
    m = M(0)
    w, b = cast(rng.normal(0, 0.1, (48, 48)), dtype), rng.normal(0, 1, 48).astype(np.float32)
    m.load_text("input name=x shape=9,48 dtype=%s\nfully_connected name=y in=x,f,b,-,-,-,-,x shape=9,48 dtype=%s do_relu=1\n" % (dtype, dtype),
                {"f": w, "b": b})
    x = cast(rng.normal(0, 1, (9, 48)), dtype)
    m.set_tensor("x", x)
    m.invoke()
    want, tol = linear_want(x, w, b, "relu", x, dtype)
    assert_close(m.get_tensor("y"), want, tol)
    m.close()


@pytest.mark.parametrize("m", [1, 40, 700])
def test_linear_rows_do_not_mix(M, m):
    """An infinity in one row stays in it."""
    rng = np.random.default_rng(17)
    x, w = cast(rng.normal(0, 1, (m, 200)), "BF16"), cast(rng.normal(0, 0.1, (100, 200)), "BF16")
    clean = run_linear(M, x, w, None, "none")
    poisoned = x.copy()
    poisoned[m // 2, 7] = np.inf
    got = run_linear(M, poisoned, w, None, "none")
    keep = np.arange(m) != m // 2
    assert np.array_equal(got[keep], clean[keep])
    assert np.array_equal(got[m // 2], np.copysign(np.inf, w[:, 7]))


def blocks(dtype, rows=70, n=2, hw=12):
    """A residual block around convolutions and a feed-forward block, as one module."""
    rng = np.random.default_rng(21)
    b = graphs.GraphBuilder(21, simulate=False)
    cw = lambda name, *s: b.weight(name, cast(rng.normal(0, (np.prod(s[1:])) ** -0.5, s), dtype))  # noqa: E731
    fw = lambda name, k, mean=0.0: b.weight(name, (mean + rng.normal(0, 0.2, k)).astype(np.float32))  # noqa: E731
    b.op("input", "img", [], (n, 64, hw, hw), dtype)
    src = "img"
    for i in (1, 2):
        b.op("group_norm", "n%d" % i, [src, fw("ng%d" % i, 64, 1.0), fw("nb%d" % i, 64)], (n, 64, hw, hw), dtype, groups=8, activation="silu")
        src = b.op("conv_2d", "c%d" % i, ["n%d" % i, cw("cf%d" % i, 64, 64, 3, 3), fw("cb%d" % i, 64)], (n, 64, hw, hw), dtype, kh=3, kw=3, sh=1,
                   sw=1, pt=1, pb=1, pl=1, pr=1, dh=1, dw=1, g=1, do_relu=0, with_bias=1)
    b.op("eltwise_add", "sum", ["img", "c2"], (n, 64, hw, hw), dtype, do_relu=0)
    b.op("input", "tok", [], (rows, 128), dtype)
    b.op("group_norm", "ln", ["tok", fw("lg", 128, 1.0), fw("lb", 128)], (rows, 128), dtype, groups=1)
    b.op("fully_connected", "up", ["ln", cw("uf", 512, 128), fw("ub", 512)], (rows, 512), dtype, activation="gelu")
    b.op("fully_connected", "down", ["up", cw("df", 128, 512), fw("db", 128), "", "", "", "", "tok"], (rows, 128), dtype)
    return b


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("graph", [0, 1])
def test_blocks_together(M, dtype, graph):
    """Each op against the oracle on the tensors that the GPU gave it, launched repeatedly as a graph and op by op."""
    b = blocks(dtype)
    rng = np.random.default_rng(22)
    m = M(0)
    m.set_option("cuda_graph", graph)
    m.load_text(b.text(), b.weights)
    assert sorted(m.get_output_details()) == ["down", "sum"]
    first = None
    for step in range(3):
        x = {"img": cast(rng.normal(0, 1, (2, 64, 12, 12)), dtype), "tok": cast(rng.normal(0, 1, (70, 128)), dtype)} if step < 2 else first[0]
        for name, v in x.items():
            m.set_tensor(name, v)
        m.launch()
        m.launch()
        m.sync()
        t = m.get_all_tensor()
        W = b.weights
        for name, src, g, ga, be, act in (("n1", "img", 8, "ng1", "nb1", "silu"), ("n2", "c1", 8, "ng2", "nb2", "silu"), ("ln", "tok", 1, "lg", "lb", "none")):
            want, tol = norm_want(t[src], g, W[ga], W[be], 1e-5, act, dtype)
            assert_close(t[name], want, tol, name)
        want, tol = linear_want(t["ln"], W["uf"], W["ub"], "gelu", None, dtype)
        assert_close(t["up"], want, tol, "up")
        want, tol = linear_want(t["up"], W["df"], W["db"], "none", t["tok"], dtype)
        assert_close(t["down"], want, tol, "down")
        if first is None:
            first = (x, t)
    for name in t:
        assert np.array_equal(t[name], first[1][name]), name
    m.close()


def test_two_modules_in_flight_and_single_ops(M):
    """Two modules with work in flight at once, each on its stream; and the ops as handles of their own."""
    b = blocks("BF16")
    rng = np.random.default_rng(23)
    data = [{"img": cast(rng.normal(0, 1, (2, 64, 12, 12)), "BF16"), "tok": cast(rng.normal(0, 1, (70, 128)), "BF16")} for _ in range(2)]
    alone, mods = [], [M(0), M(0)]
    for m, d in zip(mods, data):
        m.load_text(b.text(), b.weights)
        for name, v in d.items():
            m.set_tensor(name, v)
        m.invoke()
        alone.append(m.get_all_tensor())
    for _ in range(20):
        for m in mods:
            m.launch()
    for m, want in zip(mods, alone):
        m.sync()
        got = m.get_all_tensor()
        for name in want:
            assert np.array_equal(got[name], want[name]), name
        m.close()
    m = M(0)
    m.set_weights(b.weights)
    ops = [m.create_op(line) for line in b.text().splitlines()]
    for name, v in data[0].items():
        m.set_tensor(name, v)
    for op in ops:
        op.invoke()
    by = {op.name: op for op in ops}
    assert by["n1"].op_type == "group_norm" and by["up"].datatype == "BF16" and by["down"].shape == [70, 128]
    for name in ("n1", "ln", "up", "down"):
        assert np.array_equal(by[name].get_tensor(), alone[0][name]), name
    m.close()


def test_batch_slots(M):
    """max_batch_size = 3: a launch covers all slots, which do not interact."""
    b = blocks("BF16", rows=5, n=1)
    rng = np.random.default_rng(24)
    m = M(0, 3)
    m.load_text(b.text(), b.weights)
    img, tok = cast(rng.normal(0, 1, (3, 64, 12, 12)), "BF16"), cast(rng.normal(0, 1, (15, 128)), "BF16")
    m.set_tensor("img", img)
    m.set_tensor("tok", tok)
    m.fast_invoke_all_batch()
    W = b.weights
    for slot in range(3):
        want, tol = norm_want(img[slot:slot + 1], 8, W["ng1"], W["nb1"], 1e-5, "silu", "BF16")
        assert_close(m.get_tensor("n1", slot), want, tol)
        up, ln = m.get_tensor("up", slot), m.get_tensor("ln", slot)
        want, tol = linear_want(ln, W["uf"], W["ub"], "gelu", None, "BF16")
        assert_close(up, want, tol)
        want, tol = linear_want(up, W["df"], W["db"], "none", tok[slot * 5:slot * 5 + 5], "BF16")
        assert_close(m.get_tensor("down", slot), want, tol)
    m.close()


def test_calibration_of_a_graph_with_these_ops(M):
    """The fp32 forward and its statistics run over them."""
    from tpu_compiler_b200.calibration import ActivationCalibrator
    b = blocks("FP32")
    lines = [ln for ln in b.text().splitlines() if " name=tok " not in ln and "name=ln" not in ln and "name=up" not in ln and "name=down" not in ln]
    m = M(0)
    m.load_text("\n".join(lines) + "\n", b.weights)
    x = np.random.default_rng(25).normal(0, 1, (2, 64, 12, 12)).astype(np.float32)
    thresholds, stats = ActivationCalibrator(m, lambda: iter([x])).run()
    ref = graph_runner.run("\n".join(lines), b.weights, {"img": x})
    for name in ("n1", "n2"):
        lo, hi = ref[name].min(), ref[name].max()
        got = np.asarray(stats[name], np.float64).reshape(-1)
        assert thresholds[name] > 0
        assert np.abs(got[:2] - [lo, hi]).max() <= 1e-4 * max(abs(lo), abs(hi))  # the fp32 path's tolerance
    m.close()


def test_refusals_reach_the_caller(M):
    from tpu_compiler_b200 import TpucbError
    m = M(0)
    w = {"g": np.ones(48, np.float32), "f": np.zeros((20, 48), np.float32)}
    head = "input name=x shape=2,48 dtype=BF16\n"
    for line, why in (("group_norm name=y in=x,g,- shape=2,48 dtype=BF16 groups=5", "does not divide"),
                      ("group_norm name=y in=x,f,- shape=2,48 dtype=BF16 groups=4", "960 values, expected 48"),
                      ("group_norm name=y in=lost,g,- shape=2,48 dtype=BF16 groups=4", "not found"),
                      ("fully_connected name=y in=x,f,- shape=2,20 dtype=BF16 activation=tanh", "is none of"),
                      ("fully_connected name=y in=x,f,-,-,-,-,-,x shape=2,20 dtype=BF16", "residual x must be"),
                      ("fully_connected name=y in=x,f,-,-,-,-,-,lost shape=2,20 dtype=BF16", "not found")):
        with pytest.raises(TpucbError, match=why):
            m.load_text(head + line + "\n", w)
    m.load_text(head + "group_norm name=y in=x,g,- shape=2,48 dtype=BF16 groups=4\n", w)
    m.set_tensor("x", np.ones((2, 48), np.float32))
    m.invoke()
    assert (m.get_tensor("y") == 0).all()
    m.close()


@pytest.mark.parametrize("dtype,bound", [("BF16", "tensor"), ("FP32", "hbm")])
def test_op_info(M, dtype, bound):
    """What a module says of these ops to who accounts for its time."""
    m = M(0)
    m.load_text("input name=x shape=4,64 dtype=%s\ngroup_norm name=z in=x shape=4,64 dtype=%s groups=1\n"
                "fully_connected name=y in=z,f shape=4,32 dtype=%s activation=silu\n" % (dtype, dtype, dtype),
                {"f": np.ones((32, 64), np.float32)})
    z, y = [i for i in m.op_info if i["name"] in ("y", "z")][:2]
    size = 2 if dtype == "BF16" else 4
    assert (z["type"], z["bound"], z["bytes"]) == ("group_norm", "hbm", 2 * 4 * 64 * size + 8 * 64)
    assert (y["type"], y["bound"], y["ops"]) == ("fully_connected", bound, 2 * 4 * 64 * 32)
    m.close()


@pytest.mark.parametrize("dtype,n,tiles", [("BF16", 20, 1), ("BF16", 20, 4032), ("BF16", 200, 10064), ("BF16", 37, 10128), ("BF16", 17, 1128), ("FP32", 18, 1), ("FP32", 21, 2008)])
def test_linear_infinities_stay_infinities(M, dtype, n, tiles):
    """An infinite value of a row gives infinite sums, in the next product too: what lies behind the last channel adds no NaN to them."""
    rng = np.random.default_rng(41)
    x = cast(rng.uniform(1, 2, (300, 48)), dtype)
    x[1, 3] = np.inf
    f, f2 = (cast(rng.uniform(0.5, 1, s), dtype) for s in ((n, 48), (9, n)))
    m = M(0)
    m.set_option("linear_tiles", tiles)
    m.load_text("input name=x shape=300,48 dtype=%s\nfully_connected name=h in=x,f shape=300,%d dtype=%s activation=relu\n"
                "fully_connected name=y in=h,f2 shape=300,9 dtype=%s activation=silu\n" % (dtype, n, dtype, dtype), {"f": f, "f2": f2})
    m.set_tensor("x", x)
    m.invoke()
    for name in ("h", "y"):
        got = m.get_tensor(name)
        assert np.isposinf(got[1]).all() and np.isfinite(np.delete(got, 1, 0)).all()
    m.close()
