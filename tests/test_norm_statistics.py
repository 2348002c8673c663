"""Mean and variance of group_norm to what the kernels' sums promise, far from zero and with values far from all others.

u = 2^-24; a group has the mean m, the standard deviation s and D = max |x - m|. A thread takes at most L = 64 values one after the other on the shapes
here. Every bound is for the worst case of its roundings.
* Mean. Rows sum the values themselves: 32 in a row, five shuffles, sixteen warps, and a factor; the other forms sum distances from the first value of a
  thread, which are at most 2 D, and then join the threads' means: up to 64 of a column, 16 parts of columns, five shuffles, eight blocks, three factors.
  Together (L + 2) u 2 D + 96 u (|m| + D).
* Variance. Rows square distances from the mean: 60 u relative. Distances from a thread's first value f: (L + 4) u of the sum of (x - f)^2, which over all
  threads is at most 2 (1 + L) times that of (x - m)^2, whatever the first values are: 2 (L + 4) (L + 1) u. Joining adds 96 u.
* Result: half of the variance's relative error times z, the mean's error times 1 / s, and beta - m / s rounded: 2 u |m| / s; four roundings of z.
A variance formed as E[x^2] - m^2 in fp32 is further off than that (the test on the CPU), and twenty times as wide a tolerance would not have shown it.
"""
import numpy as np
import pytest

U = 2.0 ** -24
L = 64
EPS = 1e-5
FORMS = ["rows_warp", "rows_block", "slab", "streamed", "strided"]
KINDS = ["plain", "mean 500", "mean 4000", "channel means", "outlier", "first outlier"]
CASES = [("rows_warp", (4, 512), 1), ("rows_warp", (5, 520), 1), ("rows_warp", (2500, 200), 2), ("rows_block", (3, 2048), 1), ("rows_block", (1300, 1030), 1)] + [
    (form, shape, groups) for form in FORMS[2:] for shape, groups in (((2, 40, 24, 24), 4), ((1, 64, 40, 41), 4), ((1, 16, 150, 200), 2))
    if form != "slab" or shape[2] * shape[3] < 2000]  # (the last one does not fit the shared memory of eight blocks)


def values(shape, groups, kind):
    rng = np.random.default_rng(51)
    x = rng.normal(0, 1, shape)
    if kind.startswith("mean"):
        x = x + float(kind.split()[1])
    elif kind == "channel means":
        x = x + rng.normal(0, 1000, (1, shape[1]) + (1,) * (len(shape) - 2))
    elif kind == "outlier":
        x.reshape(-1)[x.size // 3] = 1e5
    elif kind == "first outlier":
        x.reshape(shape[0], groups, -1)[:, :, 0] = -1e5
    return x.astype(np.float32)


def want(x, groups, rows):
    """(z in 64 bits, tolerance)"""
    t = x.astype(np.float64).reshape(x.shape[0], groups, -1)
    m = t.mean(2, keepdims=True)
    rstd = 1.0 / np.sqrt(t.var(2, keepdims=True) + float(np.float32(EPS)))
    far = np.abs(t - m).max(2, keepdims=True)
    z = (t - m) * rstd
    mean = (L + 2) * U * 2 * far + 96 * U * (np.abs(m) + far)
    variance = 60 * U if rows else 2 * (L + 4) * (L + 1) * U + 96 * U
    tol = mean * rstd + 0.5 * variance * np.abs(z) + 2 * U * np.abs(m) * rstd + 4 * U * np.abs(z)
    return z.reshape(x.shape), tol.reshape(x.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form,shape,groups", CASES)
def test_statistics(form, shape, groups, kind):
    from tpu_compiler_b200 import module
    x = values(shape, groups, kind)
    d = ",".join(map(str, shape))
    m = module(0)
    m.set_option("norm_form", 1 + FORMS.index(form))
    m.load_text("input name=x shape=%s dtype=FP32\ngroup_norm name=y in=x shape=%s dtype=FP32 groups=%d variance_epsilon=%g\n" % (d, d, groups, EPS), {})
    assert m.op_form("y")["form"] == form
    m.set_tensor("x", x)
    m.invoke()
    got = m.get_tensor("y").astype(np.float64)
    m.close()
    z, tol = want(x, groups, form.startswith("rows"))
    off = np.abs(got - z) / tol
    assert off.max() <= 1.0, "%g of the tolerance at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("form,shape,groups", [c for c in CASES if c[0] in ("rows_warp", "streamed")])
def test_tolerance_tells_a_difference_of_squares(form, shape, groups):
    """What the tolerance is for: two passes in fp32 lie within it, E[x^2] - m^2 does not."""
    for kind in ("mean 500", "mean 4000"):
        x = values(shape, groups, kind)
        z, tol = want(x, groups, form.startswith("rows"))
        t = x.reshape(shape[0], groups, -1)
        m = t.mean(2, keepdims=True, dtype=np.float32)
        good = (t - m) / np.sqrt(np.square(t - m).mean(2, keepdims=True, dtype=np.float32) + np.float32(EPS))
        assert (np.abs(good.reshape(x.shape) - z) <= tol).all()
        square = np.square(t).mean(2, keepdims=True, dtype=np.float32) - m * m
        bad = (t - m) / np.sqrt(np.maximum(square, 0) + np.float32(EPS))
        assert (np.abs(bad.reshape(x.shape) - z) > tol).any()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((64, 320, 8, 8), 32), ((5, 64, 33, 35), 8), ((300, 768), 1), ((2000, 768), 1)])
def test_an_image_by_itself_has_the_same_result(shape, groups):
    """Another number of images may take another form and another order of sums, never another result than those allow."""
    from tpu_compiler_b200 import module
    x = values(shape, groups, "plain")
    got = []
    for part in (x, x[3:4]):
        d = ",".join(map(str, part.shape))
        m = module(0)
        m.load_text("input name=x shape=%s dtype=FP32\ngroup_norm name=y in=x shape=%s dtype=FP32 groups=%d\n" % (d, d, groups), {})
        m.set_tensor("x", part)
        m.invoke()
        got.append(m.get_tensor("y").astype(np.float64))
        m.close()
    z, tol = want(x, groups, False)
    assert (np.abs(got[0] - z) <= tol).all()
    assert (np.abs(got[1] - z[3:4]) <= tol[3:4]).all()
    assert (np.abs(got[0][3:4] - got[1]) <= 2 * tol[3:4]).all()
