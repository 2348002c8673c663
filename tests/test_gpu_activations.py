"""The activations of group_norm and of fully_connected over the whole range of their argument, against 64 bits.

Arguments are exact: with gamma = 0 a normalised value is beta, with weights of zero a product is its bias, and with one weight of one it is x.

Tolerances, relative to the value. u = 2^-24; h, the rounding of the result: 2^-8 (BF16) or u (fp32). Of the instructions, the PTX manual
gives 2^-22 = 4 u for ex2.approx and one unit in the last place, 2 u, for rcp.approx.
* v / (1 + 2^t) by one reciprocal for two values: 4 u, 2 u, and five roundings (the sum, the product of two denominators, its share of the
  reciprocal, v times it, and the residual's sum): 11 u; t itself is off by its constants and products, 2 u |t| (SiLU) or 4 u |t| (tanh GELU), which
  ln 2 carries into 2^t. fp32: from t = 60 on the value may count as zero: what is lost is below 2^-60 |v|. BF16: 2^-61 is taken from the quotient.
* |v| Q(|v|) = |v| 2^x P(t), x = -v^2 / 2 log2 e: 4 u of the exponential, 3 u |x| ln 2 = 1.5 u v^2 of its argument, 5 u of t = 1 / (1 + 0.35 |v|), which
  are 12 u of P (|t P' / P| < 2.3 up to |v| = 14), 16 u of P's eight steps (its terms add up to less than 1.9 times its value), two products, and P's
  fit, 3.1e-7 (fp32) or 2.4e-5 (BF16): 38 u with some room. Positive v: max(v, 0) minus that in one multiply-add.
Below 2^-126 the exponential is flushed to zero.
"""
from math import erfc, log, pi, sqrt

import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
FORMS = {"rows_warp": (1, (6, 256), 1), "rows_block": (2, (3, 2048), 1), "slab": (3, (2, 64, 6, 6), 4), "slab, odd groups": (3, (2, 60, 6, 6), 4),
         "streamed": (4, (1, 64, 40, 41), 4), "strided": (5, (1, 34, 9, 9), 2)}


@pytest.fixture(scope="module")
def M():
    from tpu_compiler_b200 import module
    return module


def value_and_tolerance(v, act, dtype):
    v = np.asarray(v, np.float32).astype(np.float64)
    h = 2.0 ** -8 if dtype == "BF16" else U
    with np.errstate(over="ignore", invalid="ignore"):
        if act == "none":
            y, own = v, 0.0 * v
        elif act == "relu":
            y = np.where(v < 0, 0.0, v)
            own = 0.0 * v
        elif act == "gelu":
            tail = 0.5 * np.vectorize(erfc, otypes=[np.float64])(np.abs(v) / sqrt(2.0)) * np.abs(v)  # (NaN at infinity)
            y = np.where(np.isposinf(v), v, np.maximum(v, 0.0) - tail)
            own = (38 * U + 1.5 * U * v * v + (2.4e-5 if dtype == "BF16" else 3.1e-7)) * tail + 2.0 ** -120
        else:
            t = -v / log(2.0) if act == "silu" else -2.0 * sqrt(2.0 / pi) * (v + 0.044715 * v ** 3) / log(2.0)
            y = v / (1.0 + np.exp2(t))
            own = (11 + (2 if act == "silu" else 4) * log(2.0) * np.abs(t)) * U * np.abs(y)
            own = own + (2.0 ** -61 if dtype == "BF16" else np.where(t >= 59.9, 2.0 ** -59.9, 0.0)) * np.abs(v)
        y = np.where(np.isnan(v), np.nan, y)
        return y, np.where(np.isfinite(y), own + h * np.abs(y), 0.0)


def check(got, v, act, dtype):
    want, tol = value_and_tolerance(v, act, dtype)
    want, tol = np.broadcast_to(want, got.shape), np.broadcast_to(tol, got.shape)
    v = np.broadcast_to(v, got.shape)
    got = got.astype(np.float64)
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    assert not bad.any(), "%d of %d: f(%r) = %r, want %r" % (bad.sum(), bad.size, v[bad][:6], got[bad][:6], want[bad][:6])


def arguments(n, far):
    """n fp32 values: from -45 to 45 densely, or over the type's whole range with infinities and a NaN between ordinary ones."""
    rng = np.random.default_rng(7)
    if not far:
        v = rng.uniform(-45, 45, n)
        v[::3] = rng.uniform(-9, 3, v[::3].size)
        v[1::7] = rng.uniform(-14, -8, v[1::7].size)
        return v.astype(np.float32)
    v = rng.normal(0, 2, n)
    hard = [-41, -42, -45, -60, -88, -104, -1e3, -1e10, -1e15, -1e20, -1e30, -3e38, -np.inf, 41, 88, 1e3, 1e10, 1e20, 3e38, np.inf, np.nan, 0.0, -0.0, 1e-30, -1e-30]
    at = rng.permutation(n)[:len(hard)]
    v[at] = hard[:at.size]
    return v.astype(np.float32)


@pytest.mark.parametrize("dtype", ["BF16", "FP32"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("far", [0, 1])
def test_group_norm(M, form, act, dtype, far):
    option, shape, groups = FORMS[form]
    x = np.random.default_rng(8).normal(0, 1, shape).astype(np.float32)
    x = O.bf16_round(x) if dtype == "BF16" else x
    v = arguments(shape[1], far)
    d = ",".join(map(str, shape))
    m = M(0)
    m.set_option("norm_form", option)
    m.load_text("input name=x shape=%s dtype=%s\ngroup_norm name=y in=x,g,b shape=%s dtype=%s groups=%d activation=%s\n" % (d, dtype, d, dtype, groups, act),
                {"g": np.zeros(shape[1], np.float32), "b": v})
    assert m.op_form("y")["form"] == form.split(",")[0]
    m.set_tensor("x", x)
    m.invoke()
    check(m.get_tensor("y"), v.reshape((1, -1) + (1,) * (len(shape) - 2)), act, dtype)
    m.close()


@pytest.mark.parametrize("dtype,tiles", [("BF16", 1064), ("BF16", 2032), ("BF16", 10128), ("FP32", 1016), ("FP32", 2040)])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("far", [0, 1])
@pytest.mark.parametrize("by", ["bias", "product"])
def test_linear(M, by, act, dtype, tiles, far):
    rows, k, n = 150, 128, 200
    m = M(0)
    m.set_option("linear_tiles", tiles)
    m.load_text("input name=x shape=%d,%d dtype=%s\nfully_connected name=y in=x,f,b shape=%d,%d dtype=%s activation=%s\n" % (rows, k, dtype, rows, n, dtype, act),
                {"f": np.eye(n, k, dtype=np.float32) if by == "product" else np.zeros((n, k), np.float32),
                 "b": arguments(n, far) if by == "bias" else np.zeros(n, np.float32)})
    x = np.zeros((rows, k), np.float32)
    v = np.broadcast_to(arguments(n, far), (rows, n))
    if by == "product":  # one value of a row beside zeros: an infinity or a NaN makes the rest of its row NaN
        a = arguments(rows, far)
        a = O.bf16_round(a) if dtype == "BF16" else a
        a = np.where(np.isfinite(a), a, 0.0).astype(np.float32)
        x[np.arange(rows), np.arange(rows) % k] = a
        v = np.zeros((rows, n), np.float32)
        v[:, :k] = x
    m.set_tensor("x", x)
    m.invoke()
    check(m.get_tensor("y"), v, act, dtype)
    m.close()
