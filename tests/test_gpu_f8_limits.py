"""The block-scaled 8-bit operators where a factor leaves float32's range though the
result does not, and where results are small beside their factors: against the
64-bit reference (f8_ref.py)."""
import math

import numpy as np
import pytest

import f8_ref as ref
from test_gpu_f8 import DTYPES, HALF, TINY, env, host, product_bound  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", [1, 2, 3])
def test_gated_gradient_of_large_factors_on_a_flat_slope(env, act, dt):
    """dh u passes float32's range, dh u act'(g) does not."""
    rng = np.random.default_rng(act)
    T, F, D = 5, 300, 70
    far = {1: -1.0, 2: -6.0, 3: -60.0}[act]  # slopes 0, -7e-10 and -5e-25
    big = {"f32": (1e20, 1e20), "bf16": (1e20, 1e20), "f16": (6e4, 1e36)}[dt]
    sign = lambda: rng.choice([-1.0, 1.0], (T, F))  # noqa: E731
    gm = ref.quantize(far * rng.uniform(1.0, 1.2, (T, F)))
    um = ref.quantize(big[1] * rng.uniform(0.5, 1.0, (T, F)) * sign())
    dh, dhv = env.matrix(big[0] * rng.uniform(0.5, 1.0, (T, F)) * sign(), dt)
    wm = [ref.quantize(rng.standard_normal((D, F)) * 1e-8, True) for _ in range(2)]
    dg, du = env.room(T, F), env.room(T, F)
    _, dx = env.out(T, D, dt)
    n = env.L.seeml_hip_gated_f8_scratch(T, D, F)
    env.call("gated_f8_bwd", dh, DTYPES[dt], F, *env.put(*gm), *env.put(*um), act, *env.put(*wm[0]), *env.put(*wm[1]),
             *dg, *du, None, 0, dx, D, T, D, F, env.scratch(n), n)
    g, u = ref.values(*gm, F), ref.values(*um, F)
    a, d = ref.act(act, g)
    for m, want in ((dg, dhv * d * u), (du, dhv * a)):
        codes, scales = host(m)
        off = np.abs(ref.values(codes, scales, F) - want)
        # A rounding to 8 bits, and what float32's slopes lose this far out (2^-24 |t|, |t| below 104).
        assert np.all(off <= ref.step(codes, scales, F) * (1 + 2.0 ** -10) + np.abs(want) * 2.0 ** -12), np.nanmax(off)
    dgv, duv = (ref.values(*host(m), F) for m in (dg, du))
    want, tol = product_bound(np.hstack([dgv, duv]), np.hstack([ref.values(*m, F) for m in wm]), dt)
    got = dx.double().cpu().numpy()
    top = {"f32": 3.4e38, "bf16": 3.38e38, "f16": 65504.0}[dt]
    fits = np.abs(want) + tol < top
    assert np.all(np.abs(got - want)[fits] <= tol[fits]) and not np.isnan(got).any()
    assert fits.all() or dt == "f16"


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", [2, 3])
def test_gated_gradient_of_small_gradients_and_large_factors(env, act, dt):
    """dh act'(g) lies below float32, dh u and dh u act'(g) do not; beside elements whose dh u
    lies above."""
    rng = np.random.default_rng(20 + act)
    T, F = 4, 260
    far = {2: -5.0, 3: -40.0}[act]  # slopes -1e-6 and -2e-16
    gm = ref.quantize(far * rng.uniform(1.0, 1.1, (T, F)))
    um = ref.quantize(1e35 * rng.uniform(0.5, 1.0, (T, F)))
    size = np.where(np.arange(F) % 7 == 0, 1e10, 1e-36)
    dh, dhv = env.matrix(size * rng.uniform(0.5, 1.0, (T, F)), dt)
    dg, du = env.room(T, F), env.room(T, F)
    env.call("gated_f8_bwd", dh, DTYPES[dt], F, *env.put(*gm), *env.put(*um), act, None, None, None, None, *dg, *du,
             None, 0, None, 0, T, F, F, None, 0)
    g, u = ref.values(*gm, F), ref.values(*um, F)
    _, d = ref.act(act, g)
    want = dhv * d * u
    codes, scales = host(dg)
    got = ref.values(codes, scales, F)
    # What is itself past float32 is an infinity there, which 8 bits hold as NaN.
    over = np.abs(want) > float(np.finfo(np.float32).max)
    np.testing.assert_array_equal(np.isnan(got), over)
    off = np.abs(got - want)[~over]
    assert np.all(off <= (ref.step(codes, scales, F) * (1 + 2.0 ** -10) + np.abs(want) * 2.0 ** -12)[~over]), off.max()
    # The same without the large ones, whose blocks' scales leave the small ones no bits.
    dh, dhv = env.matrix(np.where(size > 1, 0.0, size) * rng.uniform(0.5, 1.0, (T, F)), dt)
    env.call("gated_f8_bwd", dh, DTYPES[dt], F, *env.put(*gm), *env.put(*um), act, None, None, None, None, *dg, *du,
             None, 0, None, 0, T, F, F, None, 0)
    want = dhv * d * u
    codes, scales = host(dg)
    off = np.abs(ref.values(codes, scales, F) - want)
    assert np.all(off <= np.abs(want) * (2.0 ** -4 + 2.0 ** -11)), np.nanmax(off / np.abs(want))


# Each number of threads and registers that a row has, and rows read twice.
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows, cols", [(5, 130), (4, 2048), (3, 4100), (2, 17000)])
@pytest.mark.parametrize("scale, up", [(1e25, 1e15), (1e-30, 1e-12)])
def test_norm_gradient_where_factors_multiply_out_of_range(env, dt, rows, cols, scale, up):
    """gamma dy x leaves float32's range, as does rstd^2; the gradient does not."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)) * scale
    m = ref.quantize(x)
    gamma = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    rstd = (1 / np.sqrt((x * x).mean(-1))).astype(np.float32)
    # A direction that has much of x in it, so that the row's mean counts.
    dy, dyv = env.matrix((x / scale + 0.5 * rng.standard_normal((rows, cols))) * up, dt)
    _, dx = env.out(rows, cols, dt)
    t = env.torch
    env.call("rms_norm_bwd_f8", dy, DTYPES[dt], cols, *env.put(*m), t.from_numpy(gamma).cuda(),
             t.from_numpy(rstd).cuda(), dx, cols, rows, cols)
    xv = ref.values(*m, cols)
    r = rstd[:, None].astype(np.float64)
    g = dyv * gamma
    xh = xv * r
    mean = (g * xh).mean(-1, keepdims=True)
    want = r * (g - xh * mean)
    # gamma dy, x rstd, the sum of 8 products in float32, the coefficient, three roundings.
    along = (np.abs(g * xh)).mean(-1, keepdims=True)
    tol = 2.0 ** -24 * (4 * r * np.abs(g) + 16 * r * np.abs(xh) * along) + np.abs(want) * HALF[dt] * 1.01 + TINY[dt]
    off = np.abs(dx.double().cpu().numpy() - want)
    assert np.all(off <= tol), np.nanmax(off / tol)


# Magnitudes over the whole range in which a slope or a value differs from its limit.
def spread_x():
    m = np.concatenate([-np.exp2(np.linspace(-20, 7.2, 700)), -np.linspace(0.05, 130, 1300), np.linspace(0.01, 30, 560)])
    return np.sort(m).reshape(-1, 128)


def act_parts(act, x):
    """s, 1 - s and du/dx of x s with s = 1 / (1 + exp(-t)), and |t|."""
    if act == 3:
        t, p = x, np.ones_like(x)
    else:
        c, k = math.sqrt(2 / math.pi), 0.044715
        t, p = 2 * c * (x + k * x ** 3), 2 * c * (1 + 3 * k * x * x)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-t)), 1 / (1 + np.exp(t)), p, np.abs(t)


@pytest.mark.parametrize("act", [2, 3])
def test_slopes_and_values_keep_their_digits(env, act):
    """Far out, where both are tiny, errors are small beside the values themselves."""
    m = ref.quantize(spread_x())
    rows, cols = m[0].shape
    x = ref.values(*m, cols)
    t = env.torch
    one = t.ones(rows, cols, device="cuda")
    dx = t.empty_like(one)
    env.call("act_bwd_f8", one, 0, cols, *env.put(*m), act, dx, cols, rows, cols)
    um = ref.quantize(np.ones((rows, cols)))
    h = t.empty_like(one)
    env.call("gated_f8_bwd", one, 0, cols, *env.put(*m), *env.put(*um), act, None, None, None, None,
             *env.room(rows, cols), *env.room(rows, cols), h, cols, None, 0, rows, cols, cols, None, 0)
    a, d = ref.act(act, x)
    s, rest, p, far = act_parts(act, x)
    # s and 1 - s: the exponential's ulp, half ulps of the correction of its argument, of 1 + e
    # and of the product, the reciprocal's ulp: below 2^-21 in all. GELU's t is a
    # polynomial of four roundings and two rounded constants: below 2^-21 |t|, of which s takes
    # 1 - s and 1 - s takes s. Below 2^-126 whole steps of 2^-149 come on top.
    bent = far if act == 2 else 0.0
    rel_s, rel_rest = 2.0 ** -21 * (1 + rest * bent), 2.0 ** -21 * (1 + s * bent)
    low = 2.0 ** -126
    slope_tol = s * rel_s + np.abs(x) * p * s * rest * (rel_s + rel_rest + 2.0 ** -21) + low * (1 + np.abs(x) * p)
    value_tol = np.abs(a) * (rel_s + 2.0 ** -22) + low * np.abs(x)
    off = np.abs(dx.double().cpu().numpy() - d)
    assert np.all(off <= slope_tol), x[off > slope_tol]
    off = np.abs(h.double().cpu().numpy() - a)
    assert np.all(off <= value_tol), x[off > value_tol]


@pytest.mark.parametrize("act", [1, 2, 3])
def test_activations_end_at_zero(env, act):
    """Far below, a value and its slope are nothing, whatever multiplies them."""
    x = np.array([[-3.0e38, -1e30, -1e10, -1e4, -1000.0, -300.0, -160.0, -130.0]])
    x = np.repeat(x, 128, 1)  # a block each, so that all keep their digits
    m = ref.quantize(x)
    cols = x.shape[1]
    t = env.torch
    dy = t.full((1, cols), 1e30, device="cuda")
    dx, h = t.empty_like(dy), t.empty_like(dy)
    env.call("act_bwd_f8", dy, 0, cols, *env.put(*m), act, dx, cols, 1, cols)
    um = ref.quantize(np.full((1, cols), 1e30))
    env.call("gated_f8_bwd", dy, 0, cols, *env.put(*m), *env.put(*um), act, None, None, None, None,
             *env.room(1, cols), *env.room(1, cols), h, cols, None, 0, 1, cols, cols, None, 0)
    assert not dx.any() and not h.any()


def test_the_largest_magnitudes(env):
    """From 248 x 2^120 on a value is kept as 2^128: an infinity in float32 and in float32
    sums. Below it, everything is finite and multiplies so, on every path."""
    top = 248.0 * 2.0 ** 120
    x = np.zeros((5, 130))
    x[0, 0], x[1, 0], x[2, 129] = np.nextafter(np.float32(top), np.float32(0)), top, -3.4e38
    x[3, :] = np.nextafter(np.float32(top), np.float32(0)) * 2.0 ** -20
    xm = ref.quantize(x)
    t = env.torch
    back = t.empty(5, 130, device="cuda")
    env.call("f8_dequantize", *env.put(*xm), back, 0, 130, 5, 130)
    want = ref.values(*xm, 130)
    assert want[0, 0] == 240 * 2.0 ** 120 and want[1, 0] == 2.0 ** 128 and want[2, 129] == -2.0 ** 128
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(back.cpu().numpy(), want.astype(np.float32))
    for M in (5, 70, 3300):  # few rows, small and large tiles
        full = np.zeros((M, 130))
        full[:4], full[-1] = x[:4], x[2]
        w = np.zeros((M, 130))  # zeros, units and small factors for each of x's columns
        w[1::3, 0], w[2::3, 129] = 1.0, 2.0 ** -30
        fm, wm = ref.quantize(full), ref.quantize(w)
        _, C = env.out(M, M, "f32")
        n = env.L.seeml_hip_gemm_f8_scratch(M, M, 130)
        env.call("gemm_f8_nt", *env.put(*fm), *env.put(*wm), C, 0, M, M, M, 130, env.scratch(n), n)
        fv, wv = ref.values(*fm, 130), ref.values(*wm, 130)
        huge = np.abs(fv) >= 2.0 ** 128
        with np.errstate(invalid="ignore"):
            want = np.where(huge, np.where(fv < 0, -np.inf, np.inf), fv)
            rows = np.flatnonzero(np.arange(M) < 4) if M > 5 else np.arange(M)
            rows = np.union1d(rows, [M - 1])
            got = C.double().cpu().numpy()
            for r in rows:
                terms = want[r] * wv  # an infinity times 0 is NaN
                np.testing.assert_array_equal(got[r], terms.sum(1))
        assert not np.delete(got, rows, 0).any()
