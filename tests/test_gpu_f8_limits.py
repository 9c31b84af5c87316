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
