"""Every path of the block-scaled 8-bit products in its steady state: the large tiles
over reductions that load each stage again and again, the half-height tiles behind
them, two pairs of operands that change in the middle of a loop; and how far 16-bit
results lie from the products themselves. Which path a size takes is pinned in
test_f8_choice.py."""
import math

import numpy as np
import pytest

import f8_ref as ref
from test_gpu_f8 import DTYPES, HALF, TINY, env, gate_bounds, host, kept_ok, operand, product_bound  # noqa: F401

pytestmark = pytest.mark.gpu

# (M, N, K) that run on large tiles alone, and with half-height tiles behind them.
LARGE = [(4096, 4096, 1100), (3300, 3300, 700)]
LARGE_AND_HALF = [(4200, 4130, 1100)]
# (T, D, F) of a gated forward pass on both, and of a gradient whose product is LARGE.
GATED_LARGE_AND_HALF = (2100, 1100, 4070)
GATED_BWD_LARGE = (4096, 4096, 700)
# One of each other way.
FEW = [(16, 4096, 4096), (64, 2048, 2048)]
SMALL = [(1100, 2100, 1500)]
SPLIT = [(129, 2048, 5504)]


def product(env, a, b, dt, M, N, K):
    buf, C = env.out(M, N, dt, 1, 2)
    n = env.L.seeml_hip_gemm_f8_scratch(M, N, K)
    env.call("gemm_f8_nt", *a, *b, C, DTYPES[dt], C.stride(0), M, N, K, env.scratch(n), n)
    assert bool((buf[:, :2] == 7).all()) and bool((buf[:, 2 + N:] == 7).all())
    return C.double().cpu().numpy()


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("M, N, K", LARGE + LARGE_AND_HALF)
def test_large_products_over_many_blocks(env, dt, M, N, K):
    rng = np.random.default_rng(M + N + K)
    a, av = operand(env, rng, M, K)
    b, bv = operand(env, rng, N, K)
    got = product(env, a, b, dt, M, N, K)
    want, tol = product_bound(av, bv, dt)
    assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()
    # Whole blocks that went missing or came twice would pass no 2-norm: float32 sums
    # (random half ulps, as many inside an instruction as between), the 16-bit products'
    # 2e-5, and the output's rounding.
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= (2 * math.sqrt(K / 32) * 2.0 ** -24 if dt == "f32" else 2e-5 + HALF[dt]), off


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_special_values_on_large_tiles(env, dt):
    M, N, K = LARGE[1]
    rng = np.random.default_rng(12)
    x, w = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    # In the first, a middle and the last block of k, and in the last row.
    x[1, 5], x[M - 1, 400], w[4, K - 1] = math.nan, math.inf, math.inf
    x[2], w[7] = x[2] * 1e30, w[7] * 1e-30
    x[0], w[:, 256:384] = 0.0, 0.0
    xm, wm = ref.quantize(x), ref.quantize(w)
    got = product(env, env.put(*xm), env.put(*wm), dt, M, N, K)
    want_bad = np.zeros((M, N), bool)
    want_bad[[1, M - 1]], want_bad[:, 4] = True, True
    np.testing.assert_array_equal(np.isnan(got), want_bad)
    want, tol = product_bound(np.nan_to_num(ref.values(*xm, K)), np.nan_to_num(ref.values(*wm, K)), dt)
    assert np.all((np.abs(got - want) <= tol) | want_bad)
    assert not got[0][~want_bad[0]].any()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gated_gradient_on_large_tiles(env, dt):
    """Two pairs of operands, six steps each."""
    T, D, F = GATED_BWD_LARGE
    rng = np.random.default_rng(13)
    gm, um = ref.quantize(rng.standard_normal((T, F)) * 2), ref.quantize(rng.standard_normal((T, F)))
    dh, dhv = env.matrix(rng.standard_normal((T, F)), dt)
    wm = [ref.quantize(rng.standard_normal((D, F)) / math.sqrt(F), True) for _ in range(2)]
    dg, du = env.room(T, F), env.room(T, F)
    _, dx = env.out(T, D, dt)
    n = env.L.seeml_hip_gated_f8_scratch(T, D, F)
    env.call("gated_f8_bwd", dh, DTYPES[dt], F, *env.put(*gm), *env.put(*um), 3, *env.put(*wm[0]), *env.put(*wm[1]),
             *dg, *du, None, 0, dx, D, T, D, F, env.scratch(n), n)
    g, u = ref.values(*gm, F), ref.values(*um, F)
    a, d = ref.act(3, g)
    kept_ok(dg, dhv * u * d, np.abs(dhv * u) * (2.0 ** -20 + 2.0 ** -22 * np.abs(d)), F)
    kept_ok(du, dhv * a, np.abs(dhv) * (np.abs(g) * 2.0 ** -20 + np.abs(a) * 2.0 ** -22), F)
    dgv, duv = (ref.values(*host(m), F) for m in (dg, du))
    want, tol = product_bound(np.hstack([dgv, duv]), np.hstack([ref.values(*m, F) for m in wm]), dt)
    off = np.abs(dx.double().cpu().numpy() - want)
    assert np.all(off <= tol), off.max()


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_gated_forward_on_large_tiles(env, dt):
    T, D, F = GATED_LARGE_AND_HALF
    rng = np.random.default_rng(14)
    x, xv = operand(env, rng, T, D)
    wm = [ref.quantize(rng.standard_normal((F, D)) / math.sqrt(D), True) for _ in range(2)]
    w = [env.put(*m) for m in wm]
    gv, uv = (ref.values(*m, D) for m in wm)
    for keep in (False, True):
        (g, eg), (u, eu), (h, eh) = gate_bounds(xv, gv, uv, 3, keep or dt == "f32")
        _, out = env.out(T, F, dt)
        kept = [env.room(T, F) if keep else (None, None) for _ in range(3)]
        env.call("gated_f8_fwd", *x, *w[0], *w[1], 3, out, DTYPES[dt], F, *kept[0], *kept[1], *kept[2], T, D, F, None, 0)
        off = np.abs(out.double().cpu().numpy() - h)
        assert np.all(off <= eh + np.abs(h) * HALF[dt] * (1 + 2.0 ** -10) + TINY[dt]), off.max()
        if keep:
            for m, want, err in ((kept[0], h, eh), (kept[1], g, eg), (kept[2], u, eu)):
                kept_ok(m, want, err, F)


@pytest.mark.parametrize("M, N, K", FEW + SMALL + SPLIT + LARGE[1:])
@pytest.mark.parametrize("kind", ["even", "positive", "spread"])
def test_16_bit_products_keep_what_is_promised(env, M, N, K, kind):
    """2-norm error of half outputs beyond their rounding: 2e-5 where magnitudes are even,
    1e-4 where they spread over 2^16."""
    rng = np.random.default_rng(M + N + K)

    def values(rows):
        if kind == "even":
            return rng.standard_normal((rows, K))
        if kind == "positive":
            return rng.uniform(1, 2, (rows, K)) * 2.0 ** -4
        return rng.standard_normal((rows, K)) * np.exp2(rng.integers(-8, 8, (rows, K)) - 5)

    am, bm = ref.quantize(values(M)), ref.quantize(values(N))
    got = product(env, env.put(*am), env.put(*bm), "f16", M, N, K)
    want = ref.values(*am, K) @ ref.values(*bm, K).T
    norm = np.linalg.norm(want)
    off = np.linalg.norm(got - want) / norm
    rounding = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want) / norm
    # The product's own error and the rounding's are independent: their squares add, but
    # for a chance correlation of the order of 1 / sqrt(outputs).
    assert off ** 2 <= rounding ** 2 * (1 + 4 / math.sqrt(M * N)) + (1e-4 if kind == "spread" else 2e-5) ** 2, \
        math.sqrt(max(0.0, off ** 2 - rounding ** 2))
