"""The block-scaled 8-bit operators on the GPU, through the C-ABI, against the
64-bit reference (f8_ref.py) at the bounds of 32-bit arithmetic."""
import math

import numpy as np
import pytest

import f8_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": 0, "bf16": 1, "f16": 2}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # a rounding, relative
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


class Env:
    def __init__(self):
        import torch
        from seeml_amd import _lib
        self.torch, self.L, self._lib = torch, _lib.lib(), _lib
        self.types = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

    def call(self, name, *args, stream=None):
        args = [a.data_ptr() if hasattr(a, "data_ptr") else a for a in args]
        s = stream if stream is not None else self.torch.cuda.current_stream().cuda_stream
        rc = getattr(self.L, "seeml_hip_" + name)(*args, s)
        assert rc == 0, f"{name}: {self._lib.kernel_error()}"

    def matrix(self, x, dt, pad=0, lead=0):
        """x on the GPU in type dt, as columns of a wider buffer; and its values."""
        rows, cols = x.shape
        buf = self.torch.full((rows, cols + pad + lead), 7.0, dtype=self.types[dt], device="cuda")
        with np.errstate(over="ignore"):
            buf[:, lead:lead + cols] = self.torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(self.types[dt])
        view = buf[:, lead:lead + cols]
        return view, view.double().cpu().numpy()

    def room(self, rows, cols):
        """Codes and scales of a matrix, filled with bytes that no result has."""
        t = self.torch
        return (t.full((rows, ref.up(cols)), 0xAA, dtype=t.uint8, device="cuda"),
                t.full((ref.up(cols) // 128, ref.up(rows)), 0xAA, dtype=t.uint8, device="cuda"))

    def put(self, codes, scales):
        t = self.torch
        return t.from_numpy(codes).cuda(), t.from_numpy(scales).cuda()

    def out(self, rows, cols, dt, pad=0, lead=0):
        buf = self.torch.full((rows, cols + pad + lead), 7.0, dtype=self.types[dt], device="cuda")
        return buf, buf[:, lead:lead + cols]

    def scratch(self, n):
        return self.torch.full((n,), 0xFF, dtype=self.torch.uint8, device="cuda") if n else None


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return Env()


def host(m):
    return m[0].cpu().numpy(), m[1].cpu().numpy()


def untouched(buf, lead, cols):
    """The columns beside a strided output are as they were."""
    return bool((buf[:, :lead] == 7).all()) and bool((buf[:, lead + cols:] == 7).all())


SHAPES = [(1, 1), (1, 128), (2, 127), (3, 129), (5, 640), (130, 127), (127, 64), (257, 300), (128, 1024), (1, 5000)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_quantize_is_the_formats_definition(env, dt, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-20, 12, (rows, 1)))
    pad, lead = (0, 0) if cols % 2 else (5, 3)
    xd, xv = env.matrix(x, dt, pad, lead)
    m = env.room(rows, cols)
    env.call("f8_quantize", xd, DTYPES[dt], xd.stride(0), rows, cols, *m)
    codes, scales = host(m)
    want = ref.quantize(xv)
    np.testing.assert_array_equal(scales, want[1])
    np.testing.assert_array_equal(codes, want[0])
    buf, y = env.out(rows, cols, dt, pad, lead)
    env.call("f8_dequantize", *m, y, DTYPES[dt], y.stride(0), rows, cols)
    kept = env.torch.from_numpy(ref.values(*want, cols)).to(env.types[dt]).double().numpy()
    np.testing.assert_array_equal(y.double().cpu().numpy(), kept)
    assert untouched(buf, lead, cols)


def special_rows():
    big = float(np.finfo(np.float32).max)
    rows = [np.zeros(256), np.full(256, -0.0), np.full(256, big), np.full(256, 2.0 ** -149),
            np.full(256, math.nan), np.full(256, math.inf)]
    r = np.linspace(-3, 3, 256)
    for v in (math.nan, math.inf, -math.inf):
        q = r.copy()
        q[7] = v
        rows.append(q)
    rows.append(np.where(np.arange(256) % 2 == 0, big, 2.0 ** -140))
    rows.append(np.concatenate([ref.POSITIVE, -ref.POSITIVE, [0.0, 448.0]]))
    mid = (ref.POSITIVE[1:] + ref.POSITIVE[:-1]) / 2  # ties
    rows.append(np.concatenate([mid, [448.0, 448.0], -mid, [448.0, 448.0]]))
    rows.append(np.exp2(np.arange(256) * 0.05 - 135))
    return np.stack(rows)


def test_quantize_special_values(env):
    xd, xv = env.matrix(special_rows(), "f32")
    rows, cols = xv.shape
    m = env.room(rows, cols)
    env.call("f8_quantize", xd, 0, cols, rows, cols, *m)
    codes, scales = host(m)
    want = ref.quantize(xv)
    np.testing.assert_array_equal(scales, want[1])
    nan = np.isnan(ref.VALUES[want[0]])
    np.testing.assert_array_equal(nan, np.isnan(ref.VALUES[codes]))
    np.testing.assert_array_equal(codes[~nan], want[0][~nan])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (128, 128), (130, 127), (127, 300), (300, 129)])
def test_quantize_weight_and_its_transpose(env, dt, rows, cols):
    rng = np.random.default_rng(rows + 7 * cols)
    wd, wv = env.matrix(rng.standard_normal((rows, cols)), dt, 3, 1)
    m, mt = env.room(rows, cols), env.room(cols, rows)
    env.call("f8_quantize_weight", wd, DTYPES[dt], wd.stride(0), rows, cols, *m, *mt)
    want, want_t = ref.quantize(wv, True), ref.quantize(wv.T, True)
    for got, w in ((m, want), (mt, want_t)):
        codes, scales = host(got)
        np.testing.assert_array_equal(codes, w[0])
        np.testing.assert_array_equal(scales, w[1])
    only = env.room(cols, rows)
    env.call("f8_quantize_weight", wd, DTYPES[dt], wd.stride(0), rows, cols, None, None, *only)
    assert env.torch.equal(only[0], mt[0]) and env.torch.equal(only[1], mt[1])


def operand(env, rng, rows, cols, square=False):
    """A matrix in 8 bits on the GPU, and its values."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-3, 4, (rows, 1)))
    m = ref.quantize(x, square)
    return env.put(*m), ref.values(*m, cols)


def product_bound(a, b, dt, full=None):
    """K products, each exact, in K additions of at most an ulp of the sum of
    magnitudes; the output's rounding. With 16-bit outputs (not `full`) a block's 128 products
    are cut 16 bits below the largest first, which is at most the largest of a's row
    times the largest of b's in that block."""
    want = a @ b.T
    K = a.shape[1]
    err = (K * 2.0 ** -23) * (np.abs(a) @ np.abs(b).T)
    if not (dt == "f32" if full is None else full):
        for k in range(0, K, 128):
            top = np.abs(a[:, k:k + 128]).max(1)[:, None] * np.abs(b[:, k:k + 128]).max(1)
            err += min(K - k, 128) * 2.0 ** -16 * top
    return want, err * (1 + HALF[dt]) + np.abs(want) * HALF[dt] + TINY[dt]


# Every row group of the few-row kernel, both tile sizes, split and unsplit, a last round
# of half tiles.
GEMMS = [(1, 1, 1), (1, 17, 129), (3, 2048, 512), (16, 130, 128), (17, 33, 640), (33, 100, 1000), (64, 15, 256),
         (65, 1, 127), (100, 129, 300), (128, 128, 128), (129, 257, 2100), (300, 200, 513), (257, 4100, 384),
         (2300, 2200, 200), (2048, 2304, 260),
         (4200, 4130, 150)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M, N, K", GEMMS)
def test_product(env, dt, M, N, K):
    rng = np.random.default_rng(M + 3 * N + 5 * K)
    a, av = operand(env, rng, M, K)
    b, bv = operand(env, rng, N, K, square=True)
    lead, pad = (1, 2) if N % 2 else (0, 0)
    buf, C = env.out(M, N, dt, pad, lead)
    n = env.L.seeml_hip_gemm_f8_scratch(M, N, K)
    env.call("gemm_f8_nt", *a, *b, C, DTYPES[dt], C.stride(0), M, N, K, env.scratch(n), n)
    want, tol = product_bound(av, bv, dt)
    got = C.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()
    assert untouched(buf, lead, N)


@pytest.mark.parametrize("M", [1, 40, 200, 2100])
def test_product_of_two_activations(env, M):
    """Scales of B that differ from row to row."""
    rng = np.random.default_rng(M)
    a, av = operand(env, rng, M, 450)
    b, bv = operand(env, rng, 2050, 450)
    _, C = env.out(M, 2050, "f32")
    n = env.L.seeml_hip_gemm_f8_scratch(M, 2050, 450)
    env.call("gemm_f8_nt", *a, *b, C, 0, 2050, M, 2050, 450, env.scratch(n), n)
    want, tol = product_bound(av, bv, "f32")
    assert np.all(np.abs(C.double().cpu().numpy() - want) <= tol)


@pytest.mark.parametrize("M", [1, 130, 2100])
def test_product_keeps_to_float32(env, M):
    """2-norm error of a long reduction: that of float32 sums."""
    rng = np.random.default_rng(5 + M)
    a, av = operand(env, rng, M, 4096)
    b, bv = operand(env, rng, 2048, 4096, square=True)
    _, C = env.out(M, 2048, "f32")
    n = env.L.seeml_hip_gemm_f8_scratch(M, 2048, 4096)
    env.call("gemm_f8_nt", *a, *b, C, 0, 2048, M, 2048, 4096, env.scratch(n), n)
    want = av @ bv.T
    off = np.linalg.norm(C.double().cpu().numpy() - want) / np.linalg.norm(want)
    # 128 sums of 32 products, each rounded by half an ulp, and as much inside them.
    assert off <= 2 * math.sqrt(128) * 2.0 ** -24, off


@pytest.mark.parametrize("M, N", [(3, 40), (150, 300), (2100, 2100)])
def test_product_special_values_in_16_bits(env, M, N):
    """The 8-bit matrix cores' own NaN, zeros and ends of the scales."""
    rng = np.random.default_rng(10)
    x, w = rng.standard_normal((M, 300)), rng.standard_normal((N, 300))
    x[1, 5], w[4, 299] = math.nan, math.inf
    x[2], w[7] = x[2] * 1e30, w[7] * 1e-30
    x[0], w[:, 128:256] = 0.0, 0.0
    xm, wm = ref.quantize(x), ref.quantize(w)
    _, C = env.out(M, N, "bf16")
    n = env.L.seeml_hip_gemm_f8_scratch(M, N, 300)
    env.call("gemm_f8_nt", *env.put(*xm), *env.put(*wm), C, 1, N, M, N, 300, env.scratch(n), n)
    got = C.double().cpu().numpy()
    want_bad = np.zeros((M, N), bool)
    want_bad[1], want_bad[:, 4] = True, True
    np.testing.assert_array_equal(np.isnan(got), want_bad)
    want, tol = product_bound(np.nan_to_num(ref.values(*xm, 300)), np.nan_to_num(ref.values(*wm, 300)), "bf16")
    assert np.all(np.abs(got - want)[~want_bad] <= tol[~want_bad])
    assert not got[0][~want_bad[0]].any()


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("T, F", [(5, 40), (70, 300), (2100, 2100)])
def test_gated_special_values(env, T, F, keep):
    """A NaN or an overflow of one value leaves the others of its row and block."""
    rng = np.random.default_rng(11)
    x = rng.standard_normal((T, 130))
    x[1, 3] = math.nan
    x[2] = 0.0
    w = [rng.standard_normal((F, 130)) for _ in range(2)]
    w[0][5, 7], w[1][6, 0] = math.nan, math.inf
    xm, gm, um = ref.quantize(x), ref.quantize(w[0]), ref.quantize(w[1])
    _, h = env.out(T, F, "bf16")
    kept = [env.room(T, F) if keep else (None, None) for _ in range(3)]
    env.call("gated_f8_fwd", *env.put(*xm), *env.put(*gm), *env.put(*um), 3, h, 1, F, *kept[0], *kept[1], *kept[2],
             T, 130, F, None, 0)
    bad_g, bad_u = np.zeros((T, F), bool), np.zeros((T, F), bool)
    bad_g[1], bad_u[1], bad_g[:, 5], bad_u[:, 6] = True, True, True, True
    got = h.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), bad_g | bad_u)
    assert not got[2][~(bad_g | bad_u)[2]].any()
    if keep:
        values = lambda m: np.nan_to_num(ref.values(*m, 130))  # noqa: E731
        (g, eg), (u, eu), (hv, eh) = gate_bounds(values(xm), values(gm), values(um), 3, True)
        for m, bad, want, err in ((kept[0], bad_g | bad_u, hv, eh), (kept[1], bad_g, g, eg), (kept[2], bad_u, u, eu)):
            codes, scales = host(m)
            np.testing.assert_array_equal(np.isnan(ref.VALUES[codes[:, :F]]), bad)
            v = np.where(bad, 0.0, ref.values(codes, scales, F))
            off = np.abs(v - np.where(bad, 0.0, want))
            half = np.where(bad, 0.0, ref.step(codes, scales, F))
            assert np.all((off <= half * (1 + 2.0 ** -20) + err) | bad)


@pytest.mark.parametrize("M, N", [(3, 40), (150, 300), (2100, 2100)])
def test_product_special_values(env, M, N):
    """A NaN reaches its own row or column alone; the range's ends multiply."""
    rng = np.random.default_rng(9)
    x, w = rng.standard_normal((M, 200)), rng.standard_normal((N, 200))
    x[1, 5], w[4, 199] = math.nan, math.inf
    x[2], w[7] = x[2] * 1e38, w[7] * 1e-38
    xm, wm = ref.quantize(x), ref.quantize(w)
    _, C = env.out(M, N, "f32")
    n = env.L.seeml_hip_gemm_f8_scratch(M, N, 200)
    env.call("gemm_f8_nt", *env.put(*xm), *env.put(*wm), C, 0, N, M, N, 200, env.scratch(n), n)
    got = C.double().cpu().numpy()
    bad = np.isnan(got)
    want_bad = np.zeros_like(bad)
    want_bad[1], want_bad[:, 4] = True, True
    av, bv = np.nan_to_num(ref.values(*xm, 200)), np.nan_to_num(ref.values(*wm, 200))
    # Where the magnitudes' sum passes float32's largest number, partial sums may be
    # infinities of both signs.
    held = np.abs(av) @ np.abs(bv).T < 3.4e38
    np.testing.assert_array_equal(bad[held], want_bad[held])
    want, tol = product_bound(av, bv, "f32")
    # Row 7 of w lies below 2^-126, where the bfloat16 that codes are widened to has multiples
    # of 2^-133: each of its values may be off by 2^-134 (its codes' own step is 2^-136).
    tol[:, 7] += np.abs(av).sum(1) * 2.0 ** -134
    fine = ~bad & held
    assert np.all(np.abs(got - want)[fine] <= tol[fine])


GATES = [(1, 1, 1), (1, 300, 130), (9, 128, 256), (40, 520, 100), (64, 256, 129), (65, 200, 200), (130, 520, 1003),
         (70, 2100, 300), (2100, 300, 2200), (2100, 130, 4070)]


def gate_bounds(av, gv, uv, act, full):
    """g, u and h = act(g) u with bounds of their float32 errors."""
    g, eg = product_bound(av, gv, "f32", full)
    u, eu = product_bound(av, uv, "f32", full)
    a, _ = ref.act(act, g)
    # A slope is at most 1.13; an activation's own value is off by 2^-20 of |g|.
    ea = 1.13 * eg + np.abs(g) * 2.0 ** -20
    h = a * u
    return (g, eg), (u, eu), (h, np.abs(u) * ea + np.abs(a) * eu + ea * eu + np.abs(h) * 2.0 ** -23)


def kept_ok(m, want, err, cols):
    """8-bit values nearest to a number within `err` of `want`, padding zero."""
    codes, scales = host(m)
    rows = codes.shape[0]
    assert not codes[:, cols:].any() and not scales[:, rows:].any()
    amax = np.zeros((rows, ref.up(cols)))
    amax[:, :cols] = np.abs(want)
    amax = amax.reshape(rows, -1, 128).max(-1).T
    e = np.zeros((rows, ref.up(cols)))
    e[:, :cols] = err
    e = e.reshape(rows, -1, 128).max(-1).T
    lo, hi = ref.scale_byte(np.maximum(amax - e, 0)), ref.scale_byte(amax + e)
    s = scales[:, :rows].astype(int)
    assert np.all((lo <= s) & (s <= hi))
    off = np.abs(ref.values(codes, scales, cols) - want)
    assert np.all(off <= ref.step(codes, scales, cols) * (1 + 2.0 ** -20) + err), off.max()


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("T, D, F", GATES)
def test_gated_forward(env, act, T, D, F):
    dt = ["f32", "bf16", "f16"][(T + act) % 3]
    rng = np.random.default_rng(T + D + F + act)
    x, xv = operand(env, rng, T, D)
    w = [rng.standard_normal((F, D)) / math.sqrt(D) for _ in range(2)]
    wm = [ref.quantize(v, True) for v in w]
    gm, um = (env.put(*m) for m in wm)
    gv, uv = (ref.values(*m, D) for m in wm)
    n = env.L.seeml_hip_gated_f8_scratch(T, D, F)
    lead, pad = (2, 1) if F % 2 else (0, 0)
    for keep in (False, True):
        (g, eg), (u, eu), (h, eh) = gate_bounds(xv, gv, uv, act, keep or dt == "f32")
        buf, out = env.out(T, F, dt, pad, lead)
        kept = [env.room(T, F) if keep else (None, None) for _ in range(3)]
        env.call("gated_f8_fwd", *x, *gm, *um, act, out, DTYPES[dt], out.stride(0), *kept[0], *kept[1], *kept[2],
                 T, D, F, env.scratch(n), n)
        tol = eh + np.abs(h) * HALF[dt] * (1 + 2.0 ** -10) + TINY[dt]
        off = np.abs(out.double().cpu().numpy() - h)
        assert np.all(off <= tol), off.max()
        assert untouched(buf, lead, F)
        if keep:
            kept_ok(kept[0], h, eh, F)
            kept_ok(kept[1], g, eg, F)
            kept_ok(kept[2], u, eu, F)
    # Any one of the outputs alone has the same bits.
    only = env.room(T, F)
    env.call("gated_f8_fwd", *x, *gm, *um, act, None, DTYPES[dt], 0, None, None, None, None, *only, T, D, F, env.scratch(n), n)
    assert env.torch.equal(only[0], kept[2][0]) and env.torch.equal(only[1], kept[2][1])


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("T, D, F", [(1, 1, 1), (3, 200, 130), (70, 129, 600), (300, 300, 257), (2100, 2050, 140)])
def test_gated_backward(env, act, T, D, F):
    dt = ["bf16", "f32", "f16"][(T + act) % 3]
    rng = np.random.default_rng(T + D + F + act)
    gm, um = ref.quantize(rng.standard_normal((T, F)) * 2), ref.quantize(rng.standard_normal((T, F)))
    dh, dhv = env.matrix(rng.standard_normal((T, F)), dt, 3, 2)
    wm = [ref.quantize(rng.standard_normal((D, F)) / math.sqrt(F), True) for _ in range(2)]
    dg, du = env.room(T, F), env.room(T, F)
    _, h = env.out(T, F, dt)
    buf, dx = env.out(T, D, dt, 1, 2)
    n = env.L.seeml_hip_gated_f8_scratch(T, D, F)
    args = lambda hh, dd, s, b: (dh, DTYPES[dt], dh.stride(0), *env.put(*gm), *env.put(*um), act, *env.put(*wm[0]),  # noqa: E731
                                 *env.put(*wm[1]), *dg, *du, hh, F, dd, dd.stride(0) if dd is not None else 0, T, D, F, s, b)
    env.call("gated_f8_bwd", *args(h, dx, env.scratch(n), n))
    g, u = ref.values(*gm, F), ref.values(*um, F)
    a, d = ref.act(act, g)
    # Slopes are off by 2^-20, activations by 2^-20 |g|.
    kept_ok(dg, dhv * u * d, np.abs(dhv * u) * (2.0 ** -20 + 2.0 ** -22 * np.abs(d)), F)
    kept_ok(du, dhv * a, np.abs(dhv) * (np.abs(g) * 2.0 ** -20 + np.abs(a) * 2.0 ** -22), F)
    hv = a * u
    off = np.abs(h.double().cpu().numpy() - hv)
    assert np.all(off <= np.abs(u * g) * 2.0 ** -20 + np.abs(hv) * (HALF[dt] * 1.01 + 2.0 ** -22) + TINY[dt])
    # dx of the gradients that were kept.
    dgv, duv = (ref.values(*host(m), F) for m in (dg, du))
    w1, w2 = (ref.values(*m, F) for m in wm)
    want, tol = product_bound(np.hstack([dgv, duv]), np.hstack([w1, w2]), dt)
    off = np.abs(dx.double().cpu().numpy() - want)
    assert np.all(off <= tol), off.max()
    assert untouched(buf, 2, D)
    before = [t.clone() for t in (*dg, *du)]
    env.call("gated_f8_bwd", *args(None, None, None, 0))
    assert all(env.torch.equal(p, q) for p, q in zip(before, (*dg, *du)))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 129), (130, 300), (64, 1024)])
@pytest.mark.parametrize("inplace", [False, True])
def test_activation_backward(env, dt, act, rows, cols, inplace):
    rng = np.random.default_rng(rows + cols + act)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-4, 7, (rows, 1)))
    m = ref.quantize(x)
    dy, dyv = env.matrix(rng.standard_normal((rows, cols)), dt, 2, 1)
    buf, dx = env.out(rows, cols, dt, 4, 3)
    if inplace:
        buf, dx = None, dy
    env.call("act_bwd_f8", dy, DTYPES[dt], dy.stride(0), *env.put(*m), act, dx, dx.stride(0), rows, cols)
    _, d = ref.act(act, ref.values(*m, cols))
    off = np.abs(dx.double().cpu().numpy() - dyv * d)
    assert np.all(off <= np.abs(dyv) * (2.0 ** -20 + np.abs(d) * HALF[dt] * 1.01) + TINY[dt]), off.max()
    assert inplace or untouched(buf, 3, cols)


@pytest.mark.parametrize("act", [1, 2, 3])
def test_activation_backward_at_the_ends_of_the_range(env, act):
    x = special_rows()
    m = ref.quantize(x)
    xv = ref.values(*m, 256)
    dy = env.torch.ones(x.shape, device="cuda")
    dx = env.torch.empty_like(dy)
    env.call("act_bwd_f8", dy, 0, 256, *env.put(*m), act, dx, 256, *x.shape)
    got = dx.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(xv))
    _, d = ref.act(act, np.nan_to_num(xv))
    assert np.all(np.abs(got - d)[~np.isnan(xv)] <= 2.0 ** -20)


# Each number of registers a row's threads hold, and rows read twice.
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (5, 130), (9, 512), (3, 1000), (4, 2048), (3, 4100), (2, 9000), (2, 17000)])
@pytest.mark.parametrize("inplace", [False, True])
def test_norm_backward(env, dt, rows, cols, inplace):
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-4, 7, (rows, 1)))
    if rows > 2:
        x[1] = 0.0
    m = ref.quantize(x)
    gamma = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    rstd = (1 / np.sqrt((x * x).mean(-1) + 1e-5)).astype(np.float32)
    dy, dyv = env.matrix(rng.standard_normal((rows, cols)), dt, 1, 1)
    buf, dx = env.out(rows, cols, dt, 1, 2)
    if inplace:
        buf, dx = None, dy
    t = env.torch
    env.call("rms_norm_bwd_f8", dy, DTYPES[dt], dy.stride(0), *env.put(*m), t.from_numpy(gamma).cuda(),
             t.from_numpy(rstd).cuda(), dx, dx.stride(0), rows, cols)
    xv = ref.values(*m, cols)
    want = ref.rms_bwd(dyv, xv, gamma.astype(np.float64), rstd.astype(np.float64))
    r = rstd[:, None].astype(np.float64)
    g = np.abs(dyv * gamma)
    # gamma dy, the sum of 8 products in float32, the coefficient and three roundings.
    along = (g * np.abs(xv)).mean(-1, keepdims=True)
    tol = 2.0 ** -24 * (4 * r * g + 16 * r ** 3 * np.abs(xv) * along) + np.abs(want) * HALF[dt] * 1.01 + TINY[dt]
    off = np.abs(dx.double().cpu().numpy() - want)
    assert np.all(off <= tol), (off / tol).max()
    assert inplace or untouched(buf, 2, cols)


LORAS = [(1, 1, 1), (31, 128, 8), (33, 130, 16), (200, 300, 17), (129, 64, 33), (1000, 520, 64), (300, 257, 128),
         (5000, 200, 16), (256, 200, 16), (257, 130, 32), (700, 130, 100)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T, D, r", LORAS)
def test_lora_gradient(env, dt, T, D, r):
    rng = np.random.default_rng(T + D + r)
    x, xv = operand(env, rng, T, D)
    dtm, dtv = env.matrix(rng.standard_normal((T, r)), dt, 3, 1)
    out = env.torch.full((D + 1, r), 7.0, device="cuda")
    n = env.L.seeml_hip_gemm_tn_f8_scratch(T, D, r)
    env.call("gemm_tn_f8", *x, dtm, DTYPES[dt], dtm.stride(0), out, T, D, r, env.scratch(n), n)
    want = xv.T @ dtv
    got = out.double().cpu().numpy()
    # Up to three products a term, T of each, every sum off by at most an ulp.
    tol = 3 * T * 2.0 ** -23 * (np.abs(xv).T @ np.abs(dtv))
    assert np.all(np.abs(got[:D] - want) <= tol + 2.0 ** -126), np.abs(got[:D] - want).max()
    assert np.all(got[D] == 7.0)
    if T >= 1000:
        # Sums of ranges of rows: random half ulps of at most T / 32 + 2 additions.
        off = np.linalg.norm(got[:D] - want) / np.linalg.norm(want)
        assert off <= 2.0 ** -23 * math.sqrt(T / 32 + 2) * 1.5, off


def test_lora_gradient_special_values(env):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((70, 140))
    x[3, 5] = math.nan
    m = ref.quantize(x)
    dt = rng.standard_normal((70, 20))
    big = float(np.finfo(np.float32).max)
    dt[4, 2], dt[5, 3], dt[6, 4], dt[7, 5] = math.inf, math.nan, big, 2.0 ** -140
    dt[:, 6] = 0.0
    dt[8, 6] = 1.0 + 2.0 ** -23
    d = env.torch.from_numpy(dt.astype(np.float32)).cuda()
    out = env.torch.empty(140, 20, device="cuda")
    n = env.L.seeml_hip_gemm_tn_f8_scratch(70, 140, 20)
    env.call("gemm_tn_f8", *env.put(*m), d, 0, 20, out, 70, 140, 20, env.scratch(n), n)
    got = out.double().cpu().numpy()
    xv = ref.values(*m, 140)
    with np.errstate(invalid="ignore", over="ignore"):
        want = xv.T @ d.double().cpu().numpy()
    # A sum rounds to an infinity from half an ulp past the largest number on.
    np.testing.assert_array_equal(np.isfinite(got), np.abs(want) < big * (1 + 2.0 ** -25))
    np.testing.assert_array_equal(np.isnan(got)[:, 3], True)
    np.testing.assert_array_equal(np.isnan(got)[5], True)
    keep = np.arange(140) != 5
    # Two parts, 1 and 2^-23, of exact products: one sum, and the matrix cores' sums round
    # towards minus infinity, by less than an ulp.
    one = xv[8][keep] * (1.0 + 2.0 ** -23)
    assert np.all(np.abs(got[keep, 6] - one) <= np.abs(one) * 2.0 ** -23)


def training_step(env, s, stream=None):
    """A layer's step as a training program makes it, every tensor given."""
    c = lambda name, *a: env.call(name, *a, stream=stream)  # noqa: E731
    T, D, F, r, dt = s["T"], s["D"], s["F"], s["r"], 1
    c("f8_quantize", s["x"], dt, D, T, D, *s["x8"])
    c("gated_f8_fwd", *s["x8"], *s["wg_t"], *s["wu_t"], 3, s["h"], dt, F, *s["h8"], *s["g8"], *s["u8"], T, D, F,
      s["scratch"], s["bytes"])
    c("gemm_f8_nt", *s["h8"], *s["wd_t"], s["y"], dt, D, T, D, F, s["scratch"], s["bytes"])
    c("f8_quantize", s["dy"], dt, D, T, D, *s["dy8"])
    c("gemm_f8_nt", *s["dy8"], *s["wd"], s["dh"], dt, F, T, F, D, s["scratch"], s["bytes"])
    c("gated_f8_bwd", s["dh"], dt, F, *s["g8"], *s["u8"], 3, *s["wg"], *s["wu"], *s["dg8"], *s["du8"], s["h2"], F,
      s["dx"], D, T, D, F, s["scratch"], s["bytes"])
    c("gemm_tn_f8", *s["x8"], s["dt"], dt, r, s["da"], T, D, r, s["scratch"], s["bytes"])
    c("rms_norm_bwd_f8", s["dx"], dt, D, *s["x8"], s["gamma"], s["rstd"], s["dn"], D, T, D)
    c("act_bwd_f8", s["dy"], dt, D, *s["x8"], 2, s["da2"], D, T, D)
    return [s[k] for k in ("y", "h", "h2", "dx", "da", "dn", "da2")]


def make_step(env, seed, T=200, D=256, F=520, r=16):
    t = env.torch
    g = t.Generator(device="cuda")
    g.manual_seed(seed)
    new = lambda *s, f=t.bfloat16: t.zeros(*s, device="cuda", dtype=f)  # noqa: E731
    s = dict(T=T, D=D, F=F, r=r)
    s["x"], s["dy"] = (t.randn(T, D, generator=g, device="cuda").to(t.bfloat16) for _ in range(2))
    s["dt"] = t.randn(T, r, generator=g, device="cuda").to(t.bfloat16)
    s["gamma"] = 1 + 0.1 * t.randn(D, generator=g, device="cuda")
    s["rstd"] = t.rsqrt(s["x"].float().square().mean(-1) + 1e-5)
    for name, rows, cols in (("wg", D, F), ("wu", D, F), ("wd", F, D)):
        w = t.randn(rows, cols, generator=g, device="cuda") / math.sqrt(rows)
        s[name], s[name + "_t"] = env.room(rows, cols), env.room(cols, rows)
        env.call("f8_quantize_weight", w, 0, cols, rows, cols, *s[name], *s[name + "_t"])
    for k in ("h", "h2", "dh"):
        s[k] = new(T, F)
    for k in ("y", "dx", "dn", "da2"):
        s[k] = new(T, D)
    s["da"] = new(D, r, f=t.float32)
    for k in ("h8", "g8", "u8", "dg8", "du8"):
        s[k] = env.room(T, F)
    for k in ("x8", "dy8"):
        s[k] = env.room(T, D)
    s["bytes"] = max(env.L.seeml_hip_gated_f8_scratch(T, D, F), env.L.seeml_hip_gemm_f8_scratch(T, D, F),
                     env.L.seeml_hip_gemm_f8_scratch(T, F, D), env.L.seeml_hip_gemm_tn_f8_scratch(T, D, r), 16)
    s["scratch"] = env.scratch(s["bytes"])
    t.cuda.synchronize()
    return s


def test_a_layers_step_together(env):
    """Quantise, gated block, down projection and back, with an adapter's gradient."""
    s = make_step(env, 1)
    T, D, F = s["T"], s["D"], s["F"]
    training_step(env, s)
    d = lambda k: s[k].double().cpu().numpy()  # noqa: E731
    v = lambda k, cols: ref.values(*host(s[k]), cols)  # noqa: E731
    x8 = v("x8", D)
    np.testing.assert_array_equal(x8, ref.values(*ref.quantize(d("x")), D))
    wg, wu, wd = v("wg", F), v("wu", F), v("wd", D)
    np.testing.assert_array_equal(wg.T, v("wg_t", D))
    a, _ = ref.act(3, x8 @ wg)
    h = a * (x8 @ wu)
    assert np.linalg.norm(d("h") - h) <= 2.0 ** -8 * np.linalg.norm(h)
    # The down projection of h in 8 bits, and its gradient: exact products of what was kept.
    for got, a_, b_ in (("y", v("h8", F), wd.T), ("dh", v("dy8", D), wd)):
        want, tol = product_bound(a_, b_, "bf16")
        assert np.all(np.abs(d(got) - want) <= tol)
    # h again, from g and u in 8 bits: two roundings of 2^-4 and a slope.
    assert np.linalg.norm(d("h2") - h) <= 2.0 ** -3 * np.linalg.norm(h)
    want, tol = product_bound(np.hstack([v("dg8", F), v("du8", F)]), np.hstack([wg, wu]), "bf16")
    assert np.all(np.abs(d("dx") - want) <= tol)
    # The whole gradient against the unrounded chain: four roundings of 2^-4 at most, independent.
    g, u = x8 @ wg, x8 @ wu
    a, sl = ref.act(3, g)
    chain = (d("dh") * u * sl) @ wg.T + (d("dh") * a) @ wu.T
    assert np.linalg.norm(d("dx") - chain) <= 2 * 2.0 ** -4 * np.linalg.norm(chain)
    want = x8.T @ d("dt")
    assert np.all(np.abs(d("da") - want) <= T * 2.0 ** -23 * (np.abs(x8).T @ np.abs(d("dt"))))


def test_same_bits_eager_captured_and_on_two_streams(env):
    t = env.torch
    a, b = make_step(env, 2), make_step(env, 3, T=70, D=130, F=300, r=20)
    want_a = [o.clone() for o in training_step(env, a)]
    want_b = [o.clone() for o in training_step(env, b)]
    t.cuda.synchronize()
    graphs = []
    for s in (a, b):
        stream = t.cuda.Stream()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=stream):
            training_step(env, s)
        graphs.append((g, stream))
    outs = [[s[k] for k in ("y", "h", "h2", "dx", "da", "dn", "da2")] for s in (a, b)]
    for _ in range(3):
        for o in (*outs[0], *outs[1]):
            o.zero_()
        a["scratch"].fill_(0xFF)
        t.cuda.synchronize()
        for g, stream in graphs:
            with t.cuda.stream(stream):
                g.replay()
        t.cuda.synchronize()
        for got, want in zip((*outs[0], *outs[1]), (*want_a, *want_b)):
            assert t.equal(got, want)
    # Eager on two streams at once.
    s1, s2 = t.cuda.Stream(), t.cuda.Stream()
    for o in (*outs[0], *outs[1]):
        o.zero_()
    t.cuda.synchronize()
    training_step(env, a, stream=s1.cuda_stream)
    training_step(env, b, stream=s2.cuda_stream)
    t.cuda.synchronize()
    for got, want in zip((*outs[0], *outs[1]), (*want_a, *want_b)):
        assert t.equal(got, want)


def test_offsets_past_32_bits(env):
    """Rows whose elements lie past 2^31 and 2^32 bytes."""
    t = env.torch
    rows, cols, stride = 3, 300, (1 << 29) + 5
    buf = t.zeros(2 * stride + cols, device="cuda", dtype=t.float32)
    x = t.as_strided(buf, (rows, cols), (stride, 1))
    rng = np.random.default_rng(4)
    xv = rng.standard_normal((rows, cols)).astype(np.float32)
    x.copy_(t.from_numpy(xv))
    m = env.room(rows, cols)
    env.call("f8_quantize", x, 0, stride, rows, cols, *m)
    want = ref.quantize(xv.astype(np.float64))
    np.testing.assert_array_equal(host(m)[0], want[0])
    env.call("act_bwd_f8", x, 0, stride, *m, 1, x, stride, rows, cols)
    xq = ref.values(*want, cols)
    np.testing.assert_array_equal(x.double().cpu().numpy(), xv * (xq > 0))


def test_codes_past_32_bits(env):
    """A matrix of more than 2^32 values."""
    t = env.torch
    rows, cols = (1 << 18) + 3, 16384 + 1
    x = t.zeros(rows, cols, device="cuda", dtype=t.bfloat16)
    x[-1] = t.linspace(-2, 2, cols, device="cuda")
    x[rows // 2] = 1.0
    m = (t.empty(rows, ref.up(cols), device="cuda", dtype=t.uint8),
         t.empty(ref.up(cols) // 128, ref.up(rows), device="cuda", dtype=t.uint8))
    env.call("f8_quantize", x, 1, cols, rows, cols, *m)
    last = x[-1:].double().cpu().numpy()
    want = ref.quantize(last)
    np.testing.assert_array_equal(m[0][-1:].cpu().numpy(), want[0])
    np.testing.assert_array_equal(m[1][:, rows - 1].cpu().numpy(), want[1][:, 0])
    assert int(m[0][rows // 2, 0]) == 0x78 and int(m[0][rows // 2 + 1].max()) == 0
    # One row of products and a gradient at the far end.
    w = ref.quantize(np.eye(3, cols))
    _, C = env.out(rows, 3, "f32")
    n = env.L.seeml_hip_gemm_f8_scratch(rows, 3, cols)
    env.call("gemm_f8_nt", *m, *env.put(*w), C, 0, 3, rows, 3, cols, env.scratch(n), n)
    np.testing.assert_array_equal(C[-1].double().cpu().numpy(), ref.values(*want, cols)[0, :3])
    assert float(C[:-1].abs().sum()) == 3.0
    dt = t.zeros(rows, 1, device="cuda")
    dt[-1] = 1.0
    out = t.empty(cols, 1, device="cuda")
    n = env.L.seeml_hip_gemm_tn_f8_scratch(rows, cols, 1)
    env.call("gemm_tn_f8", *m, dt, 0, 1, out, rows, cols, 1, env.scratch(n), n)
    np.testing.assert_array_equal(out[:, 0].double().cpu().numpy(), ref.values(*want, cols)[0])
