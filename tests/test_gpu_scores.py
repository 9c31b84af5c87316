"""Token scores and top-k distillation on the GPU, through the C-ABI, against
the 64-bit reference (scores_ref.py) at the bounds of 32-bit arithmetic."""
import math

import numpy as np
import pytest

import scores_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": 0, "bf16": 1, "f16": 2}


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from seeml_amd import _lib

    class Env:
        pass

    e = Env()
    e.torch, e.L = torch, _lib.lib()
    e.types = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

    def call(name, *args):
        args = [a.data_ptr() if hasattr(a, "data_ptr") else a for a in args]
        rc = getattr(e.L, "seeml_hip_" + name)(*args, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, f"{name}: {_lib.kernel_error()}"

    def dev(a, dtype=None):
        t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
        return t if dtype is None else t.to(dtype)

    def logits(x, dt, pad=0, lead=0):
        """x [N, C] on the GPU in type dt, as columns of a wider buffer; and its values."""
        N, C = x.shape
        buf = torch.full((N, C + pad + lead), 7.0, dtype=e.types[dt], device="cuda")
        with np.errstate(over="ignore"):
            buf[:, lead:lead + C] = dev(x.astype(np.float32)).to(e.types[dt])
        view = buf[:, lead:lead + C]
        return view, view.float().cpu().numpy()

    def scratch(n):
        return torch.empty(n, dtype=torch.uint8, device="cuda") if n else None

    e.call, e.dev, e.logits, e.scratch = call, dev, logits, scratch
    e.nan = lambda *s: torch.full(s, math.nan, device="cuda")
    return e


class Score:
    """One token_logprobs_fwd with every output, guarded by a sentinel row."""

    def __init__(self, env, x, dt, targets, T, k, **kw):
        t = env.torch
        N, C = x.shape
        self.env, self.x, self.dt, self.T, self.k = env, x, DTYPES[dt], T, k
        self.targets = env.dev(np.asarray(targets, np.int32))
        self.logp, self.ent, self.stats = env.nan(N + 1), env.nan(N + 1), env.nan(N + 1, 4)
        self.ids = t.full((N + 1, max(k, 1)), -77, dtype=t.int32, device="cuda")
        self.top = env.nan(N + 1, max(k, 1))
        n = env.L.seeml_hip_token_logprobs_scratch(N, C, self.dt, k)
        self.scratch, self.n = env.scratch(n), n
        self.run()

    def run(self):
        N, C = self.x.shape
        self.env.call("token_logprobs_fwd", self.x, self.dt, self.x.stride(0), self.targets, self.T,
                      self.k, self.logp, self.ent, self.stats, self.ids if self.k else None,
                      self.top if self.k else None, N, C, self.scratch, self.n)

    def bits(self):
        v = [a.cpu().numpy() for a in (self.logp, self.ent, self.stats, self.ids, self.top)]
        return [a.view(np.uint32).copy() for a in v]


def close(got, want, tol, what):
    got, want = float(got), float(want)
    if abs(want) > float(np.finfo(np.float32).max):  # rounds to an infinity of float32
        want = math.copysign(math.inf, want)
    if math.isnan(want):
        assert math.isnan(got), (what, got)
    elif math.isinf(want):
        assert got == want, (what, got, want)
    else:
        assert abs(got - want) <= tol + ref.U * abs(want) + ref.TINY, (what, got, want, tol)


def check_score(s, vals, targets):
    logp, ent = s.logp.cpu().numpy(), s.ent.cpu().numpy()
    N, k = vals.shape[0], s.k
    ids, top = s.ids.cpu().numpy().reshape(-1), s.top.cpu().numpy().reshape(-1)
    ids = ids[:N * k].reshape(N, k) if k else None
    top = top[:N * k].reshape(N, k) if k else None
    for r in range(N):
        lp, h, alt, e1, e2 = ref.score_row(vals[r], s.T, int(targets[r]), k)
        close(logp[r], lp, e1 + 2 * ref.U * abs(lp) if math.isfinite(lp) else 0, ("logp", r))
        close(ent[r], h, e2, ("entropy", r))
        if k:
            assert ids[r].tolist() == [i for i, _ in alt], ("ids", r)
            for i in range(k):
                close(top[r][i], alt[i][1], e1, ("top", r, i))
    assert math.isnan(logp[N]) and math.isnan(ent[N]) and np.isnan(s.stats.cpu().numpy()[N]).all()
    if k:
        assert (s.ids.cpu().numpy().reshape(-1)[N * k:] == -77).all()


def rand_rows(N, C, seed, spread=2.0, peaks=3):
    r = np.random.default_rng(seed)
    x = r.standard_normal((N, C)) * spread
    for _ in range(peaks):
        x[np.arange(N), r.integers(0, C, N)] += r.random(N) * 9.0
    return x, r


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 3), (2, 63, 63), (5, 64, 1), (4, 65, 20), (300, 33, 5),
          (3, 255, 128), (7, 1000, 17), (2, 1999, 128), (3, 4096, 64), (5, 8191, 20), (2, 10007, 100),
          (3, 32000, 20), (1, 32768, 8), (2, 50001, 33), (1, 131072, 128), (2, 140003, 8),
          (1100, 300, 7), (1100, 1999, 32), (1100, 600, 33), (66, 66001, 40), (9, 65536, 127)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,C,k", SHAPES)
def test_scores(env, N, C, k, dt):
    x, r = rand_rows(N, C, N * 1000 + C)
    for pad, lead, T in ((0, 0, 1.0), (5, 3, 0.7)):
        v, vals = env.logits(x, dt, pad, lead)
        t = r.integers(-1, C, N)
        s = Score(env, v, dt, t, T, k)
        check_score(s, vals, t)
        first = s.bits()
        s.run()
        assert all(np.array_equal(a, b) for a, b in zip(first, s.bits())), "bits differ"


@pytest.mark.parametrize("N,C", [(1, 5), (3, 777), (2, 9001), (2, 40000), (1, 150001)])
@pytest.mark.parametrize("kind", ["equal", "zeros", "up", "down", "whole", "stripe", "two_values",
                                  "few", "lowest", "one_column", "late"])
def test_top_classes_of_rows_made_against_the_selection(env, kind, N, C):
    """Ties, order, masks and layouts that crowd the candidates together."""
    r = np.random.default_rng(C)
    j = np.arange(C)
    low = float(np.finfo(np.float32).min)
    row = {
        "equal": np.full(C, -3.25), "zeros": np.where(j % 2, 0.0, -0.0), "up": j * 1e-3,
        "down": -j * 1e-3, "whole": r.integers(0, 4, C).astype(float),
        "stripe": np.where(j % 1024 < 4, 5.0 + j * 1e-5, r.standard_normal(C)),
        "two_values": np.where(r.random(C) < 0.5, 1.0, 1.0 + 2.0 ** -20),
        "few": np.where(j % (C // 3 + 1) == 1, 1.0 + j * 1e-4, -np.inf),
        "lowest": np.where(j % (C // 3 + 1) == 1, 1.0 + j * 1e-4, low),
        "one_column": np.where(j % 256 == 7 % C, 3.0 + j * 1e-6, -50.0),
        "late": np.where(j >= C - 300, 20.0 + (j - C) * 1e-3, -5.0),
    }[kind]
    x = np.broadcast_to(row, (N, C))
    for dt in ("f32", "bf16"):
        if dt == "bf16" and kind == "lowest":
            low = float(env.torch.finfo(env.torch.bfloat16).min)
            x = np.where(x < -1e38, low, x)
        v, vals = env.logits(x, dt)
        for k in (1, min(5, C), min(128, C)):
            t = np.full(N, C - 1)
            check_score(Score(env, v, dt, t, 1.0, k), vals, t)


def test_rows_without_a_distribution(env):
    """NaN, +inf, all masked, all but one masked, all at the lowest value."""
    for C in (3, 300, 5000, 40001):
        x, r = rand_rows(9, C, C)
        x[0, C // 2] = np.nan
        x[1, C - 1] = np.inf
        x[2, :] = -np.inf
        x[3, :] = -np.inf
        x[3, C // 3] = -4.0
        x[4, :] = np.finfo(np.float32).min
        x[5, :] = np.inf
        x[6, :] = -np.inf
        x[6, 0] = np.nan
        x[7, 1:] = -np.inf
        t = np.array([0, 0, 1, C // 3, 0, 0, -1, C, C - 1])
        for dt in ("f32", "bf16", "f16"):
            if dt != "f32":
                x[4, :] = float(env.torch.finfo(env.types[dt]).min)
            v, vals = env.logits(x, dt)
            for T in (1.0, 1e-3, 50.0):
                check_score(Score(env, v, dt, t, T, min(C, 9)), vals, t)


def test_extreme_values_and_temperatures(env):
    big = float(np.finfo(np.float32).max)
    x = np.array([[big, -big, 0.0, 1.0], [-big, -big, -big, -np.inf], [1e30, 1e30, -1e30, 5.0],
                  [1e-40, 0.0, -1e-40, 2e-40], [88.0, -88.0, 700.0, -700.0]])
    v, vals = env.logits(x, "f32")
    t = np.array([1, 0, 1, 3, 0])
    for T in (1.0, 1e-30, 1e30, 3e-7, 1e5):
        check_score(Score(env, v, "f32", t, T, 4), vals, t)


def test_outputs_left_out_do_not_change_the_others(env):
    t = env.torch
    x, r = rand_rows(6, 3001, 4)
    v, vals = env.logits(x, "f32")
    tg = r.integers(0, 3001, 6)
    s = Score(env, v, "f32", tg, 1.0, 10)
    N, C = x.shape
    ent, logp = env.nan(N), env.nan(N)
    n0 = env.L.seeml_hip_token_logprobs_scratch(N, C, 0, 0)
    sc = env.scratch(n0)
    env.call("token_logprobs_fwd", v, 0, C, None, 1.0, 0, None, ent, None, None, None, N, C, sc, n0)
    env.call("token_logprobs_fwd", v, 0, C, s.targets, 1.0, 0, logp, None, None, None, None, N, C, sc, n0)
    ids, top = t.empty(N, 10, dtype=t.int32, device="cuda"), env.nan(N, 10)
    env.call("token_logprobs_fwd", v, 0, C, None, 1.0, 10, None, None, None, ids, top, N, C,
             s.scratch, s.n)
    assert t.equal(ent, s.ent[:N]) and t.equal(logp, s.logp[:N])
    assert t.equal(ids, s.ids[:N]) and t.equal(top, s.top[:N])


def check_grad(got, want, tol, dt, what=""):
    """Elementwise: the 32-bit bound, then one rounding to the gradient's type."""
    got = got.astype(np.float64)
    fine = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all(), what
    off = np.abs(got - want)[fine]
    lim = (tol + ref.HALF_STEP[dt] * (np.abs(want) + tol) + ref.SMALLEST[dt])[fine]
    assert (off <= lim).all(), (what, int(np.argmax(off - lim)), float((off / lim).max()))


GRADS = [(1, 1), (2, 2), (3, 7), (70, 65), (4, 1000), (3, 1999), (2, 8191), (2, 32000), (1, 131073),
         (2, 70001)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,C", GRADS)
def test_score_gradients(env, N, C, dt):
    t = env.torch
    x, r = rand_rows(N, C, C + N)
    if C > 5:
        x[0, C // 2] = -np.inf
    v, vals = env.logits(x, dt, 3, 2)
    tg = r.integers(-1, C, N)
    up, ent = r.standard_normal(N).astype(np.float32), r.standard_normal(N).astype(np.float32)
    s = Score(env, v, dt, tg, 1.3, 0)
    for a, b in ((up, ent), (up, None), (None, ent)):
        buf = t.full((N, C + 4), 9.0, dtype=env.types[dt], device="cuda")
        dx = buf[:, 1:1 + C]
        env.call("token_logprobs_bwd", v, DTYPES[dt], v.stride(0), s.targets, 1.3, s.stats,
                 env.dev(a) if a is not None else None, env.dev(b) if b is not None else None, dx,
                 C + 4, N, C)
        got = dx.float().cpu().numpy()
        for i in range(N):
            want, tol = ref.score_grad_row(vals[i], 1.3, int(tg[i]), 0.0 if a is None else float(a[i]),
                                           0.0 if b is None else float(b[i]))
            check_grad(got[i], want, tol, dt, (i, a is None, b is None))
        edge = buf.float().cpu().numpy()
        assert (edge[:, 0] == 9.0).all() and (edge[:, 1 + C:] == 9.0).all()
    # in place: the logits become the gradient, bit for bit
    w = v.clone()
    wide = t.full((N, C + 5), 7.0, dtype=env.types[dt], device="cuda")
    wide[:, 2:2 + C] = w
    inside = wide[:, 2:2 + C]
    a, b = env.dev(up), env.dev(ent)
    ref_dx = t.empty(N, C, dtype=env.types[dt], device="cuda")
    env.call("token_logprobs_bwd", inside, DTYPES[dt], C + 5, s.targets, 1.3, s.stats, a, b, ref_dx, C, N, C)
    env.call("token_logprobs_bwd", inside, DTYPES[dt], C + 5, s.targets, 1.3, s.stats, a, b, inside,
             C + 5, N, C)
    assert t.equal(inside.contiguous().view(t.uint8), ref_dx.view(t.uint8))
    assert (wide[:, :2] == 7.0).all() and (wide[:, 2 + C:] == 7.0).all()


def test_score_gradients_of_rows_without_a_distribution(env):
    for C in (5, 3000):
        x, r = rand_rows(6, C, 8)
        x[0, 1] = np.nan
        x[1, :] = -np.inf
        x[2, 0] = np.inf
        x[3, :] = -np.inf
        x[3, 2] = 1.0
        v, vals = env.logits(x, "f32")
        tg = np.array([0, 1, 1, 2, C, -1])
        s = Score(env, v, "f32", tg, 1.0, 0)
        up, ent = np.ones(6, np.float32), np.full(6, 0.5, np.float32)
        dx = env.nan(6, C)
        env.call("token_logprobs_bwd", v, 0, C, s.targets, 1.0, s.stats, env.dev(up), env.dev(ent),
                 dx, C, 6, C)
        got = dx.cpu().numpy()
        for i in range(6):
            want, tol = ref.score_grad_row(vals[i], 1.0, int(tg[i]), 1.0, 0.5)
            check_grad(got[i], want, tol, "f32", i)


# ---- distillation ------------------------------------------------------------


def teacher(x, r, T, k, noise=0.7):
    """The k likeliest classes of a noisy copy of x [N, C], at temperature T."""
    z = (x + noise * r.standard_normal(x.shape)) / T
    z = np.where(np.isnan(z) | np.isinf(z), -1e4, z)
    lp = z - z.max(1, keepdims=True)
    lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
    ids = np.argsort(-lp, axis=1, kind="stable")[:, :k]
    return ids.astype(np.int32), np.take_along_axis(lp, ids, 1).astype(np.float32)


class Distill:
    def __init__(self, env, x, dt, ids, v, weight, T, tail, seed=None):
        t = env.torch
        N, C = x.shape
        self.env, self.x, self.dt, self.T, self.tail = env, x, dt, T, tail
        self.ids, self.v = env.dev(ids), env.dev(v)
        self.k = ids.shape[1]
        self.weight = env.dev(np.asarray(weight, np.float32)) if weight is not None else None
        self.seed = env.dev(np.array([seed], np.float32)) if seed is not None else None
        self.loss, self.rows, self.stats = env.nan(2), env.nan(N + 1), env.nan(N + 1, 8)
        self.wide = t.full((N, C + 6), 9.0, dtype=env.types[dt], device="cuda")
        self.dx = self.wide[:, 3:3 + C]
        self.n = env.L.seeml_hip_topk_distill_scratch(N, C, DTYPES[dt], self.k)
        self.scratch = env.scratch(self.n)

    def head(self):
        return (self.x, DTYPES[self.dt], self.x.stride(0), self.ids, self.v, self.k, self.weight)

    def two(self):
        N, C = self.x.shape
        self.env.call("topk_distill_fwd", *self.head(), self.T, self.tail, self.loss, self.rows,
                      self.stats, N, C, self.scratch, self.n)
        self.env.call("topk_distill_bwd", *self.head(), self.seed, self.T, self.tail, self.stats,
                      self.dx, C + 6, N, C)
        return self

    def one(self):
        N, C = self.x.shape
        self.env.call("topk_distill_fwd_bwd", *self.head(), self.seed, self.T, self.tail, self.loss,
                      self.rows, self.dx, C + 6, N, C, self.scratch, self.n)
        return self

    def bits(self):
        t = self.env.torch
        return [a.contiguous().view(t.uint8).cpu().numpy().copy()
                for a in (self.loss, self.rows, self.wide)]


def check_distill(d, vals, ids, v, weight, seed, what=""):
    N, C = vals.shape
    w = np.full(N, 1.0 / N) if weight is None else np.asarray(weight, np.float32).astype(np.float64)
    up = 1.0 if seed is None else float(np.float32(seed))
    rows, got = d.rows.cpu().numpy(), d.dx.float().cpu().numpy()
    total = bound = 0.0
    for r in range(N):
        if w[r] == 0.0:
            assert rows[r] == 0.0 and (got[r] == 0.0).all(), (what, r)
            continue
        L, g, L_tol, tol = ref.distill_row(vals[r], ids[r], v[r], d.T, d.tail)
        close(rows[r], L, L_tol, (what, "row", r))
        s = w[r] * up
        check_grad(got[r], g * s, (tol + 4 * ref.U * np.abs(g)) * abs(s), d.dt, (what, r))
        total += w[r] * L
        bound += abs(w[r]) * (L_tol + ref.U * abs(L)) if math.isfinite(L) else 0.0
    close(d.loss.cpu().numpy()[0], total, bound, (what, "loss"))
    assert math.isnan(d.loss[1].item()) and math.isnan(d.rows[N].item())
    wide = d.wide.float().cpu().numpy()
    assert (wide[:, :3] == 9.0).all() and (wide[:, 3 + C:] == 9.0).all()


DISTILL = [(1, 1, 1), (2, 2, 1), (3, 7, 7), (65, 40, 3), (4, 300, 128), (5, 1999, 50), (3, 8192, 16),
           (2, 10007, 128), (2, 32000, 64), (2, 32769, 5), (1, 65536, 20), (2, 66000, 9),
           (1, 131072, 100), (2, 131075, 30), (1100, 1500, 9), (2, 40000, 12), (66, 70001, 5),
           (9, 65536, 65)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,C,k", DISTILL)
def test_distillation(env, N, C, k, dt):
    x, r = rand_rows(N, C, N + C)
    for tail, T, pad in ((1, 2.0, 0), (0, 0.8, 5)):
        vv, vals = env.logits(x, dt, pad, pad // 2)
        ids, v = teacher(vals, r, T, k)
        perm = r.permutation(k)
        ids, v = ids[:, perm].copy(), v[:, perm].copy()
        if k > 2:
            ids[0, :k // 2] = -1
        w = r.random(N).astype(np.float32)
        if N > 2:
            w[1] = 0.0
        for weight, seed in ((w, 1.7), (None, None)):
            d = Distill(env, vv, dt, ids, v, weight, T, tail, seed).two()
            check_distill(d, vals, ids, v, weight, seed, "two calls")
            first = d.bits()
            d.two()
            assert all(np.array_equal(a, b) for a, b in zip(first, d.bits()))
            d = Distill(env, vv, dt, ids, v, weight, T, tail, seed).one()
            check_distill(d, vals, ids, v, weight, seed, "one call")
            first = d.bits()
            d.one()
            assert all(np.array_equal(a, b) for a, b in zip(first, d.bits()))


@pytest.mark.parametrize("C", [6, 700, 9000, 40000])
def test_distillation_lists_and_rows_that_are_no_distribution(env, C):
    """Each row: what is wrong with it, and what the header says of it."""
    N, k = 16, 5
    x, r = rand_rows(N, C, C)
    ids, v = teacher(x, r, 1.0, k)
    ids[0, 2] = C                       # no class: NaN
    ids[1, 3] = ids[1, 0]               # twice: NaN
    v[2, 1] = np.nan                    # NaN
    v[3, 0] = np.inf                    # NaN
    v[4, 1] = -np.inf                   # a class without mass
    ids[5, :] = -1                      # no entries: 0
    x[6, C // 2] = np.nan               # NaN
    x[7, :] = -np.inf                   # +inf, zero gradient
    x[8, ids[8, 0]] = -np.inf           # a listed class masked: +inf
    out = np.setdiff1d(np.arange(C), ids[9])
    x[9, out] = -np.inf                 # nothing outside the list
    v[10, :] = -np.inf                  # no mass at all
    ids[11, 1:] = -7                    # one entry, empties of another value
    v[11, 1:] = np.nan                  # ... whose values are not read
    x[12, out[:1]] = np.inf             # NaN
    x[13, ids[13]] = -np.inf            # every listed class masked
    v[14, :] += 0.5                     # more mass than one
    ids[15, 0], ids[15, 1] = 2 ** 31 - 1, -2 ** 31  # NaN
    for tail in (0, 1):
        for dt in ("f32", "bf16"):
            vv, vals = env.logits(x, dt)
            for form in ("two", "one"):
                d = Distill(env, vv, dt, ids, v, np.ones(N, np.float32), 1.0, tail, 0.5)
                getattr(d, form)()
                rows, got = d.rows.cpu().numpy(), d.dx.float().cpu().numpy()
                for i in range(N):
                    L, g, L_tol, tol = ref.distill_row(vals[i], ids[i], v[i], 1.0, tail)
                    close(rows[i], L, L_tol, (form, tail, i))
                    check_grad(got[i], 0.5 * g, 0.5 * (tol + 4 * ref.U * np.abs(g)), dt,
                               (form, tail, i))
                assert math.isnan(d.loss[0].item())
                # a weight of 0 takes the bad rows out of the sum and the gradient
                w = np.where([not math.isfinite(float(a)) for a in rows], 0.0, 0.25)
                d = Distill(env, vv, dt, ids, v, w, 1.0, tail, 0.5)
                getattr(d, form)()
                check_distill(d, vals, ids, v, w, 0.5, (form, tail, "weighted"))


@pytest.mark.parametrize("C", [6, 2000, 33000])
def test_distillation_weights_and_temperatures(env, C):
    """Weights below zero and NaN; temperatures from the coldest to the hottest."""
    N, k = 4, 3
    x, r = rand_rows(N, C, C + 1)
    w = np.array([-0.5, 0.0, 2.0, 1.0], np.float32)
    for T in (1e-30, 1e-3, 40.0, 1e30):
        vv, vals = env.logits(x, "f32")
        ids, v = teacher(vals, r, max(T, 1e-2), k)
        for tail in (0, 1):
            for form in ("two", "one"):
                d = Distill(env, vv, "f32", ids, v, w, T, tail, 0.75)
                getattr(d, form)()
                check_distill(d, vals, ids, v, w, 0.75, (T, tail, form))
    w[3] = np.nan
    for form in ("two", "one"):
        d = Distill(env, vv, "f32", ids, v, w, 1.0, 1)
        getattr(d, form)()
        got = d.dx.cpu().numpy()
        assert np.isnan(got[3]).all() and np.isfinite(got[:3]).all() and math.isnan(d.loss[0].item())
        assert np.isfinite(d.rows.cpu().numpy()[:N]).all()


@pytest.mark.parametrize("C,dt", [(20000003, "f32"), (70000001, "bf16")])
def test_very_wide_rows(env, C, dt):
    t = env.torch
    N, k = 2, 40
    g = t.Generator(device="cuda")
    g.manual_seed(C)
    v = (t.randn(N, C, generator=g, device="cuda") * 2.0).to(env.types[dt])
    v[0, C - 2], v[1, 1] = 30.0, 25.0
    tg = np.array([C - 1, 5])
    s = Score(env, v, dt, tg, 1.0, k)
    lp = t.log_softmax(v.double(), -1)
    # every term that counts is above 2^-45 of the maximum: |d| <= 45
    lim = ref.U * (70.0 + 5.0 * 45.0)
    got = s.logp[:N].double()
    want = lp.gather(1, t.from_numpy(tg).cuda()[:, None])[:, 0]
    assert ((got - want).abs() <= lim + 2 * ref.U * want.abs()).all()
    h = -(lp.exp() * lp).sum(-1)
    assert ((s.ent[:N].double() - h).abs() <= 45 * lim + 2 * ref.U * h).all()
    top = t.sort(v.float(), dim=-1, descending=True, stable=True)
    assert t.equal(s.ids[:N].long(), top.indices[:, :k])
    del top
    dx = t.empty_like(v)
    up = t.tensor([0.5, -2.0], device="cuda")
    env.call("token_logprobs_bwd", v, DTYPES[dt], C, s.targets, 1.0, s.stats, up, None, dx, C, N, C)
    p = lp.exp()
    want = -up[:, None] * p
    want[t.arange(N), t.from_numpy(tg).cuda()] += up
    # |d| up to 60, relative to p; and one rounding to the type
    off = (dx.double() - want).abs()
    assert (off <= want.abs() * (ref.U * 500 + 2 * lim + ref.HALF_STEP[dt]) + ref.SMALLEST[dt]).all()
    del want, off
    ids, q = lp.topk(k, -1).indices.int(), lp.topk(k, -1).values.float()
    d = Distill(env, v, dt, ids.cpu().numpy(), q.cpu().numpy(), None, 1.0, 1).one()
    # a student that is its own teacher: no loss, no gradient
    assert d.rows[:N].abs().max().item() <= 3 * lim
    assert (d.dx.double().abs() <= p * (ref.U * 500 + 6 * lim) / N + ref.SMALLEST[dt]).all()


@pytest.mark.parametrize("C", [50, 5000, 33000])
def test_a_tail_far_below_the_listed_classes_keeps_its_digits(env, C):
    """The student gives the unlisted classes e^-80, e^-200 and e^-600."""
    r = np.random.default_rng(C)
    N, k = 3, 4
    x = r.standard_normal((N, C))
    ids = np.argsort(r.random((N, C)), axis=1)[:, :k].astype(np.int32)
    for i, gap in enumerate((80.0, 200.0, 600.0)):
        x[i, ids[i]] += gap
    v = np.log(np.tile([0.4, 0.3, 0.15, 0.1], (N, 1))).astype(np.float32)
    vv, vals = env.logits(x, "f32")
    for form in ("two", "one"):
        d = Distill(env, vv, "f32", ids, v, np.ones(N, np.float32), 1.0, 1)
        getattr(d, form)()
        check_distill(d, vals, ids, v, np.ones(N), None, form)
        assert np.abs(d.dx.cpu().numpy()).sum(1).min() > 0.05


@pytest.mark.parametrize("N,C", [(3, 500), (2, 20000), (1, 131073), (300, 1000)])
def test_distillation_in_place(env, N, C):
    t = env.torch
    x, r = rand_rows(N, C, 5)
    ids, v = teacher(x, r, 1.0, 9)
    w = r.random(N).astype(np.float32)
    w[-1] = 0.0 if N > 1 else w[-1]
    for dt in ("f32", "bf16"):
        vv, _ = env.logits(x, dt)
        d = Distill(env, vv, dt, ids, v, w, 1.0, 1, 1.5).one()
        inside = vv.clone()
        d2 = Distill(env, inside, dt, ids, v, w, 1.0, 1, 1.5)
        env.call("topk_distill_fwd_bwd", *d2.head(), d2.seed, 1.0, 1, d2.loss, d2.rows, inside, C, N,
                 C, d2.scratch, d2.n)
        assert t.equal(inside.view(t.uint8), d.dx.contiguous().view(t.uint8))
        assert t.equal(d.rows[:N], d2.rows[:N]) and d.loss[0] == d2.loss[0]
        d.two()
        inside = vv.clone()
        d3 = Distill(env, inside, dt, ids, v, w, 1.0, 1, 1.5)
        env.call("topk_distill_fwd", *d3.head(), 1.0, 1, d3.loss, d3.rows, d3.stats, N, C,
                 d3.scratch, d3.n)
        env.call("topk_distill_bwd", *d3.head(), d3.seed, 1.0, 1, d3.stats, inside, C, N, C)
        assert t.equal(inside.view(t.uint8), d.dx.contiguous().view(t.uint8))


def test_gradient_beside_the_logits_in_one_buffer(env):
    t = env.torch
    N, C, k = 5, 601, 7
    x, r = rand_rows(N, C, 6)
    ids, v = teacher(x, r, 1.0, k)
    wide = t.full((N, 2 * C + 3), 4.0, device="cuda")
    wide[:, :C] = env.dev(x.astype(np.float32))
    d = Distill(env, wide[:, :C], "f32", ids, v, None, 1.0, 1).one()
    keep = wide.clone()
    env.call("topk_distill_fwd_bwd", *d.head(), None, 1.0, 1, d.loss, d.rows, wide[:, C + 1:],
             wide.stride(0), N, C, d.scratch, d.n)
    assert t.equal(wide[:, C + 1:2 * C + 1], d.dx)
    keep[:, C + 1:2 * C + 1] = d.dx
    assert t.equal(wide, keep)


def test_a_score_feeds_the_distillation(env):
    """The chain: a teacher's pass is scored, its lists are what the student
    learns from. A student equal to the teacher has no loss and no gradient;
    one step against the gradient brings another one nearer."""
    t = env.torch
    N, C, k, T = 40, 3001, 24, 1.6
    x, r = rand_rows(N, C, 12)
    tv, tvals = env.logits(x, "f32")
    s = Score(env, tv, "f32", np.zeros(N), T, k)
    check_score(s, tvals, np.zeros(N))
    ids, lp = s.ids[:N].cpu().numpy(), s.top[:N].cpu().numpy()
    for tail in (0, 1):
        d = Distill(env, tv, "f32", ids, lp, None, T, tail).one()
        check_distill(d, tvals, ids, lp, None, None, ("itself", tail))
        if tail:
            assert abs(d.loss[0].item()) < 1e-5 and d.dx.abs().max().item() < 1e-5
        sv, svals = env.logits(x + 0.8 * r.standard_normal((N, C)), "f32")
        d = Distill(env, sv, "f32", ids, lp, None, T, tail).one()
        check_distill(d, svals, ids, lp, None, None, ("other", tail))
        before = d.loss[0].item()
        sv -= 0.5 * N * d.dx
        assert d.one().loss[0].item() < before
        # differences of the loss along a direction
        u = env.dev(r.standard_normal((N, C)).astype(np.float32))
        g = (d.dx * u).double().sum().item()
        h = 2.0 ** -6
        base = sv.clone()
        val = []
        for sign in (1, -1):
            sv.copy_(base + sign * h * u)
            val.append(d.one().loss[0].item())
        # central difference: third derivatives of a softmax loss are below 1 per
        # unit of u^3; each loss is off by less than 1e-6
        lim = h * h * float((u.abs() ** 3).amax()) + 2e-6 / (2 * h)
        assert abs((val[0] - val[1]) / (2 * h) - g) <= lim


# ---- streams and graphs -------------------------------------------------------


def test_another_stream(env):
    t = env.torch
    x, r = rand_rows(9, 20011, 2)
    v, vals = env.logits(x, "f32")
    tg = r.integers(0, 20011, 9)
    ids, lp = teacher(x, r, 1.0, 8)
    t.cuda.synchronize()
    side = t.cuda.Stream()
    with t.cuda.stream(side):
        s = Score(env, v, "f32", tg, 1.0, 12)
        d = Distill(env, v, "f32", ids, lp, None, 1.0, 1).one()
    side.synchronize()
    check_score(s, vals, tg)
    check_distill(d, vals, ids, lp, None, None)


@pytest.mark.parametrize("N,C,dt", [(3, 40000, "f32"), (64, 1500, "bf16"), (1, 131072, "bf16")])
def test_captured_calls_replay_with_new_inputs(env, N, C, dt):
    """Two graphs, each with scratch of its own, replayed in turn with eager
    work between; every replay gives the eager bits of the inputs it then has."""
    t = env.torch
    k = 20
    sets = []
    for seed in range(3):
        x, r = rand_rows(N, C, 50 + seed)
        ids, lp = teacher(x, r, 1.0, k)
        sets.append((env.logits(x, dt)[0], ids, lp, r.integers(0, C, N).astype(np.int32)))

    def fresh(i):
        v, ids, lp, tg = sets[i]
        return (Score(env, v.clone(), dt, tg, 1.0, k),
                Distill(env, v.clone(), dt, ids, lp, None, 1.0, 1, 0.5),
                Distill(env, v.clone(), dt, ids, lp, None, 1.0, 0, 0.5))

    def passes(s, one, two):
        s.run()
        one.one()
        two.two()

    want = []
    for i in range(3):
        g = fresh(i)
        passes(*g)
        want.append([a.bits() for a in g])
    t.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = fresh(0)
        passes(*g)
        t.cuda.synchronize()
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            passes(*g)
        graphs.append((graph, g))
    for turn in range(6):
        for n, (graph, g) in enumerate(graphs):
            i = (turn + n) % 3
            v, ids, lp, tg = sets[i]
            s, one, two = g
            s.targets.copy_(env.dev(tg))
            for a in g:
                a.x.copy_(v)
            for a in (one, two):
                a.ids.copy_(env.dev(ids))
                a.v.copy_(env.dev(lp))
                a.wide.fill_(9.0)
                a.loss.fill_(math.nan)
            s.ids.fill_(-77)
            (v.float() * 2).sum().item()  # eager work and a wait between replays
            graph.replay()
            t.cuda.synchronize()
            for a, b in zip(g, want[i]):
                assert all(np.array_equal(p, q) for p, q in zip(a.bits(), b)), (turn, n)


def test_two_streams_at_once(env):
    """Calls that overlap on two streams, each with scratch of its own."""
    t = env.torch
    x, r = rand_rows(4, 100003, 3)
    ids, lp = teacher(x, r, 1.0, 16)
    v, vals = env.logits(x, "f32")
    tg = r.integers(0, 100003, 4)
    work = []
    for _ in range(2):
        s = Score(env, v.clone(), "f32", tg, 1.0, 16)
        d = Distill(env, v.clone(), "f32", ids, lp, None, 1.0, 1).one()
        t.cuda.synchronize()
        want = s.bits() + d.bits()
        work.append((t.cuda.Stream(), s, d, want))
    t.cuda.synchronize()
    for _ in range(20):
        for st, s, d, _ in work:
            with t.cuda.stream(st):
                s.run()
                d.one()
    t.cuda.synchronize()
    for _, s, d, want in work:
        assert all(np.array_equal(a, b) for a, b in zip(s.bits() + d.bits(), want))


def test_two_host_threads(env):
    """Entries called from two threads at once, each on a stream of its own; one
    thread's refusals do not show in the other."""
    import threading
    t = env.torch
    jobs, failed = [], []
    for seed in range(2):
        x, r = rand_rows(3, 9001 + seed, 70 + seed)
        v, _ = env.logits(x, "f32")
        s = Score(env, v, "f32", r.integers(0, 9001, 3), 1.0, 11)
        ids, lp = teacher(x, r, 1.0, 5)
        d = Distill(env, v, "f32", ids, lp, None, 1.0, 1).one()
        jobs.append((t.cuda.Stream(), s, d, s.bits() + d.bits()))
    t.cuda.synchronize()

    def work(stream, s, d, want):
        try:
            with t.cuda.stream(stream):
                for i in range(50):
                    s.run()
                    d.one()
                    if i % 10 == 0:
                        rc = env.L.seeml_hip_token_logprobs_scratch(1, 1, 0, 2)
                        assert rc == 0
            stream.synchronize()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
    for _, s, d, want in jobs:
        assert all(np.array_equal(a, b) for a, b in zip(s.bits() + d.bits(), want))


def test_offsets_past_32_bits(env):
    """Rows of a wide buffer more than 2^32 elements apart in all: 2^33 bytes of
    16-bit logits, of which five rows are used."""
    t = env.torch
    C, stride, N = 2000, 1 << 30, 5
    buf = t.empty((N - 1) * stride + C, dtype=t.bfloat16, device="cuda")
    v = t.as_strided(buf, (N, C), (stride, 1))
    x, r = rand_rows(N, C, 9)
    v.copy_(env.dev(x.astype(np.float32)))
    vals = v.float().cpu().numpy()
    tg = r.integers(0, C, N)
    check_score(Score(env, v, "bf16", tg, 1.0, 6), vals, tg)
    ids, lp = teacher(x, r, 1.0, 6)
    d = Distill(env, v, "bf16", ids, lp, None, 1.0, 1).one()
    check_distill(d, vals, ids, lp, None, None)
    d = Distill(env, v, "bf16", ids, lp, None, 1.0, 1)
    want = Distill(env, v, "bf16", ids, lp, None, 1.0, 1).one()
    env.call("topk_distill_fwd_bwd", *d.head(), None, 1.0, 1, d.loss, d.rows, v, stride, N, C,
             d.scratch, d.n)
    assert t.equal(v.contiguous(), want.dx.contiguous())


def test_many_rows(env):
    """More rows than a grid has processors, by the sum of a few checks."""
    t = env.torch
    N, C = 70000, 6
    x, r = rand_rows(N, C, 10)
    v, vals = env.logits(x, "f32")
    tg = r.integers(0, C, N)
    s = Score(env, v, "f32", tg, 1.0, 2)
    lp = t.log_softmax(v.double(), -1)
    # bound: the reference's for C = 6 and |d| <= 30
    lim = ref.U * (70.0 + 5.0 * 3.0) + 40 * ref.U
    assert (s.logp[:N] - lp.gather(1, s.targets.long()[:, None])[:, 0]).abs().max().item() < lim
    assert t.equal(s.ids[:N, 0].long(), v.argmax(-1))
    ids, q = teacher(x, r, 1.0, 2)
    d = Distill(env, v, "f32", ids, q, None, 1.0, 1).one()
    some = [0, 1, 255, 256, 65535, 65536, N - 1]
    rows, got = d.rows.cpu().numpy(), d.dx.cpu().numpy()
    for i in some:
        L, g, L_tol, tol = ref.distill_row(vals[i], ids[i], q[i], 1.0, 1)
        close(rows[i], L, L_tol, i)
        check_grad(got[i] * N, g, tol + 8 * ref.U * np.abs(g), "f32", i)
    close(d.loss[0].item(), rows[:N].astype(np.float64).mean(), 1e-9, "loss")
