"""Token scores and distillation where a factor of the gradient leaves float32's
range though the gradient does not, and lists that are off by a large constant:
against the 64-bit reference (scores_ref.py)."""
import math

import numpy as np
import pytest

import scores_ref as ref
from test_gpu_scores import DTYPES, Distill, Score, check_grad, close, env, rand_rows, teacher  # noqa: F401

pytestmark = pytest.mark.gpu

FLT_MAX = float(np.finfo(np.float32).max)


def check_wide(got, want, tol, dt, what):
    """check_grad, where a gradient past float32's range is an infinity."""
    over = np.abs(want) > FLT_MAX * (1 + 2.0 ** -7)
    assert (got[over] == np.sign(want[over]) * np.inf).all(), what
    check_grad(np.where(over, 0.0, got), np.where(over, 0.0, want), np.where(over, 0.0, tol), dt, what)


def score_grad(x, T, target, up, bonus):
    """The reference's gradient and bound, with what a flush to zero takes: a
    probability below 2^-126 may count as 0."""
    want, tol = ref.score_grad_row(x, T, target, up, bonus)
    r = ref.softmax_row(x, T)
    if r["kind"] != "ok":
        return want, tol
    p = r["p"]
    lp = np.where(p > 0, np.abs(r["lp"]), 0.0)
    h = (p * lp).sum()
    lost = np.where(p < 2.0 ** -100, np.minimum(p, 2.0 ** -126), 0.0)
    return want, tol + lost * (abs(up) + abs(bonus) * (lp + h)) / T


@pytest.mark.parametrize("T", [1e-30, 1e-20, 1e-9, 1e-4, 1.0, 1e30])
@pytest.mark.parametrize("C", [5, 63, 3000, 9001])
def test_score_gradients_at_extreme_temperatures(env, C, T):  # noqa: F811
    """A class with p = 0, masked or far below, has no gradient through p,
    whatever dlogp / T and dentropy / T are."""
    N = 10
    x, r = rand_rows(N, C, C)
    x[1::2] *= T                       # rows that stay spread out at T
    x[:, 2::7] = -np.inf
    x[8, :] = -np.inf
    tg = r.integers(0, 2, N)
    tg[4] = tg[5] = -1
    tg[7] = C                          # NaN
    tg[6] = int(np.argmax(x[6]))       # the likeliest class: its p is 1 where T is small
    up = np.array([1, 1, 65536, 65536, 7, 7, 1e9, 1, 1, -3e-5], np.float32)
    ent = np.array([1, 1, 65536, -65536, -3, -3, 1e9, 1, 1, 65536], np.float32)
    for dt in ("f32", "bf16"):
        v, vals = env.logits(x, dt)
        s = Score(env, v, dt, tg, T, 0)
        for a, b in ((up, ent), (up, None), (None, ent)):
            dx = env.torch.full((N, C), 9.0, dtype=env.types[dt], device="cuda")
            env.call("token_logprobs_bwd", v, DTYPES[dt], C, s.targets, T, s.stats,
                     env.dev(a) if a is not None else None, env.dev(b) if b is not None else None,
                     dx, C, N, C)
            got = dx.float().cpu().numpy()
            for i in range(N):
                want, tol = score_grad(vals[i], T, -1 if a is None else int(tg[i]),
                                       0.0 if a is None else float(a[i]),
                                       0.0 if b is None else float(b[i]))
                check_wide(got[i], want, tol, dt, (dt, i, a is None, b is None))


@pytest.mark.parametrize("C", [6, 40, 3000, 40000, 70003])
@pytest.mark.parametrize("shift", [100.0, -100.0, 1e4, -1e4, 1e5, 1e30, -3e38])
def test_distillation_of_lists_off_by_a_constant(env, C, shift):  # noqa: F811
    """A renormalised list may be off by any constant per row: the loss and the
    gradient are those of the differences between its values, which float32
    holds. A row's gradient sums to zero."""
    N, k, T = 4, min(C, 9), 1.0
    x, r = rand_rows(N, C, C + 3)
    for dt in ("f32", "bf16"):
        vv, vals = env.logits(x, dt)
        ids, v = teacher(vals, r, T, k)
        v = (v.astype(np.float64) + shift * np.array([1.0, 0.75, 0.5, 0.3])[:, None]).astype(np.float32)
        ids[1, k // 2:] = -1
        apart = v.astype(np.float64)
        apart -= np.where(ids >= 0, apart, -np.inf).max(1, keepdims=True)
        for form in ("two", "one"):
            d = Distill(env, vv, dt, ids, v, np.ones(N, np.float32), T, 0, 0.75)
            getattr(d, form)()
            rows, got = d.rows.cpu().numpy(), d.dx.float().cpu().numpy()
            for i in range(N):
                L, g, L_tol, tol = ref.distill_row(vals[i], ids[i], apart[i], T, 0)
                close(rows[i], L, L_tol, (dt, form, "row", i))
                tol = 0.75 * (tol + 4 * ref.U * np.abs(g))
                check_grad(got[i], 0.75 * g, tol, dt, (dt, form, i))
                if dt == "f32":
                    assert abs(got[i].astype(np.float64).sum()) <= \
                        (tol + ref.U * np.abs(got[i]) + ref.TINY).sum(), (form, i)


@pytest.mark.parametrize("C", [6, 3000, 40000, 70003])
def test_distillation_whose_scale_leaves_float32(env, C):  # noqa: F811
    """w seed / T of 1e39 times a gradient of 0, or of 1e-7, is 0, or 1e32."""
    N, k, T, seed = 3, 2, 1e-30, 1e9
    x, r = rand_rows(N, C, C)
    x[:, 3::7] = -np.inf
    top = np.argmax(x, 1)
    ids = np.stack([top, (top == 0).astype(int)], 1).astype(np.int32)
    v = np.tile(np.array([0.0, -np.inf], np.float32), (N, 1))  # all of the mass at the top
    w = np.array([1.0, 0.0, 1e-9], np.float32)
    vv, vals = env.logits(x, "f32")
    for tail in (0, 1):
        for form in ("two", "one"):
            d = Distill(env, vv, "f32", ids, v, w, T, tail, seed)
            getattr(d, form)()
            assert (d.rows.cpu().numpy()[:N] == 0.0).all()
            assert (d.dx.cpu().numpy() == 0.0).all(), (tail, form)
    # a tiny gradient: two equal logits, a teacher that prefers one by 2e-7 of its mass
    x = np.full((1, C), -np.inf)
    x[0, :2] = 1.0
    ids = np.array([[0, 1]], np.int32)
    v = np.log(np.array([[0.5 + 1e-7, 0.5 - 1e-7]])).astype(np.float32)
    vv, vals = env.logits(x, "f32")
    L, g, _, tol = ref.distill_row(vals[0], ids[0], v[0], T, 0)
    for form in ("two", "one"):
        d = Distill(env, vv, "f32", ids, v, np.ones(1, np.float32), T, 0, seed)
        getattr(d, form)()
        check_wide(d.dx.cpu().numpy()[0], g * seed, (tol + 4 * ref.U * np.abs(g)) * seed, "f32", form)
        assert math.isfinite(d.rows[0].item())
