"""The 64-bit reference of the token scores and the distillation against
differences of its own values and against closed forms."""
import math

import numpy as np
import pytest

import scores_ref as ref


def rows(seed, C):
    r = np.random.default_rng(seed)
    x = r.standard_normal(C) * 2.0
    x[r.integers(0, C)] += 5.0
    return r, x


@pytest.mark.parametrize("C,T", [(2, 1.0), (7, 0.6), (33, 2.5)])
def test_score_gradient_is_the_difference_of_its_values(C, T):
    r, x = rows(C, C)
    t = int(r.integers(0, C))
    a, b = 0.7, -0.3
    f = lambda y: a * ref.score_row(y, T, t, 0)[0] + b * ref.score_row(y, T, t, 0)[1]  # noqa: E731
    g, _ = ref.score_grad_row(x, T, t, a, b)
    h = 1e-5
    for j in range(C):
        e = np.zeros(C)
        e[j] = h
        assert abs((f(x + e) - f(x - e)) / (2 * h) - g[j]) < 1e-8


@pytest.mark.parametrize("C,k,tail", [(5, 2, 1), (5, 2, 0), (30, 7, 1), (30, 7, 0), (9, 9, 1)])
def test_distill_gradient_is_the_difference_of_its_values(C, k, tail):
    r, x = rows(C + k, C)
    T = 1.7
    tx = x + 0.5 * r.standard_normal(C)
    ids = np.argsort(-tx)[:k]
    z = tx / T
    v = (z - np.log(np.exp(z).sum()))[ids]
    ids = np.concatenate([ids, [-1]])
    v = np.concatenate([v, [0.0]])
    L, g, _, _ = ref.distill_row(x, ids, v, T, tail)
    assert L >= -1e-12
    h = 1e-5
    for j in range(C):
        e = np.zeros(C)
        e[j] = h
        d = (ref.distill_row(x + e, ids, v, T, tail)[0] - ref.distill_row(x - e, ids, v, T, tail)[0])
        assert abs(d / (2 * h) - g[j]) < 1e-8


def test_distilling_all_classes_is_the_divergence_and_none_from_itself():
    r, x = rows(3, 12)
    y = x + r.standard_normal(12)
    lp = lambda z: z - math.log(np.exp(z).sum())  # noqa: E731
    want = (np.exp(lp(y)) * (lp(y) - lp(x))).sum()
    for tail in (0, 1):
        L, _, _, _ = ref.distill_row(x, np.arange(12), lp(y), 1.0, tail)
        assert abs(L - want) < 1e-12
        ids = np.argsort(-x)[:4]
        L, g, _, _ = ref.distill_row(x, ids, lp(x)[ids], 1.0, tail)
        if tail:
            assert abs(L) < 1e-12 and np.abs(g).max() < 1e-12


def test_uniform_rows():
    lp, h, top, _, _ = ref.score_row(np.zeros(8), 3.0, 5, 3)
    assert abs(lp + math.log(8)) < 1e-15 and abs(h - math.log(8)) < 1e-15
    assert [i for i, _ in top] == [0, 1, 2]
