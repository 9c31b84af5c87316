"""Distillation steps of the engine on the lists of rows that do not count."""
import numpy as np
import pytest

from helpers import compile_workload
from seeml_amd import PROGRAM_TRAIN, configs
from test_gpu_scores_engine import engine, lists, torch_gpu  # noqa: F401

pytestmark = pytest.mark.gpu


def state(e, p):
    return e.read(0, p.header["persistent_size"] // 4).view(np.uint32)


def test_lists_of_rows_without_weight_are_not_looked_at(torch_gpu):  # noqa: F811
    """Host lists as device lists: a row of weight 0 may hold anything."""
    up = lambda z: torch_gpu.from_numpy(np.ascontiguousarray(z)).cuda()  # noqa: E731
    w, p = compile_workload("c3s")
    host, dev, plain = engine(p), engine(p), engine(p)
    x, _ = configs.batch(w, 0)
    rows, C = host.softmax_shape(PROGRAM_TRAIN)
    ids, v = lists(host, x, 4, 1.0)
    weight = np.full(rows, 1.0 / rows, np.float32)
    weight[1::3] = 0.0
    bad, badv = ids.copy(), v.copy()
    bad[1::3, 0] = C
    bad[1::3, 2] = 2 ** 31 - 1
    badv[1::3] = np.nan
    want = plain.distill_step(x, ids, v, weight)
    assert dev.distill_step(up(x), up(bad), up(badv), up(weight)) == want
    assert host.distill_step(x, bad, badv, weight) == want
    assert np.array_equal(state(host, p), state(plain, p))
    assert np.array_equal(state(dev, p), state(plain, p))
    # a row that counts is still refused, before anything runs
    bad = ids.copy()
    bad[0, 1] = C
    with pytest.raises(RuntimeError, match="outside"):
        host.distill_step(x, bad, v, weight)
    bad = ids.copy()
    bad[1, 1] = C
    with pytest.raises(RuntimeError, match="outside"):  # no weights: every row counts
        host.distill_step(x, bad, v)
    assert host.step == 1 and np.array_equal(state(host, p), state(plain, p))
    for e in (host, dev, plain):
        e.close()
