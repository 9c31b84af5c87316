"""Token scores and distillation through the engine: a compiled plan's eval
program scored against its labels, and train steps on a teacher's lists in
place of the labels, against the CPU oracle running the plan's own instructions
around a 64-bit loss."""
import numpy as np
import pytest

import scores_ref as ref
from helpers import TOL_STEP, HostPlanRunner, compile_workload, rel_err
from seeml_amd import PROGRAM_EVAL, PROGRAM_TRAIN, configs, planner

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def engine(plan, **kw):
    from seeml_amd import DeviceUpdateEngine
    return DeviceUpdateEngine(plan.blob, **kw)


def xent(words):
    return [i for i, w in enumerate(words) if w["opcode"] == planner.OP["SoftmaxXEntFwd"]][-1]


def lists(e, x, k, T):
    s = e.token_logprobs(x, None, k, T)
    return s["top_ids"], s["top_logp"]


def close(got, want, tol):
    return np.all(np.abs(np.asarray(got, np.float64) - want) <= tol)


@pytest.mark.parametrize("name", ["c1", "c3s", "c5s"])
def test_eval_scores_are_those_of_the_programs_logits(torch_gpu, name):
    t = torch_gpu
    w, p = compile_workload(name)
    e = engine(p)
    f = p.eval[xent(p.eval)]
    rows, C = f["out"][0], f["out"][1]
    assert e.softmax_shape(PROGRAM_EVAL) == (rows, C) == e.softmax_shape(PROGRAM_TRAIN)
    x, y = configs.batch(w, 3)
    for k, T in ((0, 1.0), (7, 1.0), (min(C, 40), 1.7)):
        s = e.token_logprobs(x, y, k, T)
        loss = e.loss()
        logits = e.read(f["inp"][0], rows * C).reshape(rows, C)
        for r in range(0, rows, max(1, rows // 16)):
            lp, h, top, e1, e2 = ref.score_row(logits[r], T, int(y[r]), k)
            assert close(s["logp"][r], lp, e1 + 3 * ref.U * abs(lp))
            assert close(s["entropy"][r], h, e2 + 2 * ref.U * h)
            if k:
                assert s["top_ids"][r].tolist() == [i for i, _ in top]
                assert close(s["top_logp"][r], [v for _, v in top], e1 + 3 * ref.U * 30)
        if T == 1.0:  # the program's own loss is the mean of -logp, to its bar
            assert abs(loss + s["logp"].astype(np.float64).mean()) <= TOL_STEP * abs(loss)
        d = e.token_logprobs(t.from_numpy(x).cuda(), t.from_numpy(y).cuda(), k, T)
        assert set(d) == set(s)
        for n in s:
            assert np.array_equal(d[n].cpu().numpy().view(np.uint32), s[n].view(np.uint32)), n
        u = e.token_logprobs(x, None, k, T)
        assert "logp" not in u and np.array_equal(u["entropy"], s["entropy"])
    # evaluating and scoring do not disturb each other, nor a train step
    a = e.train_step(x, y)
    e2 = engine(p)
    assert e2.train_step(x, y) == a
    n = p.header["persistent_size"] // 4
    assert np.array_equal(e.read(0, n).view(np.uint32), e2.read(0, n).view(np.uint32))
    e.close()
    e2.close()


class OracleDistill(HostPlanRunner):
    """The oracle's train program with its loss replaced by a 64-bit one."""

    def distill_step(self, plan, x, ids, v, w, T, tail):
        self.step += 1
        self.stage(x, None)
        f = xent(plan.train)
        words, n = self.programs[0]
        fwd, bwd = plan.train[f], plan.train[f + 2]
        N, C = fwd["out"][0], fwd["out"][1]
        whole = self.programs[0]
        self.programs[0] = (words[:64 * f].copy(), f)
        self.run(0)
        logits = self.read(fwd["inp"][0], N * C).reshape(N, C)
        dl, loss = np.zeros((N, C)), 0.0
        for r in range(N):
            if w[r] == 0.0:
                continue
            L, g, _, _ = ref.distill_row(logits[r], ids[r], v[r], T, tail)
            dl[r] = g * float(w[r])
            loss += float(w[r]) * L
        self.write(bwd["inp"][3], dl.astype(np.float32).reshape(-1))
        self.programs[0] = (words[64 * (f + 3):].copy(), n - f - 3)
        self.run(0)
        self.programs[0] = whole
        return loss


@pytest.mark.parametrize("name,tail,T", [("c1", 1, 1.0), ("c3s", 1, 2.0), ("c3s", 0, 1.0),
                                         ("c4s", 1, 1.3), ("c5s", 0, 2.0)])
def test_distill_steps_match_the_oracle(torch_gpu, orc, name, tail, T):
    """The adapters and moments after steps on a teacher's lists: the teacher is
    the same plan with adapters of its own. Host and device batches, graph and
    eager engines give the same bits."""
    t = torch_gpu
    w, p = compile_workload(name)
    teacher = engine(p)
    r = np.random.default_rng(4)
    for pid, pref, _, cnt in p.params:
        if pid.endswith("lora_B"):
            teacher.write(pref, (0.1 * r.standard_normal(cnt)).astype(np.float32))
    e, eager, dev = engine(p), engine(p, use_graph=False), engine(p)
    r = OracleDistill(p, orc)
    rows, C = e.softmax_shape(PROGRAM_TRAIN)
    n = p.header["persistent_size"] // 4
    k = min(16, C)
    for s in range(3):
        x, _ = configs.batch(w, 10 + s)
        ids, v = lists(teacher, x, k, T)
        weight = np.full(rows, 1.0 / rows, np.float32)
        if s == 1:  # some rows do not count, some lists are short
            weight[::3] = 0.0
            ids[1::4, k // 2:] = -1
        a = e.distill_step(x, ids, v, weight if s else None, T, bool(tail))
        b = r.distill_step(p, x, ids, v, weight, T, tail)
        assert abs(a - b) <= TOL_STEP * max(abs(b), 1e-3), (s, a, b)
        assert eager.distill_step(x, ids, v, weight if s else None, T, bool(tail)) == a
        up = lambda z: t.from_numpy(np.ascontiguousarray(z)).cuda()  # noqa: E731
        assert dev.distill_step(up(x), up(ids), up(v), up(weight) if s else None, T, bool(tail)) == a
    got = e.read(0, n)
    assert rel_err(got, r.read(0, n)) <= TOL_STEP
    for other in (eager, dev):
        assert np.array_equal(got.view(np.uint32), other.read(0, n).view(np.uint32))
    assert e.step == 3
    # ordinary steps go on from there, as on an engine that was handed the state
    x, y = configs.batch(w, 30)
    fresh = engine(p)
    fresh.write(0, got)
    fresh.set_step(3)
    assert e.train_step(x, y) == fresh.train_step(x, y)
    assert np.array_equal(e.read(0, n).view(np.uint32), fresh.read(0, n).view(np.uint32))
    for z in (teacher, e, eager, dev, fresh):
        z.close()


def test_a_marked_program_distils_to_the_same_bits(torch_gpu):
    w, p = compile_workload("c3s")
    e, m = engine(p), engine(p)
    x, y = configs.batch(w, 0)
    rows, C = e.softmax_shape(PROGRAM_TRAIN)
    ids, v = lists(e, x, 8, 1.0)
    v = v - 0.1
    m.mark_timed(PROGRAM_TRAIN, [xent(p.train)])
    e.train_step(x, y)
    m.train_step(x, y)
    assert e.distill_step(x, ids, v) == m.distill_step(x, ids, v)
    n = p.header["persistent_size"] // 4
    assert np.array_equal(e.read(0, n).view(np.uint32), m.read(0, n).view(np.uint32))
    e.close()
    m.close()


def test_refusals(torch_gpu):
    t = torch_gpu
    w, p = compile_workload("c3s")
    e = engine(p)
    x, y = configs.batch(w, 0)
    rows, C = e.softmax_shape()
    ids, v = lists(e, x, 4, 1.0)
    n = p.header["persistent_size"] // 4
    before = e.read(0, n)
    for kw, text in ((dict(k=129), "bad list"), (dict(k=C + 1), "bad list"),
                     (dict(temperature=0.0), "temperature")):
        with pytest.raises(RuntimeError, match=text):
            e.token_logprobs(x, y, **kw)
    with pytest.raises(RuntimeError, match="size does not match"):
        e.token_logprobs(x[:-1], y)
    with pytest.raises(RuntimeError, match="size does not match"):
        e.token_logprobs(x, y[:-1])
    with pytest.raises(RuntimeError, match="outside"):
        e.token_logprobs(x, np.full_like(y, C))
    with pytest.raises(ValueError, match="different memory"):
        e.token_logprobs(x, t.from_numpy(y).cuda())
    bad = ids.copy()
    bad[1, 2] = C
    with pytest.raises(RuntimeError, match="outside"):
        e.distill_step(x, bad, v)
    with pytest.raises(RuntimeError, match="temperature"):
        e.distill_step(x, ids, v, temperature=float("nan"))
    with pytest.raises(ValueError, match="t_ids and t_logp"):
        e.distill_step(x, ids[:-1], v[:-1])
    with pytest.raises(ValueError, match="row_weight"):
        e.distill_step(x, ids, v, np.ones(rows - 1, np.float32))
    with pytest.raises(ValueError, match="host memory"):
        e.distill_step(t.from_numpy(x).cuda(), ids, v)
    with pytest.raises(ValueError, match="type"):
        e.distill_step(t.from_numpy(x).cuda(), t.from_numpy(ids).long().cuda(), t.from_numpy(v).cuda())
    assert e.step == 0 and np.array_equal(e.read(0, n), before)
    # a list that stands twice poisons the loss: the step aborts like any other
    bad = ids.copy()
    bad[0, 1] = bad[0, 0]
    with pytest.raises(RuntimeError, match="non-finite"):
        e.distill_step(x, bad, v)
    e.close()
    for name, text in (("c2s", "no softmax"), ("k1", "no softmax")):
        w, p = compile_workload(name)
        e = engine(p)
        with pytest.raises(RuntimeError, match=text):
            e.token_logprobs(configs.batch(w, 0)[0], None, 2)
        e.close()
    w, p = compile_workload("k2")  # a loss of two parts
    e = engine(p)
    rows, _ = e.softmax_shape(PROGRAM_TRAIN)
    with pytest.raises(RuntimeError, match="not one softmax"):
        e.distill_step(configs.batch(w, 0)[0], np.zeros((rows, 1), np.int32),
                       np.zeros((rows, 1), np.float32))
    e.close()


def _changed(plan, i, word, more):
    """The plan with its train program's instruction i replaced, and `more` put
    behind the next one."""
    from helpers import PlanView, append_train_instructions
    mat = 4 * int(np.prod([int(v) for v in plan.train[i - 1]["out"][:2]]))
    blob, h = append_train_instructions(plan, more, extra_arena=mat)
    at, end = h["train_instr_offset"], 64 * h["train_instr_count"]
    t = [bytes(blob[at + b:at + b + 64]) for b in range(0, end, 64)]
    t = t[:i] + [word, t[i + 1]] + more + t[i + 2:len(t) - len(more)]
    blob[at:at + end] = b"".join(t)
    return PlanView(append_train_instructions(PlanView(blob, h), [])[0], None)


@pytest.mark.parametrize("case,text", [
    ("as it is", None), ("another copy", None), ("seed of a half", "not its loss's own"),
    ("seed of another slot", "not its loss's own"), ("probabilities read", "probabilities or seed"),
    ("seed read", "probabilities or seed")])
def test_a_train_program_that_distillation_would_change_elsewhere_is_refused(torch_gpu, case, text):
    """The step leaves out the program's own loss, its seed and its gradient: a
    program in which they mean more than that is refused, before anything runs."""
    from helpers import instr
    w, p = compile_workload("c3s")
    f = xent(p.train)
    fwd, seed = p.train[f], p.train[f + 1]
    n = int(fwd["out"][0]) * int(fwd["out"][1])
    spare = planner.align_up(p.header["arena_size"])
    fill = lambda slot, v: instr(planner.OP["Fill"], (slot, planner.f32_bits(v)), (1,))  # noqa: E731
    copy = lambda src, m: [instr(planner.OP["Copy"], (src, spare), (m,))]  # noqa: E731
    own = fill(int(seed["inp"][0]), 1.0)
    word, more = {
        "as it is": (own, []),
        "another copy": (own, copy(int(p.params[0][1]), 4)),
        "seed of a half": (fill(int(seed["inp"][0]), 0.5), []),
        "seed of another slot": (fill(spare, 1.0), []),
        "probabilities read": (own, copy(int(fwd["inp"][3]), n)),
        "seed read": (own, copy(int(seed["inp"][0]), 1)),
    }[case]
    e, plain = engine(_changed(p, f + 1, word, more)), engine(p)
    x, _ = configs.batch(w, 0)
    ids, v = lists(plain, x, 4, 1.0)
    m = p.header["persistent_size"] // 4
    before = e.read(0, m)
    if text:
        with pytest.raises(RuntimeError, match=text):
            e.distill_step(x, ids, v)
        assert e.step == 0 and np.array_equal(e.read(0, m), before)
    else:
        assert e.distill_step(x, ids, v) == plain.distill_step(x, ids, v)
        assert np.array_equal(e.read(0, m).view(np.uint32), plain.read(0, m).view(np.uint32))
    e.close()
    plain.close()
