"""Arguments that the token-score and top-k distillation entries refuse. The
checks come before anything touches a GPU, so these run without one; pointers
are addresses that nothing reads."""
import pytest

from seeml_amd import _lib

BASE = 0x7F0000000000
N, C, K = 6, 40, 5


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def at(i):
    """A 16-byte aligned address of its own, 1 MiB from the next."""
    return BASE + (i << 20)


def fwd(L, **kw):
    a = dict(logits=at(0), dtype=0, stride=C, targets=at(1), T=1.0, k=K, logp=at(2), entropy=at(3),
             stats=at(4), top_ids=at(5), top_logp=at(6), N=N, C=C, scratch=at(7), nbytes=1 << 20)
    a.update(kw)
    return L.seeml_hip_token_logprobs_fwd(*a.values(), None), _lib.kernel_error()


def bwd(L, **kw):
    a = dict(logits=at(0), dtype=0, stride=C, targets=at(1), T=1.0, stats=at(4), dlogp=at(2),
             dentropy=at(3), dlogits=at(8), dstride=C, N=N, C=C)
    a.update(kw)
    return L.seeml_hip_token_logprobs_bwd(*a.values(), None), _lib.kernel_error()


def dfwd(L, **kw):
    a = dict(logits=at(0), dtype=0, stride=C, ids=at(1), lp=at(2), k=K, weight=at(3), T=1.0, tail=1,
             loss=at(4), row_loss=at(5), stats=at(6), N=N, C=C, scratch=at(7), nbytes=1 << 20)
    a.update(kw)
    return L.seeml_hip_topk_distill_fwd(*a.values(), None), _lib.kernel_error()


def dbwd(L, **kw):
    a = dict(logits=at(0), dtype=0, stride=C, ids=at(1), lp=at(2), k=K, weight=at(3), seed=at(4),
             T=1.0, tail=1, stats=at(6), dlogits=at(8), dstride=C, N=N, C=C)
    a.update(kw)
    return L.seeml_hip_topk_distill_bwd(*a.values(), None), _lib.kernel_error()


def dboth(L, **kw):
    a = dict(logits=at(0), dtype=0, stride=C, ids=at(1), lp=at(2), k=K, weight=at(3), seed=at(9),
             T=1.0, tail=1, loss=at(4), row_loss=at(5), dlogits=at(8), dstride=C, N=N, C=C,
             scratch=at(7), nbytes=1 << 20)
    a.update(kw)
    return L.seeml_hip_topk_distill_fwd_bwd(*a.values(), None), _lib.kernel_error()


ALL = [fwd, bwd, dfwd, dbwd, dboth]
SHARED = [
    (dict(dtype=3), "unknown logits type 3"),
    (dict(dtype=-1), "unknown logits type"),
    (dict(N=0), "empty input"),
    (dict(C=0, stride=0), "empty input"),
    (dict(stride=C - 1), "row stride below"),
    (dict(stride=1 << 62), "row stride too large"),
    (dict(N=1 << 22), "too many rows"),
    (dict(N=1 << 21, C=1 << 15, stride=1 << 15), "more than 2^37 bytes"),
    (dict(C=(1 << 30) + 1, stride=1 << 31), "too many classes"),
    (dict(T=0.0), "temperature"),
    (dict(T=-1.0), "temperature"),
    (dict(T=float("nan")), "temperature"),
    (dict(T=float("inf")), "temperature"),
    (dict(T=1e-31), "temperature"),
    (dict(logits=None), "null"),
    (dict(logits=at(0) + 2), "logits is not aligned"),
]


@pytest.mark.parametrize("call", ALL)
@pytest.mark.parametrize("kw,text", SHARED)
def test_every_entry_refuses(L, call, kw, text):
    rc, msg = call(L, **kw)
    assert rc == 1 and text in msg and msg.startswith("UpdateEngine: T"), msg


@pytest.mark.parametrize("call,kw,text", [
    (fwd, dict(k=129, C=1000, stride=1000), "more than 128"),
    (fwd, dict(k=C + 1), "more listed classes than classes"),
    (fwd, dict(targets=None), "go together"),
    (fwd, dict(logp=None), "go together"),
    (fwd, dict(top_ids=None), "null top_ids"),
    (fwd, dict(top_logp=None), "null top_ids or top_logp"),
    (fwd, dict(targets=None, logp=None, entropy=None, stats=None, k=0), "no output"),
    (fwd, dict(entropy=at(2)), "overlaps"),
    (fwd, dict(entropy=at(0)), "entropy overlaps logits"),
    (fwd, dict(logp=at(1)), "logp overlaps targets"),
    (fwd, dict(top_logp=at(5) + 4 * K * (N - 1)), "overlaps"),
    (fwd, dict(entropy=at(3) + 2), "entropy is not aligned"),
    (bwd, dict(stats=None), "null"),
    (bwd, dict(dlogits=None), "null"),
    (bwd, dict(dlogp=None, dentropy=None), "no gradient"),
    (bwd, dict(targets=None), "dlogp without targets"),
    (bwd, dict(dstride=C - 1), "gradient row stride"),
    (bwd, dict(dlogits=at(0), dstride=C + 4), "another row stride"),
    (bwd, dict(dlogits=at(0) + 4), "dlogits overlaps logits"),
    (bwd, dict(stride=3 * C, dstride=3 * C, dlogits=at(0) + 4 * (2 * C + 1)), "dlogits overlaps"),
    (bwd, dict(dlogits=at(4)), "dlogits overlaps row_stats"),
    (bwd, dict(dlogits=at(1)), "dlogits overlaps targets"),
    (dfwd, dict(k=0), "no listed classes"),
    (dfwd, dict(k=129, C=1000, stride=1000), "more than 128"),
    (dfwd, dict(k=C + 1), "more listed classes than classes"),
    (dfwd, dict(ids=None), "null"),
    (dfwd, dict(lp=None), "null"),
    (dfwd, dict(row_loss=None), "null row_loss"),
    (dfwd, dict(tail=2), "tail is 0 or 1"),
    (dfwd, dict(loss=at(5)), "overlaps"),
    (dfwd, dict(scratch=None), "needed"),
    (dfwd, dict(nbytes=7), "scratch of 7 bytes"),
    (dfwd, dict(scratch=at(7) + 8), "scratch is not aligned"),
    (dfwd, dict(stats=at(0)), "overlaps logits"),
    (dbwd, dict(stats=None), "null row_stats"),
    (dbwd, dict(dlogits=None), "null dlogits"),
    (dbwd, dict(dlogits=at(6)), "overlaps row_stats"),
    (dbwd, dict(dlogits=at(2)), "overlaps t_logp"),
    (dboth, dict(dlogits=at(7)), "overlaps"),
    (dboth, dict(dlogits=at(9)), "dlogits overlaps seed"),
    (dboth, dict(loss=at(9)), "overlaps"),
    (dboth, dict(scratch=None), "needed"),
])
def test_refused(L, call, kw, text):
    rc, msg = call(L, **kw)
    assert rc == 1 and text in msg, msg


@pytest.mark.parametrize("call", ALL)
def test_what_passes_the_checks_is_stopped_where_there_is_no_device_memory(L, call):
    """The addresses above are nobody's: refused without a launch."""
    rc, msg = call(L)
    assert rc == 1 and ("not device memory" in msg or "hipGetDevice" in msg), msg


@pytest.mark.parametrize("kw", [
    dict(dlogits=at(0)),                                              # in place
    dict(stride=3 * C, dstride=3 * C, dlogits=at(0) + 4 * C),         # the next columns
    dict(stride=3 * C, dstride=3 * C, dlogits=at(0) + 4 * 2 * C),     # the last ones
    dict(logits=at(0) + 8 * C, stride=3 * C, dstride=3 * C, dlogits=at(0)),
    dict(dlogp=None, targets=None), dict(dentropy=None),
])
def test_gradient_places_that_are_allowed(L, kw):
    rc, msg = bwd(L, **kw)
    assert rc == 1 and ("not device memory" in msg or "hipGetDevice" in msg), msg


def test_scratch_queries(L):
    for f in (L.seeml_hip_token_logprobs_scratch, L.seeml_hip_topk_distill_scratch):
        assert f(0, C, 0, K) == 0 and f(N, C, 9, K) == 0 and f(N, C, 0, C + 1) == 0
        assert f(N, C, 0, K) % 4 == 0
