"""Refused calls on two host threads: each reads its own error text."""
import threading

from test_scores_refusals import L, bwd, dboth, dfwd, fwd  # noqa: F401


def test_a_threads_refusals_are_its_own(L):  # noqa: F811
    from seeml_amd import _lib
    jobs = [(fwd, dict(T=0.0), "temperature"), (dboth, dict(k=41), "more listed classes than classes"),
            (bwd, dict(dstride=39), "gradient row stride"), (dfwd, dict(tail=2), "tail is 0 or 1")]
    all_failed, failed = threading.Barrier(len(jobs), timeout=60), []

    def work(call, kw, text):
        try:
            for _ in range(50):
                rc, msg = call(L, **kw)
                assert rc == 1 and text in msg, msg
                all_failed.wait()  # the others have failed since
                assert _lib.kernel_error() == msg
                all_failed.wait()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
            all_failed.abort()

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
