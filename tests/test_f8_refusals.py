"""Arguments that the block-scaled 8-bit entries refuse. The checks come before
anything touches a GPU, so these run without one; pointers are addresses that
nothing reads."""
import ctypes
import threading

import pytest

from seeml_amd import _lib

BASE = 0x7E0000000000
T, D, F, R = 70, 200, 300, 8


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def at(i):
    """A 16-byte aligned address of its own, 16 MiB from the next."""
    return BASE + (i << 24)


def quantize(L, **kw):
    a = dict(x=at(0), dtype=0, stride=D, rows=T, cols=D, codes=at(1), scales=at(2))
    a.update(kw)
    return L.seeml_hip_f8_quantize(*a.values(), None), _lib.kernel_error()


def weight(L, **kw):
    a = dict(w=at(0), dtype=0, stride=D, rows=T, cols=D, codes=at(1), scales=at(2), codes_t=at(3), scales_t=at(4))
    a.update(kw)
    return L.seeml_hip_f8_quantize_weight(*a.values(), None), _lib.kernel_error()


def dequantize(L, **kw):
    a = dict(codes=at(1), scales=at(2), x=at(0), dtype=0, stride=D, rows=T, cols=D)
    a.update(kw)
    return L.seeml_hip_f8_dequantize(*a.values(), None), _lib.kernel_error()


def gemm(L, **kw):
    a = dict(ac=at(0), asc=at(1), bc=at(2), bsc=at(3), C=at(4), dtype=0, stride=F, M=T, N=F, K=D, scratch=at(5),
             nbytes=1 << 30)
    a.update(kw)
    return L.seeml_hip_gemm_f8_nt(*a.values(), None), _lib.kernel_error()


def gated(L, **kw):
    a = dict(xc=at(0), xs=at(1), gc=at(2), gs=at(3), uc=at(4), us=at(5), act=3, h=at(6), dtype=0, h_stride=F,
             hc=at(7), hs=at(8), g8=at(9), g8s=at(10), u8=at(11), u8s=at(12), T=T, D=D, F=F, scratch=at(13),
             nbytes=1 << 24)
    a.update(kw)
    return L.seeml_hip_gated_f8_fwd(*a.values(), None), _lib.kernel_error()


def gated_bwd(L, **kw):
    a = dict(dh=at(0), dtype=0, dh_stride=F, g8=at(1), g8s=at(2), u8=at(3), u8s=at(4), act=3, gc=at(5), gs=at(6),
             uc=at(7), us=at(8), dg=at(9), dgs=at(10), du=at(11), dus=at(12), h=at(13), h_stride=F, dx=at(14),
             dx_stride=D, T=T, D=D, F=F, scratch=at(15), nbytes=1 << 24)
    a.update(kw)
    return L.seeml_hip_gated_f8_bwd(*a.values(), None), _lib.kernel_error()


def act_bwd(L, **kw):
    a = dict(dy=at(0), dtype=0, stride=D, codes=at(1), scales=at(2), act=2, dx=at(3), dx_stride=D, rows=T, cols=D)
    a.update(kw)
    return L.seeml_hip_act_bwd_f8(*a.values(), None), _lib.kernel_error()


def norm_bwd(L, **kw):
    a = dict(dy=at(0), dtype=0, stride=D, codes=at(1), scales=at(2), gamma=at(4), rstd=at(5), dx=at(3), dx_stride=D,
             rows=T, cols=D)
    a.update(kw)
    return L.seeml_hip_rms_norm_bwd_f8(*a.values(), None), _lib.kernel_error()


def lora(L, **kw):
    a = dict(xc=at(0), xs=at(1), dt=at(2), dtype=0, stride=R, out=at(3), T=T, D=D, r=R, scratch=at(4), nbytes=1 << 24)
    a.update(kw)
    return L.seeml_hip_gemm_tn_f8(*a.values(), None), _lib.kernel_error()


ALL = [quantize, weight, dequantize, gemm, gated, gated_bwd, act_bwd, norm_bwd, lora]


@pytest.mark.parametrize("call", ALL)
@pytest.mark.parametrize("dtype", [-1, 3])
def test_unknown_types(L, call, dtype):
    rc, msg = call(L, dtype=dtype)
    assert rc == 1 and f"unknown type {dtype}" in msg


@pytest.mark.parametrize("call", [gated, gated_bwd, act_bwd])
@pytest.mark.parametrize("act", [0, 4, -1])
def test_unknown_activations(L, call, act):
    rc, msg = call(L, act=act)
    assert rc == 1 and f"unknown activation {act}" in msg


# (entry, its extents, its pointers that must not be null, its strides)
SHAPES = {
    quantize: ("rows cols", "x codes scales", "stride"),
    weight: ("rows cols", "w", "stride"),
    dequantize: ("rows cols", "codes scales x", "stride"),
    gemm: ("M N K", "ac asc bc bsc C", "stride"),
    gated: ("T D F", "xc xs gc gs uc us", "h_stride"),
    gated_bwd: ("T D F", "dh g8 g8s u8 u8s dg dgs du dus gc gs uc us", "dh_stride h_stride dx_stride"),
    act_bwd: ("rows cols", "dy codes scales dx", "stride dx_stride"),
    norm_bwd: ("rows cols", "dy codes scales gamma rstd dx", "stride dx_stride"),
    lora: ("T D", "xc xs dt out", "stride"),
}


@pytest.mark.parametrize("call", ALL)
def test_extents(L, call):
    for name in SHAPES[call][0].split():
        for value, text in ((0, "empty input"), ((1 << 24) + 1, "more than 2^24"), (1 << 63, "more than 2^24")):
            rc, msg = call(L, **{name: value})
            assert rc == 1 and text in msg, (name, value, msg)
    names = SHAPES[call][0].split()
    rc, msg = call(L, **{names[0]: 1 << 24, names[1]: 1 << 10})
    assert rc == 1 and "2^33 values or more" in msg


@pytest.mark.parametrize("call", ALL)
def test_null_pointers(L, call):
    for name in SHAPES[call][1].split():
        rc, msg = call(L, **{name: None})
        assert rc == 1 and ("null" in msg or "without" in msg), (name, msg)


@pytest.mark.parametrize("call", ALL)
def test_strides(L, call):
    for name in SHAPES[call][2].split():
        rc, msg = call(L, **{name: 7})
        assert rc == 1 and "row stride below the row length" in msg, (name, msg)
        rc, msg = call(L, **{name: 1 << 61})
        assert rc == 1 and "row stride too large" in msg, (name, msg)


@pytest.mark.parametrize("call, kw, text", [
    (weight, dict(scales=None), "codes and scales go together"),
    (weight, dict(codes_t=None), "codes and scales go together"),
    (weight, dict(codes=None, scales=None, codes_t=None, scales_t=None), "no output"),
    (gated, dict(hc=None), "codes and scales go together"),
    (gated, dict(g8s=None), "codes and scales go together"),
    (gated, dict(u8=None), "codes and scales go together"),
    (gated, dict(h=None, hc=None, hs=None, g8=None, g8s=None, u8=None, u8s=None), "no output"),
    (lora, dict(r=0), "empty input"),
    (lora, dict(r=129, stride=129), "rank above 128"),
    (lora, dict(T=1000, scratch=None), "scratch of"),
    (gemm, dict(K=4096, scratch=None), "scratch of"),
    (gemm, dict(K=4096, nbytes=15), "scratch of 15 bytes"),
    (gated_bwd, dict(F=4096, dh_stride=4096, h_stride=4096, scratch=None), "scratch of"),
])
def test_what_goes_together(L, call, kw, text):
    rc, msg = call(L, **kw)
    assert rc == 1 and text in msg, msg


@pytest.mark.parametrize("call, kw, text", [
    (quantize, dict(x=at(0) + 2), "x is not aligned"),
    (quantize, dict(codes=at(1) + 8), "codes is not aligned"),
    (quantize, dict(scales=at(2) + 8), "scales is not aligned"),
    (gemm, dict(bc=at(2) + 4), "b_codes is not aligned"),
    (norm_bwd, dict(gamma=at(4) + 1), "gamma is not aligned"),
    (lora, dict(T=1000, scratch=at(4) + 8), "scratch is not aligned"),
    (quantize, dict(x=2 ** 64 - 64), "passes the end of memory"),
    (quantize, dict(codes=at(0) + 16), "codes overlaps x"),
    (quantize, dict(scales=at(1) + T * 256 - 16), "overlaps"),
    (weight, dict(codes_t=at(1)), "overlaps"),
    (dequantize, dict(x=at(1)), "x overlaps codes"),
    (gemm, dict(C=at(0)), "C overlaps a_codes"),
    (gemm, dict(K=4096, scratch=at(4)), "overlaps"),
    (gated, dict(h=at(2)), "h overlaps wg_codes_t"),
    (gated, dict(u8=at(9)), "overlaps"),
    (gated_bwd, dict(dg=at(1)), "dg_codes overlaps g_codes"),
    (gated_bwd, dict(h=at(0)), "overlaps"),
    (gated_bwd, dict(dx=at(5)), "dx overlaps wg_codes"),
    (act_bwd, dict(dx=at(0), dx_stride=D + 4), "dx overlaps dy with another row stride"),
    (act_bwd, dict(dx=at(0) + 16), "dx overlaps dy"),
    (act_bwd, dict(dx=at(2)), "dx overlaps scales"),
    (norm_bwd, dict(dx=at(5)), "dx overlaps rstd"),
    (norm_bwd, dict(dx=at(0) + 4 * D), "dx overlaps dy"),
    (lora, dict(out=at(2)), "out overlaps dt"),
])
def test_places(L, call, kw, text):
    rc, msg = call(L, **kw)
    assert rc == 1 and text in msg, msg


def test_sizes(L):
    assert L.seeml_hip_f8_codes_bytes(70, 200) == 70 * 256
    assert L.seeml_hip_f8_scales_bytes(70, 200) == 2 * 128
    assert L.seeml_hip_f8_codes_bytes(0, 5) == 0 and L.seeml_hip_f8_scales_bytes(5, (1 << 24) + 1) == 0
    assert L.seeml_hip_f8_codes_bytes(1 << 24, 1 << 10) == 0
    assert L.seeml_hip_gemm_f8_scratch(0, 1, 1) == 0 and L.seeml_hip_gated_f8_scratch(1, 0, 1) == 0
    assert L.seeml_hip_gemm_tn_f8_scratch(100000, 64, 129) == 0


def test_a_threads_refusals_are_its_own(L):
    jobs = [(quantize, dict(dtype=9), "unknown type 9"), (gemm, dict(M=0), "empty input"),
            (lora, dict(r=200, stride=200), "rank above"), (act_bwd, dict(act=7), "unknown activation 7")]
    all_failed, failed = threading.Barrier(len(jobs), timeout=60), []

    def work(call, kw, text):
        try:
            for _ in range(50):
                rc, msg = call(L, **kw)
                assert rc == 1 and text in msg, msg
                all_failed.wait()
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


def test_host_memory_is_refused(L):
    """Pointers that name no device memory end in an error, not in a launch."""
    buf = ctypes.create_string_buffer(1 << 16)
    x = (ctypes.addressof(buf) + 15) // 16 * 16
    rc = L.seeml_hip_f8_quantize(x, 0, 4, 2, 4, x + 1024, x + 8192, None)
    assert rc == 1
