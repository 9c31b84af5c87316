"""How an 8-bit product of given sizes runs (csrc/f8_choice.h): that the GPU tests
meet every path, and that no size leaves work out. Host only."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import test_gpu_f8 as shapes
import test_gpu_f8_paths as paths

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "f8_choice.h"
extern "C" void choose(uint64_t M, uint64_t N, uint64_t k_blocks, int gated, int keep, uint32_t* out) {
  const seeml_hip::f8::Choice c = seeml_hip::f8::ChooseF8(M, N, k_blocks, gated, keep);
  out[0] = c.skinny; out[1] = c.big; out[2] = c.columns; out[3] = c.splits; out[4] = c.blocks_per_split;
}
"""


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("f8_choice")
    (d / "choose.cc").write_text(SOURCE)
    so = str(d / "choose.so")
    subprocess.run(["g++", "-std=c++20", "-shared", "-fPIC", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "see-ml_amd", "csrc"), str(d / "choose.cc"), "-o", so],
                   check=True, capture_output=True, text=True)
    fn = C.CDLL(so).choose
    fn.argtypes = [C.c_uint64] * 3 + [C.c_int] * 2 + [C.POINTER(C.c_uint32)]

    def ask(M, N, K, gated=False, keep=False, pairs=1):
        out = (C.c_uint32 * 5)()
        fn(M, N, -(-K // 128) * pairs, gated, keep, out)
        skinny, big, columns, splits, per = out
        if skinny:
            return "few", skinny, 1
        if big:
            return ("large and half" if columns else "large"), columns, 1
        return ("split" if splits > 1 else "small"), per, splits

    return ask


def test_the_gpu_tests_meet_every_path(choose):
    for want, sizes in (("few", paths.FEW), ("small", paths.SMALL), ("split", paths.SPLIT), ("large", paths.LARGE),
                        ("large and half", paths.LARGE_AND_HALF)):
        for s in sizes:
            assert choose(*s)[0] == want, s
            # Each of at most four stages is loaded again.
            assert want == "few" or (choose(*s)[1] if want == "split" else -(-s[2] // 128)) >= 6, s
    T, D, F = paths.GATED_LARGE_AND_HALF
    for keep in (False, True):
        assert choose(T, F, D, gated=True, keep=keep)[0] == "large and half"
    assert -(-D // 128) >= 9
    T, D, F = paths.GATED_BWD_LARGE
    assert choose(T, D, F, pairs=2)[0] == "large"
    met = {choose(*s)[:2] for s in shapes.GEMMS if choose(*s)[0] == "few"}
    assert met == {("few", 1), ("few", 2), ("few", 4)}
    met = {choose(*s)[0] for s in shapes.GEMMS}
    assert met == {"few", "small", "split", "large and half"}
    met = {choose(T, F, D, gated=True, keep=keep)[0] for T, D, F in shapes.GATES for keep in (False, True)}
    assert met == {"few", "small", "large", "large and half"}


@pytest.mark.parametrize("M", [1, 16, 17, 64, 65, 129, 777, 2048, 4200, 1 << 20])
@pytest.mark.parametrize("N", [1, 127, 1003, 5504, 16384])
@pytest.mark.parametrize("K", [1, 128, 2048, 5504, 1 << 14])
def test_slices_cover_a_reduction_once(choose, M, N, K):
    way, per, splits = choose(M, N, K)
    blocks = -(-K // 128)
    if way == "split":
        assert (splits - 1) * per < blocks <= splits * per
        assert splits * -(-M // 128) * -(-N // 128) <= 256
    if way == "large and half":
        # Whole rounds of large tiles, one round of half tiles.
        high = -(-M // 256)
        assert 0 < per < -(-N // 256) and -(-M // 128) * (-(-N // 256) - per) <= 256
