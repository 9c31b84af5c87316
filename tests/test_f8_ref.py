"""The 64-bit reference of the block-scaled 8-bit operators checks itself: its
number format against torch's, its slopes and gradients against differences."""
import numpy as np
import pytest

import f8_ref as ref


def test_code_values_are_e4m3s():
    import torch
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(t, ref.VALUES)


def test_encoding_rounds_as_the_conversion_does():
    import torch
    rng = np.random.default_rng(1)
    y = np.concatenate([rng.standard_normal(20000) * 2.0 ** rng.integers(-12, 8, 20000), ref.POSITIVE,
                        (ref.POSITIVE[1:] + ref.POSITIVE[:-1]) / 2, [0.0, -0.0]])
    y = np.clip(y, -448, 448).astype(np.float32)
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(ref.encode(y), want)


@pytest.mark.parametrize("amax, byte", [(448.0, 127), (448.0001, 128), (1.75, 119), (1.7500001, 120),
                                        (0.0, 0), (2.0 ** -119, 0), (2.0 ** -118, 1), (2.0 ** -149, 0),
                                        (3.4028234e38, 247)])
def test_scale_is_the_least_that_fits(amax, byte):
    assert ref.scale_byte(np.array(amax)) == byte
    e = byte - 127
    assert amax / 2.0 ** e <= 448 and (byte == 0 or amax / 2.0 ** (e - 1) > 448)


@pytest.mark.parametrize("kind", [1, 2, 3])
def test_slopes_are_the_differences(kind):
    x = np.concatenate([np.linspace(-12, 12, 4001) + 1e-3, [-200.0, 200.0, -1e30, 1e30]])
    a, d = ref.act(kind, x)
    h = 1e-5 * np.maximum(1.0, np.abs(x))
    diff = (ref.act(kind, x + h)[0] - ref.act(kind, x - h)[0]) / (2 * h)
    # Third derivatives are below 2, rounding of a below 2^-52 |a| / h.
    np.testing.assert_allclose(d, diff, rtol=1e-6, atol=1e-9)


def test_norm_gradient_is_the_difference():
    rng = np.random.default_rng(2)
    x, dy, gamma = rng.standard_normal((3, 7)), rng.standard_normal((3, 7)), rng.standard_normal(7)
    f = lambda v: (dy * gamma * v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-5)).sum()  # noqa: E731
    got = ref.rms_bwd(dy, x, gamma, 1.0 / np.sqrt((x * x).mean(-1) + 1e-5))
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-5
        assert abs((f(x + e) - f(x - e)) / 2e-5 - got[i]) < 1e-7
