"""The block-scaled 8-bit format and its operators in 64 bits, from their
definitions (numpy only)."""
import math

import numpy as np

NAN = 0x7F


def _value(code: int) -> float:
    s, e, m = code >> 7, code >> 3 & 15, code & 7
    if code & 0x7F == NAN:
        return math.nan
    v = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    return -v if s else v


VALUES = np.array([_value(c) for c in range(256)])
POSITIVE = VALUES[:NAN]  # ascending, 0 to 448


def up(n: int) -> int:
    return -(-n // 128) * 128


def encode(y):
    """Codes of values up to 448 in magnitude, nearest, ties to the even code; NaN for NaN."""
    y = np.asarray(y, np.float64)
    a = np.where(np.isnan(y), 0.0, np.abs(y))
    assert a.max(initial=0.0) <= 448.0
    hi = np.searchsorted(POSITIVE, a).clip(max=NAN - 1)
    lo = np.maximum(hi - 1, 0)
    near = np.abs(POSITIVE[hi] - a) - np.abs(a - POSITIVE[lo])
    code = np.where((near < 0) | ((near == 0) & (hi % 2 == 0)), hi, lo)
    code = np.where(POSITIVE[hi] == a, hi, code)
    code = np.where(np.signbit(y), code | 0x80, code)
    return np.where(np.isnan(y), NAN, code).astype(np.uint8)


def scale_byte(amax):
    m, ex = np.frexp(amax)  # amax = m 2^ex, m in [1/2, 1)
    e = ex - 9 + (m > 448 / 512)
    return np.where(amax > 0, np.maximum(e, -127) + 127, 0).astype(np.int64)


def quantize(x, square=False):
    """(codes [rows, up(cols)], scales [up(cols) / 128, up(rows)]) of x."""
    rows, cols = x.shape
    full = np.zeros((up(rows), up(cols)))
    full[:rows, :cols] = x
    b = full.reshape(up(rows) // 128, 128, up(cols) // 128, 128)
    mag = np.where(np.isfinite(b), np.abs(b), 0.0)
    amax = mag.max((1, 3), keepdims=True) if square else mag.max(3, keepdims=True)
    byte = np.broadcast_to(scale_byte(amax), b.shape[:3] + (1,))
    with np.errstate(invalid="ignore"):
        y = np.where(np.isfinite(b), b * 2.0 ** (127.0 - byte), np.nan)
    codes = encode(y).reshape(full.shape)[:rows]
    scales = byte[..., 0].reshape(up(rows), -1).copy()
    scales[rows:] = 0
    return codes, np.ascontiguousarray(scales.T).astype(np.uint8)


def values(codes, scales, cols):
    """What codes and scales stand for, [rows, cols]."""
    rows = codes.shape[0]
    f = np.exp2(scales[:, :rows].T.astype(np.float64) - 127)
    return (VALUES[codes].reshape(rows, -1, 128) * f[:, :, None]).reshape(rows, -1)[:, :cols]


def step(codes, scales, cols):
    """Half the gap to the next code, at the magnitude of each value."""
    rows = codes.shape[0]
    f = np.exp2(scales[:, :rows].T.astype(np.float64) - 127)
    v = np.abs(VALUES[codes]).reshape(rows, -1, 128)
    half = np.maximum(v * 2.0 ** -4, 2.0 ** -10)
    return (half * f[:, :, None]).reshape(rows, -1)[:, :cols]


def act(kind, x):
    """(a(x), a'(x), a''(x) bound aside) of 1 ReLU, 2 GELU (tanh form), 3 SiLU."""
    if kind == 1:
        return np.maximum(x, 0.0), (x > 0).astype(np.float64)
    with np.errstate(over="ignore"):
        if kind == 3:
            s = 1.0 / (1.0 + np.exp(-x))
            r = 1.0 / (1.0 + np.exp(x))
            return x * s, s + x * s * r
        c, k = math.sqrt(2.0 / math.pi), 0.044715
        y = np.clip(x, -30.0, 30.0)
        t = 2.0 * c * (y + k * y ** 3)
        s, r = 1.0 / (1.0 + np.exp(-t)), 1.0 / (1.0 + np.exp(t))
        return x * s, s + y * s * r * 2.0 * c * (1.0 + 3.0 * k * y * y)


def rms_bwd(dy, x, gamma, rstd):
    g, r = dy * gamma, rstd[:, None]
    return r * g - x * r ** 3 * (g * x).mean(-1, keepdims=True)
