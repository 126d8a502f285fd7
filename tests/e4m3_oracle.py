"""Values in eight bits (e4m3) and their groups' powers of two by the definition, on the host."""
import numpy as np

LOWEST = -100


def _value(code):
    sign, e, m = -1.0 if code & 0x80 else 1.0, code >> 3 & 15, code & 7
    if e == 15 and m == 7:
        return np.nan
    return sign * (m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10))


VALUES = np.array([_value(c) for c in range(256)])


def exponent(top):
    """The least e >= LOWEST with top <= 448 2^e, for top >= 0 in float64."""
    top = np.asarray(top, np.float64)
    part, e = np.frexp(top)
    return np.where(top > 0, np.maximum(e - 9 + (part > 0.875), LOWEST), LOWEST).astype(np.int64)


def encode(x):
    """The codes of x (|x| <= 448 or not finite), rounded to nearest, ties to even: by the distance to every value."""
    x = np.asarray(x, np.float64)
    good = VALUES[:127]  # 0 to 448, rising
    size = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(good, size, "left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = size - good[lo], good[hi] - size
    code = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isfinite(x), code, 0x7F)
    return (code + np.where(np.signbit(x) & np.isfinite(x), 128, 0)).astype(np.uint8)


def half_step(x, e):
    """Half the distance between values around x under the exponent e."""
    size = np.maximum(np.abs(np.asarray(x, np.float64)) * 2.0 ** -np.asarray(e, np.float64), 2.0**-6)
    return 2.0 ** (np.floor(np.log2(size)) - 4) * 2.0 ** np.asarray(e, np.float64)
