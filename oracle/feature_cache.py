"""The feature cache in 64 bits: codes and scales of a group of values, and the values that codes stand for."""
import numpy as np

LARGEST = {"int8": 127.0, "e4m3": 448.0}


def e4m3_numbers():
    """Value of each of the 256 bit patterns (no infinities, two NaNs)."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[b] = np.nan if (b & 127) == 127 else -v if b & 128 else v
    return out


def group_scale(x, code):
    """x: (..., dim) float64 -> float32 scales."""
    x = np.where(x == -np.inf, 0.0, x)
    largest = np.abs(x).max(-1)
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.maximum((largest / LARGEST[code]).astype(np.float32), np.float32(2.0 ** -126))
        s = np.where(s * np.float32(LARGEST[code]) == np.inf, np.nextafter(s, np.float32(0)), s)
    return np.where(np.isfinite(largest), s, np.float32(np.nan)).astype(np.float32)


def encode(x, code):
    """x: (..., dim) float64 -> (bytes as uint8, float32 scales)."""
    x = np.asarray(x, np.float64)
    s = group_scale(x, code)
    with np.errstate(invalid="ignore"):
        y = np.where(x == -np.inf, 0.0, x) / s[..., None].astype(np.float64)
    y = np.where(np.isfinite(y), y, 0.0)
    if code == "int8":
        q = np.rint(y).astype(np.int64).astype(np.uint8)
        empty = np.uint8(0x80)
    else:
        numbers = e4m3_numbers()[:127]
        middle = (numbers[1:] + numbers[:-1]) / 2
        low, high = np.searchsorted(middle, np.abs(y), "left"), np.searchsorted(middle, np.abs(y), "right")
        q = np.where(low % 2 == 0, low, high).astype(np.uint8)
        q = np.where(np.signbit(y), q | 0x80, q).astype(np.uint8)
        empty = np.uint8(0xFF)
    q = np.where(x == -np.inf, empty, q)
    return np.where(np.isnan(s)[..., None], np.uint8(0), q).astype(np.uint8), s


def decode(q, s, code):
    """Bytes (..., dim) and scales (...) -> float64 values, before they are rounded to the rows' type."""
    q = np.asarray(q, np.uint8)
    numbers = np.where(q == 0x80, 0, q.view(np.int8)).astype(np.float64) if code == "int8" else e4m3_numbers()[q]
    v = numbers * np.asarray(s, np.float64)[..., None]
    return np.where(q == (0x80 if code == "int8" else 0xFF), -np.inf, v)
