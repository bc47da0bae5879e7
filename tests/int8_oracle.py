"""Plain numpy forms of the 8-bit path, in 64 bits where a decision is made."""
import numpy as np


def quantize(x):
    """(q int8, scale float32) of fp32 rows: the exact quotient x / scale rounded to even."""
    x = np.asarray(x, dtype=np.float32)
    if x.shape[1] == 0:
        return np.zeros(x.shape, np.int8), np.zeros(x.shape[0], np.float32)
    amax = np.abs(x).max(axis=1)
    s = (amax.astype(np.float64) / 127.0).astype(np.float32)
    s[~np.isfinite(amax)] = np.nan
    none = ~(s > 0)
    # fp32 / fp32 in 64 bits: a quotient that is not a border itself never rounds onto one
    # (|x - b * s| >= 2^-32 |x| where it is not 0)
    d = np.where(none, 1.0, s.astype(np.float64))[:, None]
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.clip(np.rint(x.astype(np.float64) / d), -127, 127)
    q[none] = 0
    return q.astype(np.int8), s


def linear(q, sx, w, sw, b, relu):
    """The transform with its fp32 steps: the kernel's bits."""
    with np.errstate(invalid="ignore", over="ignore"):
        acc = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)  # whole numbers below 2^53
        y = (acc * sx.astype(np.float32)[:, None]) * sw.astype(np.float32)[None, :]
        if b is not None:
            y = y + b.astype(np.float32)[None, :]
        if relu:
            y = np.where(y < 0, np.float32(0), y)
    return y


def same_bits(a, b):
    """Equal fp32 arrays, any NaN equal to any other."""
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    both = np.isnan(a) & np.isnan(b)
    return a.shape == b.shape and bool(np.all(both | (a.view(np.uint32) == b.view(np.uint32))))
