"""The norm of an attention row's error over an 8-bit pool, held to what the kernels'
roundings make of it (oracle/kv_q8.py: typical_error)."""
import numpy as np


def check_error(got, want, typical, what):
    """got, want [rows][heads][hd], typical [rows][heads].

    typical is the root mean square that the roundings of a row leave, so over rows the mean
    square of error / typical is 1 at most: 4 (a ratio of 2) where there are 8 or more rows
    and heads to take it over.  One row's error is a sum of many independent roundings; past
    5 times its root mean square a normal variable is once in 1.7 million."""
    ratio = np.linalg.norm(np.asarray(got, np.float64) - want, axis=-1) / typical
    assert np.isfinite(ratio).all(), what
    assert ratio.max() <= 5, f"{what}: a row is off by {ratio.max():.1f} times the typical error"
    rms = np.sqrt((ratio ** 2).mean())
    assert ratio.size < 8 or rms <= 2, f"{what}: rows are off by {rms:.1f} times the typical error"
