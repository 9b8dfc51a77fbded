"""Rows held in 8 bits and products of them in 64 bits, from their definition."""
from __future__ import annotations

import math

import numpy as np

EPS32 = 2.0 ** -24  # half a step of fp32


def hold(y):
    """codes, scales of fp32 rows."""
    y = np.asarray(y, np.float32)
    codes, scales = np.zeros(y.shape, np.int8), np.zeros(len(y), np.float32)
    for i, row in enumerate(y):
        if not np.isfinite(row).all():
            scales[i] = np.nan
            continue
        top = np.abs(row).max()
        if top < 2.0 ** -100:
            continue
        scales[i] = np.float32(top) / np.float32(127)
        codes[i] = np.rint(row.astype(np.float64) * np.float64(np.float32(127) / np.float32(top))).astype(np.int8)
    return codes, scales


def normed(x, weight, residual=None, eps=1e-5):
    """(sum, y) of the norm, y as the fp32 numbers that are held."""
    h = np.asarray(x, np.float32)
    if residual is not None:
        h = h + np.asarray(residual, np.float32)
    h64 = h.astype(np.float64)
    with np.errstate(all="ignore"):
        r = 1 / np.sqrt((h64 * h64).mean(-1, keepdims=True) + eps)
        return h, (h64 * r * np.asarray(weight, np.float64)).astype(np.float32)


def matrix(rng, d, n):
    """BlockQ8 rows, uint8 [d][n / 32][36], with their codes and scales."""
    q = rng.integers(-127, 128, (d, n // 32, 32)).astype(np.int8)
    s = ((0.5 + rng.random((d, n // 32))) / (127 * math.sqrt(n))).astype(np.float32)
    w = np.empty((d, n // 32, 36), np.uint8)
    w[..., :4] = s[..., None].view(np.uint8)
    w[..., 4:] = q.view(np.uint8)
    return w, q, s


def act(p, name):
    with np.errstate(all="ignore"):
        if name == "relu":
            return np.where(p < 0, 0.0, p)
        if name == "silu":
            return p / (1 + np.exp(-p))
        if name == "gelu":
            import torch

            return (0.5 * torch.from_numpy(p) * torch.special.erfc(torch.from_numpy(-p * math.sqrt(0.5)))).numpy()
        if name == "gelu_tanh":
            return p / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)))
    return p


def product(mats, codes, scales, bias=None, residual=None, activation="none"):
    """(out, bound): the 64-bit result and what fp32 may leave of it.

    A block's sum is exact; one fma per block into the running sum rounds it by half a step
    of the sum's magnitude, at most sum_j |ws_j * block_j|, and adding the waves' parts (up
    to 16) likewise; the row's scale and the bias round once each.  The activations'
    slopes are below 1.13.  Their own arithmetic is off by a few roundings (16 counted)
    of the result, and as many of their exponent E times the result (an argument off by
    a rounding moves exp(E) by E of them): |E| is |p| for silu, p^2 for gelu (erfc(-p /
    sqrt 2) falls as exp(-p^2 / 2), and a square doubles its argument's error), 1.6 |p| +
    0.072 |p|^3 for gelu_tanh."""
    xs = np.asarray(scales, np.float64)[:, None]
    parts, bounds = [], []
    for i, (q, s) in enumerate(mats):
        d, nb, _ = q.shape
        p = np.zeros((len(codes), d))
        mag = np.zeros_like(p)
        for j in range(nb):
            block = codes[:, 32 * j:32 * j + 32].astype(np.float64) @ q[:, j].astype(np.float64).T
            p += block * s[:, j].astype(np.float64)
            mag += np.abs(block * s[:, j].astype(np.float64))
        p, e = p * xs, mag * xs * EPS32 * (nb + 16 + 1)
        if bias is not None:
            p = p + np.asarray(bias, np.float64)[i * d:(i + 1) * d]
            e = e + EPS32 * (np.abs(p) + e)
        parts.append(p)
        bounds.append(e)
    y = act(parts[0], activation)
    e = bounds[0] * 1.13
    if activation not in ("none", "relu"):
        p = np.abs(parts[0])
        exponent = {"silu": p, "gelu": p * p, "gelu_tanh": 1.6 * p + 0.072 * p ** 3}[activation]
        e = e + 16 * EPS32 * (1 + exponent) * np.abs(y) + 1e-35
    if len(parts) > 1:
        e = e * (np.abs(parts[1]) + bounds[1]) + bounds[1] * np.abs(y) + EPS32 * np.abs(y * parts[1])
        y = y * parts[1]
    if residual is not None:
        y = y + np.asarray(residual, np.float64)
        e = e + EPS32 * (np.abs(y) + e)
    return y, e + EPS32 * np.abs(y)
