"""What the accuracy check of 8-bit attention notices, on the CPU: a model of the kernels'
arithmetic passes it with the 24 bits they have, and fails it with fewer."""
import numpy as np
import pytest

from kv_q8_error import check_error
from oracle import kv_q8

f32 = np.float32


def row(q, kc, ks, vc, vs, group, q_units, w_units):
    """One query row over codes [n][hd] and scales [n]: the kernels' steps in fp32 and
    integers, with q and the weights as multiples of 1/q_units and 1/w_units."""
    hd = q.size
    top = np.abs(q).max()
    inv = f32(f32(q_units) / top)
    digits = np.rint(q * inv).astype(np.int64)
    scale = f32(top * f32(f32(1.4426950408889634 / np.sqrt(hd)) * f32(256.0 * 2.0 ** 20 / q_units)))
    m, l, o = f32(-np.inf), f32(0), np.zeros(hd, f32)
    for t in range(0, len(ks), group):
        K, V = kc[t:t + group].astype(np.int64), vc[t:t + group].astype(np.int64)
        s = (((K @ digits + 128) >> 8).astype(f32) * (ks[t:t + group] * f32(2.0 ** -20))).astype(f32)
        base = f32(s.max() * scale)
        p = np.exp2((s.astype(np.float64) * np.float64(scale) - np.float64(base)).astype(f32)).astype(f32)
        w = (p * vs[t:t + group]).astype(f32)
        big = w.max()
        held = np.rint(w.astype(np.float64) * np.float64(f32(f32(w_units) * f32(1 / big)))).astype(np.int64)
        new = max(m, base)
        f, alpha = f32(np.exp2(f32(base - new))), f32(0) if m == -np.inf else f32(np.exp2(f32(m - new)))
        l, m = f32(f32(l * alpha) + f32(p.sum() * f)), new
        unit = f32(f32(big * f32(256 / w_units)) * f)
        joined = ((held @ V + 128) >> 8).astype(f32).astype(np.float64)
        o = (joined * np.float64(unit) + (o * alpha).astype(f32)).astype(f32)
    return o * f32(1 / l)


def case(seed, hd, n, group, scale, q_units, w_units, rows=12):
    rng = np.random.default_rng(seed)
    got, want, typical = [], [], []
    for _ in range(rows):
        q = (rng.standard_normal(hd) * scale).astype(f32)
        k, v = (rng.standard_normal((n, 1, hd)).astype(f32) for _ in range(2))
        kc, ks, vc, vs = kv_q8.quantise(k, v)
        o, e = kv_q8.typical_error(q[None, None], [n - 1], kc * ks[..., None].astype(np.float64),
                                   vc * vs[..., None].astype(np.float64), ks.astype(np.float64), vs.astype(np.float64), group)
        got.append(row(q, kc[:, 0], ks[:, 0], vc[:, 0], vs[:, 0], group, q_units, w_units))
        want.append(o[0, 0]), typical.append(e[0, 0])
    return np.array(got)[:, None], np.array(want)[:, None], np.array(typical)[:, None]


SIZES = [(hd, n, group) for hd in (4, 36, 64, 128, 256) for n in (4, 64, 300, 2500) for group in (64, 128)]


@pytest.mark.parametrize("hd,n,group", SIZES + [(64, 1, 64), (128, 1, 128)])
@pytest.mark.parametrize("scale", [1.0, 30.0])
def test_24_bits_pass(hd, n, group, scale):
    got, want, typical = case(1, hd, n, group, scale, kv_q8.UNITS, kv_q8.UNITS)
    check_error(got, want, typical, "24 bits")


@pytest.mark.parametrize("hd,n,group", SIZES)
@pytest.mark.parametrize("bits", [16, 20])
@pytest.mark.parametrize("which", ["q", "weights", "both"])
def test_fewer_bits_fail(hd, n, group, bits, which):
    few = kv_q8.UNITS / 2 ** (24 - bits)
    got, want, typical = case(1, hd, n, group, 1.0, kv_q8.UNITS if which == "weights" else few,
                              kv_q8.UNITS if which == "q" else few)
    with pytest.raises(AssertionError, match="typical error"):
        check_error(got, want, typical, f"{bits} bits of {which}")
