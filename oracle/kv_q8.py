"""Plain 64-bit restatement of the 8-bit K/V cache: its records, the rows put into
them, and attention over the values they hold (numpy; test infrastructure only).
The reference has no 8-bit K/V cache: this follows the definition in
include/nitro_paged_attn.h."""
from __future__ import annotations

import numpy as np

PAGE = 16
LEAST = 2.0 ** -100


def padded(head_dim: int) -> int:
    return (head_dim + 15) // 16 * 16


def record_bytes(head_dim: int) -> int:
    return 32 * padded(head_dim) + 8 * PAGE


def rotate(x, cos, sin):
    """x [rows][heads][head_dim], cos / sin [rows][head_dim/2] fp32 -> fp32."""
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    out = np.empty(x.shape, np.float32)
    out[..., 0::2] = (a * c - b * s).astype(np.float32)
    out[..., 1::2] = (a * s + b * c).astype(np.float32)
    return out


def quantise(k, v):
    """(k codes, k scales, v codes, v scales) of fp32 rows [...][head_dim]."""
    with np.errstate(all="ignore"):
        finite = np.isfinite(k).all(-1) & np.isfinite(v).all(-1)
        got = []
        for x in (k, v):
            top = np.where(finite, np.abs(x).max(-1), 0).astype(np.float32)
            live = top >= np.float32(LEAST)
            safe = np.where(live, top, np.float32(1))
            inverse = np.where(live, np.float32(127) / safe, np.float32(0)).astype(np.float32)
            scale = np.where(live, safe / np.float32(127), np.float32(0)).astype(np.float32)
            exact = np.where(finite[..., None], x, 0).astype(np.float64) * inverse[..., None].astype(np.float64)
            got += [np.rint(exact).astype(np.int8), np.where(finite, scale, np.float32("nan")).astype(np.float32)]
        return tuple(got)


class Cache:
    """Records [pages][layers][kv_heads][record_bytes] as one uint8 array."""

    def __init__(self, data, head_dim):
        self.data, self.hd, self.hdp = data, head_dim, padded(head_dim)

    def _places(self, token):
        """Byte offsets of a token's K codes and V codes for each padded dimension."""
        d = np.arange(self.hdp)
        return ((token // 4 * (self.hdp // 16) + d // 16) * 4 + token % 4) * 16 + d % 16, 16 * self.hdp + d * PAGE + token

    def put(self, layer, slots, k, v):
        """Rows k, v [rows][kv_heads][head_dim] into slots (page * 16 + token)."""
        kc, ks, vc, vs = quantise(k, v)
        pad = ((0, 0), (0, self.hdp - self.hd))
        for r, slot in enumerate(slots):
            page, t = divmod(int(slot), PAGE)
            at_k, at_v = self._places(t)
            rec = self.data[page, layer]
            rec[:, at_k] = np.pad(kc[r], pad).view(np.uint8)
            rec[:, at_v] = np.pad(vc[r], pad).view(np.uint8)
            for base, s in ((0, ks[r]), (64, vs[r])):
                at = 32 * self.hdp + base + 4 * t
                rec[:, at:at + 4] = s[:, None].view(np.uint8)

    def scales(self, layer, table, tokens):
        """K and V scales of a sequence's first `tokens` tokens, float64 [tokens][kv_heads]."""
        at = np.arange(tokens)
        rec = self.data[np.asarray(table)[at // PAGE], layer]
        s = np.ascontiguousarray(rec[:, :, 32 * self.hdp:]).view(np.float32).astype(np.float64)
        return s[at, :, at % PAGE], s[at, :, PAGE + at % PAGE]

    def values(self, layer, table, tokens):
        """K and V of a sequence's first `tokens` tokens, float64 [tokens][kv_heads][head_dim]."""
        k = np.empty((tokens, self.data.shape[2], self.hd))
        v = np.empty_like(k)
        with np.errstate(invalid="ignore"):
            for t in range(PAGE):
                which = np.arange(t, tokens, PAGE)
                if not which.size:
                    continue
                rec = self.data[np.asarray(table)[which // PAGE], layer]  # [n][kv_heads][record]
                at_k, at_v = self._places(t)
                s = np.ascontiguousarray(rec[:, :, 32 * self.hdp:]).view(np.float32).astype(np.float64)
                k[which] = rec[:, :, at_k[:self.hd]].view(np.int8) * s[:, :, t, None]
                v[which] = rec[:, :, at_v[:self.hd]].view(np.int8) * s[:, :, 16 + t, None]
        return k, v


def held(x, heads):
    """fp32 rows [rows][heads * head_dim] as the values they are held as."""
    r = np.ascontiguousarray(x, np.float32).reshape(x.shape[0], heads, -1)
    codes, scale = quantise(r, r)[:2]
    return (codes.astype(np.float32) * scale[..., None]).reshape(x.shape)


class HeldAttention:
    """oracle.attn whose appends put the values that 8 bits hold into the fp32 pools."""

    def __init__(self, attn, heads):
        self._attn, self._heads = attn, heads

    def __getattr__(self, name):
        return getattr(self._attn, name)

    def kv_append_decode(self, k_pool, v_pool, layer, k, v, tables, positions):
        return self._attn.kv_append_decode(k_pool, v_pool, layer, held(k, self._heads), held(v, self._heads), tables,
                                           positions)

    def kv_scatter_prefill(self, k_pool, v_pool, layer, k, v, table, start_pos):
        return self._attn.kv_scatter_prefill(k_pool, v_pool, layer, held(k, self._heads), held(v, self._heads), table,
                                             start_pos)


def attention(q, positions, k, v):
    """q [rows][heads][hd] at `positions` over keys 0..position; with a bound on what
    fp32 arithmetic with 24-bit fixed point may be off, elementwise [rows][heads][1].

    The bound: an entry of q is off by at most 6e-8 of its row's largest a (half a unit
    of a/8355000), so a score is off by that times the key's 1-norm; its joined integer
    by half of 256 units times the key's scale, at most 128 a/8355000 * max|k|/127 =
    1.21e-7 a max|k|; fp32 rounds it about six times (conversions, the two factors, the
    difference from the maximum).  A weight is then off by that, relative, and 2^-22
    (exp2, its sum).  As numerator and denominator: twice.  The weights' own fixed
    point: half a unit (6e-8) of the largest of those that share it, at most 128 of them
    (prefill's two tiles), and the sum of those largest ones is at most the denominator;
    the joined integers of an output half of 256 units once for them, 1.21e-7 of it.
    Joining the tiles: two roundings each."""
    rows, heads, hd = q.shape
    out, bound = np.empty((rows, heads, hd)), np.empty((rows, heads, 1))
    per = heads // k.shape[1]
    for r in range(rows):
        n = int(positions[r]) + 1
        for h in range(heads):
            kh, vh = k[:n, h // per], v[:n, h // per]
            x = q[r, h].astype(np.float64)
            s = kh @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            out[r, h] = p @ vh / p.sum()
            off = np.abs(x).max() * (6e-8 * np.abs(kh).sum(-1).max() + 1.21e-7 * np.abs(kh).max()) / np.sqrt(hd)
            off += 6 * 2.0 ** -24 * np.abs(s).max()
            weight = off + 2.0 ** -22
            tiles = (n + 63) // 64
            bound[r, h] = np.abs(vh).max() * (2 * weight + 128 * 6e-8 + 1.21e-7 + (2 * tiles + 20) * 2.0 ** -24) + 1e-30
    return out, bound


UNITS = 8355000.0  # of a row's largest entry (q) and a group of keys' largest weight


def typical_error(q, positions, k, v, k_scales, v_scales, group, units=UNITS):
    """attention(), and the root mean square of each output row's error norm [rows][heads]
    as the kernels' roundings make it: q and weights in 24-bit fixed point, the integers'
    sums rounded to 256 units, everything else in fp32.  `group` keys share a weight's unit
    (64 in decode, 128 in prefill).

    Each rounding to a step d is taken as uniform in +-d/2 (variance d^2/12; for fp32,
    relative, 2^-48/3) and independent of the others; u_j = v_j - out is what a relative
    change of weight p_j moves the output by, times p_j.
      q        entries off by a step a/units (a: the row's largest; the product before it is
               rounded costs a quarter more): moves along sum_j p_j k_ji u_j / sqrt(hd)
      scores   a step of 256 a/units * ks_j / sqrt(hd) each; two fp32 roundings of s_j, one
               of its distance from the maximum; a factor common to all of a row (four
               roundings), which moves along sum_j p_j s_j u_j
      weights  2^-23 of exp2, a rounding of p vs; a step W/units, W = max p vs of the group,
               times the codes v_j/vs_j
      sums     a step 256 W/units per group and dimension; the group's own factor (2^-23,
               in the output alone) and its place in the softmax (2^-22); two roundings for
               each group of what is summed so far; the sum of the weights and the division"""
    rows, heads, hd = q.shape
    out, typical = np.empty((rows, heads, hd)), np.empty((rows, heads))
    per = heads // k.shape[1]
    eps2 = 2.0 ** -48 / 3
    for r in range(rows):
        n = int(positions[r]) + 1
        starts = np.arange(0, n, group)
        for h in range(heads):
            g = h // per
            kh, vh, ks, vs = k[:n, g], v[:n, g], k_scales[:n, g], v_scales[:n, g]
            x = q[r, h].astype(np.float64)
            a = np.abs(x).max()
            s = kh @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            o = p @ vh
            u = vh - o
            u2, v2 = (u * u).sum(-1), (vh * vh).sum(-1)
            step = a / units
            var = step ** 2 * (5 / 48) / hd * (((kh * p[:, None]).T @ u) ** 2).sum()
            each = (256 * step * ks) ** 2 / (12 * hd) + eps2 * (2 * s * s + (s - s.max()) ** 2)
            var += (p * p * (each + 4 * eps2) * u2).sum() + (p * p * v2).sum() * eps2
            var += 16 * 2.0 ** -48 * (((p * (s - p @ s)) @ u) ** 2).sum()
            W = np.maximum.reduceat(p * vs, starts) / units
            codes2 = v2 / np.where(vs > 0, vs, 1) ** 2
            var += (np.add.reduceat(codes2, starts) / 12 + hd * 256 ** 2 / 12) @ (W * W)
            own, moved = (np.add.reduceat(p[:, None] * z, starts) for z in (vh, u))
            var += 2.0 ** -46 * (own ** 2).sum() + 2.0 ** -44 * (moved ** 2).sum()
            var += 2 * eps2 * (np.cumsum(own, 0) ** 2).sum()
            var += eps2 * (20 + 2 * len(starts)) * (o * o).sum()
            out[r, h], typical[r, h] = o, np.sqrt(var)
    return out, typical
