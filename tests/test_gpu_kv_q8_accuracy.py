"""Attention over an 8-bit pool at every build of its kernels, with each row's error norm
held to what 24-bit fixed point and fp32 sums make of it (a lost digit, or 20 bits, fail;
test_kv_q8_accuracy.py)."""
import numpy as np
import pytest

from gpu_helpers import to_gpu
from kv_q8_error import check_error
from oracle import kv_q8
from test_gpu_kv_q8 import HEADS, Case, say

pytestmark = pytest.mark.gpu

# One of each number of 16-dimension runs that HEADS lacks, head sizes that fill the last
# run and ones that do not, and workgroups of two waves (16 query heads or more to a K/V
# head at head sizes past 248), one with two groups of query heads.
MORE = [(3, 3, 32), (4, 2, 48), (2, 1, 100), (4, 4, 112), (2, 2, 132), (6, 3, 144), (2, 1, 164), (3, 1, 176), (2, 2, 180),
        (4, 2, 192), (2, 1, 196), (3, 3, 208), (2, 2, 212), (4, 2, 224), (2, 1, 228), (5, 5, 240), (16, 1, 256), (16, 1, 252),
        (20, 1, 256)]


class Tight(Case):
    def check(self, got, what, group):
        super().check(got, what)
        got = self.heads(got.cpu().numpy())
        want, typical, row = [], [], 0
        for b, (start, n) in enumerate(self.spans):
            if n == 0:
                continue
            table = self.tables[b]
            k, v = self.ref.values(self.layer, table, start + n)
            o, e = kv_q8.typical_error(self.heads(self.q)[row:row + n], self.pos[row:row + n], k, v,
                                       *self.ref.scales(self.layer, table, start + n), group)
            want.append(o), typical.append(e)
            row += n
        check_error(got, np.concatenate(want), np.concatenate(typical), what)


def filled(*a, **kw):
    c = Tight(*a, **kw)
    c.fill()
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))
    return c


@pytest.mark.parametrize("ctx", [[1, 4], [17, 64, 65, 129], [300, 2, 2500]])
@pytest.mark.parametrize("heads", HEADS + MORE)
def test_decode(heads, ctx):
    import torch

    from nitrorag_amd import _native as N

    say("decode", heads, ctx)
    c = filled(61, [(n - 1, 1) for n in ctx], heads)
    q = to_gpu(c.q)
    out, again, fixed = (torch.full_like(q, float("nan")) for _ in range(3))
    c.upload(False)
    c.pool.decode(c.layer, q, out, *heads)
    c.check(out, "decode", 64)
    c.pool.decode(c.layer, q, again, *heads)
    assert torch.equal(out, again)
    t, p = to_gpu(c.tables), to_gpu(np.array(ctx, np.int32) - 1)
    assert N.lib().nitro_paged_attn_decode_static(
        c.pool.handle, c.layer, q.data_ptr(), fixed.data_ptr(), t.data_ptr(), p.data_ptr(), len(ctx), c.tables.shape[1],
        max(ctx), *heads, 1, torch.cuda.current_stream().cuda_stream) == N.OK
    c.check(fixed, "static decode", 64)
    # two sequences over the same pages (loads that stay in the caches)
    twice = to_gpu(np.repeat(c.q[-1:], 2, 0))
    shared = torch.full_like(twice, float("nan"))
    c.pool.upload_decode_batch(np.repeat(c.tables[-1:], 2, 0), np.repeat(c.pos[-1:], 2))
    c.pool.decode(c.layer, twice, shared, *heads)
    assert torch.equal(shared[0], shared[1])
    c.check(torch.cat([out[:-1], shared[:1]]), "shared pages", 64)
    assert c.pool.take_device_errors() == 0


@pytest.mark.parametrize("spans", [[(0, 17), (0, 1)], [(0, 150), (63, 66), (5, 1)]])
@pytest.mark.parametrize("heads", HEADS + MORE)
def test_prefill(heads, spans):
    import torch

    say("prefill", heads, spans)
    c = Tight(62, spans, heads)
    c.fill()
    c.upload(True)
    q = to_gpu(c.q)
    out = torch.full((c.rows + 3, q.shape[1]), -7.0, device="cuda")
    c.pool.prefill_append(c.layer, q, to_gpu(c.k), to_gpu(c.v), out[:c.rows], *heads)
    c.put()
    c.same_cache()
    c.check(out[:c.rows], "prefill", 128)
    assert (out[c.rows:] == -7).all()
    assert c.pool.take_device_errors() == 0


@pytest.mark.parametrize("heads", [(4, 2, 128), (6, 3, 64), (2, 1, 176)])
def test_peaked_weights(heads):
    import torch

    say("peaked", heads)
    c = filled(63, [(1499, 1), (70, 1), (0, 90)], heads, scale=30.0)
    for prefill in (False, True):
        out = torch.full_like(to_gpu(c.q), float("nan"))
        if prefill:
            c.upload(True)
            c.pool.prefill(c.layer, to_gpu(c.q), out, *heads)
        else:
            c.pool.upload_decode_batch(np.repeat(c.tables, [1, 1, 90], 0), c.pos)
            c.pool.decode(c.layer, to_gpu(c.q), out, *heads)
        c.check(out, "prefill" if prefill else "decode", 128 if prefill else 64)


@pytest.mark.parametrize("heads,ctx", [((4, 1, 64), [5000] + [1, 90, 300] * 43 + [4100, 7]),
                                       ((2, 2, 128), [700, 1, 1, 64, 65, 3000] * 11 + [1]),
                                       ((12, 12, 64), [1000, 16, 300, 65, 1] * 7),
                                       ((16, 1, 256), [3000, 100, 1500])])
def test_decode_of_unequal_sequences(heads, ctx):
    import torch

    say("decode, unequal", heads, len(ctx))
    c = filled(64, [(n - 1, 1) for n in ctx], heads)
    c.upload(False)
    out = torch.full_like(to_gpu(c.q), float("nan"))
    c.pool.decode(c.layer, to_gpu(c.q), out, *heads)
    c.check(out, "decode", 64)


@pytest.mark.parametrize("heads,tokens", [((8, 1, 64), 131072), ((8, 2, 64), 131072 - 37), ((1, 1, 64), 131072),
                                          ((16, 1, 256), 32768 + 5)])
def test_joins_of_many_splits(heads, tokens):
    """One long sequence over few heads: more splits than a wave has lanes."""
    import torch

    import nitrorag_amd as na

    H, G, hd = heads
    say("join", heads, tokens)
    rng = np.random.default_rng(65)
    pages = (tokens + 15) // 16
    data = rng.integers(0, 256, (pages, 1, G, kv_q8.record_bytes(hd)), dtype=np.uint8)
    scales = (rng.uniform(0.5, 1.5, (pages, 1, G, 32)) / 60).astype(np.float32)  # values near N(0, 1.2)
    data[..., 32 * hd:] = scales.view(np.uint8)
    ref, cache = kv_q8.Cache(data, hd), to_gpu(data)
    pool = na.KVPool.wrap_q8(cache, hd)
    table = rng.permutation(pages).astype(np.int32)[None]
    q = rng.standard_normal((1, H * hd)).astype(np.float32)
    dq = to_gpu(q)
    out, again = torch.full_like(dq, float("nan")), torch.full_like(dq, float("nan"))
    pool.upload_decode_batch(table, [tokens - 1])
    pool.decode(0, dq, out, *heads)
    pool.decode(0, dq, again, *heads)
    assert torch.equal(out, again)
    k, v = ref.values(0, table[0], tokens)
    want, typical = kv_q8.typical_error(q.reshape(1, H, hd), [tokens - 1], k, v, *ref.scales(0, table[0], tokens), 64)
    check_error(out.cpu().numpy().reshape(1, H, hd), want, typical, "join")
    assert pool.take_device_errors() == 0


@pytest.mark.parametrize("prefill", [False, True])
def test_the_range_of_scores(prefill):
    """Scores up to fp32's end, of either sign, are one-hot weights; a row whose scores pass it
    leaves the others as they were; a q below 2^-100 counts as zeros."""
    import torch

    heads = (2, 2, 64)
    say("range of scores", prefill)
    c = Tight(66, [(0, 130)], heads)
    K = c.heads(c.k)
    K *= np.float32(1e3)
    K[..., 0] = 3000 + 7 * c.rng.permutation(130)[:, None]
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))
    k, v = c.ref.values(c.layer, c.tables[0], 130)
    plain = c.q.copy()
    Q = c.heads(c.q)
    far = {}
    for i, power in enumerate((2, 3, 4, 5, 6, 7, 8, 9, 10, 15, 20, 30, 32)):
        far[30 + 3 * i] = power + 1.0
        Q[30 + 3 * i] *= np.float32(10.0 ** (power + 1))
        for row, sign in ((31 + 3 * i, 1), (32 + 3 * i, -1)):  # scores of one sign
            far[row] = sign
            Q[row] = 0
            Q[row, :, 0] = sign * np.float32(10.0 ** power)
    Q[80] *= np.float32(1e36)   # scores past 1e39
    Q[85] *= np.float32(2e-31)  # below 2^-100 (8e-31)
    outs = []
    for q in (plain, c.q):
        out = torch.full((130, 128), float("nan"), device="cuda")
        if prefill:
            c.upload(True)
            c.pool.prefill(c.layer, to_gpu(q), out, *heads)
        else:
            c.pool.upload_decode_batch(np.repeat(c.tables, 130, 0), c.pos)
            c.pool.decode(c.layer, to_gpu(q), out, *heads)
        outs.append(c.heads(out.cpu().numpy()))
    same = np.ones(130, bool)
    same[[80, 85, *far]] = False
    assert np.isfinite(outs[0]).all()
    np.testing.assert_array_equal(outs[1][same], outs[0][same])
    seen = 0
    for row in far:
        for h in range(2):
            s = k[:row + 1, h] @ Q[row, h].astype(np.float64) / 8
            first, second = np.sort(s)[[-1, -2]]
            # (a score is off by the steps of q and of the joined integer, and six roundings)
            off = np.abs(Q[row, h]).max() * (6e-8 * np.abs(k[:row + 1, h]).sum(-1).max() + 1.21e-7 * np.abs(k).max()) / 8
            if first - second < 40 + 2 * (off + 6 * 2.0 ** -24 * np.abs(s).max()):
                continue
            seen += 1
            # one weight of 1 beside 130 of e^-40: its step, the joined integer's, three roundings
            want = v[int(np.argmax(s)), h]
            assert np.abs(outs[1][row, h] - want).max() <= np.abs(want).max() * 5e-7, (row, far[row], h)
    assert seen >= 60, seen
    for h in range(2):
        mean = v[:86, h].mean(0)
        assert np.abs(outs[1][85, h] - mean).max() <= np.abs(v[:86, h]).max() * 128 * 6e-8
