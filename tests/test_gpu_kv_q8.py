"""Append, decode and prefill over an 8-bit K/V pool against the plain 64-bit form.

Codes, scales and rotated rows are compared bit for bit (every rounding is part of
the definition); attention within the bound that oracle/kv_q8.py derives."""
import ctypes

import numpy as np
import pytest

from gpu_helpers import random_tables, to_gpu
from oracle import kv_q8

pytestmark = pytest.mark.gpu

# (query heads, K/V heads, head size): one to a K/V head, grouped by 2 to 32, odd sizes
HEADS = [(2, 2, 64), (4, 2, 128), (6, 1, 36), (32, 1, 4), (17, 1, 20), (8, 1, 256), (3, 3, 252), (10, 2, 96), (2, 1, 80),
         (5, 5, 160)]


# head counts with which a prefill of 150 rows is taken by whole pages
PAGEWISE = [(900, 900, 4), (200, 100, 36), (128, 64, 64), (50, 50, 80), (60, 30, 128), (23, 23, 160), (14, 14, 252),
            (14, 14, 256)]


def say(*a):
    print(*a, flush=True)


def freqs(top, hd):
    angle = np.arange(top)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class Case:
    """A pool over a cache of stale bytes (NaN scales among them), tables, and rows."""

    def __init__(self, seed, spans, heads, layers=2, layer=1, spare=3, scale=1.0):
        import nitrorag_amd as na

        self.H, self.G, self.hd = heads
        self.layer, self.spans = layer, spans
        rng = self.rng = np.random.default_rng(seed)
        ctx = np.array([s + n for s, n in spans])
        pages = int(((ctx + 15) // 16).sum()) + spare
        self.tables = random_tables(rng, ctx, pages)
        data = rng.integers(0, 256, (pages, layers, self.G, kv_q8.record_bytes(self.hd)), dtype=np.uint8)
        data[..., 32 * kv_q8.padded(self.hd):] = 0xFF  # scales left: NaN
        self.ref = kv_q8.Cache(data.copy(), self.hd)
        self.cache = to_gpu(data)
        self.pool = na.KVPool.wrap_q8(self.cache, self.hd)
        self.rows = sum(n for _, n in spans)
        self.pos = np.concatenate([np.arange(s, s + n) for s, n in spans])
        self.seq = np.repeat(np.arange(len(spans)), [n for _, n in spans])
        self.slots = self.tables[self.seq, self.pos // 16] * 16 + self.pos % 16
        self.q = (rng.standard_normal((self.rows, self.H * self.hd)) * scale).astype(np.float32)
        self.k, self.v = (rng.standard_normal((self.rows, self.G * self.hd)).astype(np.float32) for _ in range(2))

    def fill(self):
        """Earlier tokens of every sequence, put into both caches."""
        for b, (start, n) in enumerate(self.spans):
            p = np.arange(start)
            k, v = (self.rng.standard_normal((start, self.G, self.hd)).astype(np.float32) for _ in range(2))
            self.ref.put(self.layer, self.tables[b, p // 16] * 16 + p % 16, k, v)
        self.cache.copy_(to_gpu(self.ref.data))

    def heads(self, x):
        return x.reshape(x.shape[0], -1, self.hd)

    def put(self, k=None, v=None):
        self.ref.put(self.layer, self.slots, self.heads(self.k if k is None else k), self.heads(self.v if v is None else v))

    def upload(self, prefill):
        if prefill:
            self.pool.upload_prefill_batch(self.tables, [s for s, _ in self.spans], [n for _, n in self.spans])
        else:
            self.pool.upload_decode_batch(self.tables, [s for s, _ in self.spans])

    def want(self):
        out, bound, row = [], [], 0
        for b, (start, n) in enumerate(self.spans):
            k, v = self.ref.values(self.layer, self.tables[b], start + n)
            o, e = kv_q8.attention(self.heads(self.q)[row:row + n], self.pos[row:row + n], k, v)
            out.append(o), bound.append(e)
            row += n
        return np.concatenate(out), np.concatenate(bound)

    def check(self, got, what):
        want, bound = self.want()
        got = self.heads(got.cpu().numpy().astype(np.float64))
        assert np.isfinite(got).all(), what
        off = np.abs(got - want) / bound
        assert off.max() <= 1, f"{what}: {off.max():.2f} times the bound"

    def same_cache(self):
        np.testing.assert_array_equal(self.cache.cpu().numpy(), self.ref.data)


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("heads", HEADS + PAGEWISE)
def test_append_and_read(heads, prefill, rope):
    import torch

    say("append", heads, "prefill" if prefill else "decode", "rope" if rope else "")
    spans = [(0, 1), (15, 1), (16, 1), (37, 1), (63, 1)]
    if prefill:
        spans = [(0, 1), (5, 40), (16, 16), (31, 17), (0, 0), (40, 2), (14, 1), (15, 1), (8, 70), (3, 2)]
    c = Case(1, spans, heads)
    c.upload(prefill)
    q, k, v = to_gpu(c.q), to_gpu(c.k), to_gpu(c.v)
    if rope:
        cos, sin = freqs(80, c.hd)
        (c.pool.rope_kv_append_prefill if prefill else c.pool.rope_kv_append)(
            c.layer, q, k, v, to_gpu(cos), to_gpu(sin), c.H, c.G, c.hd)
        want_q = kv_q8.rotate(c.heads(c.q), cos[c.pos], sin[c.pos]).reshape(c.q.shape)
        want_k = kv_q8.rotate(c.heads(c.k), cos[c.pos], sin[c.pos]).reshape(c.k.shape)
        np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    else:
        (c.pool.kv_append_prefill if prefill else c.pool.kv_append)(c.layer, k, v)
        want_k = c.k
    np.testing.assert_array_equal(k.cpu().numpy(), want_k)
    c.put(want_k)
    c.same_cache()
    got_k, got_v = torch.full_like(k, np.nan), torch.full_like(v, np.nan)
    (c.pool.kv_read_prefill if prefill else c.pool.kv_read)(c.layer, got_k, got_v)
    kc, ks, vc, vs = kv_q8.quantise(c.heads(want_k), c.heads(c.v))
    np.testing.assert_array_equal(got_k.cpu().numpy(), (kc.astype(np.float32) * ks[..., None]).reshape(c.k.shape))
    np.testing.assert_array_equal(got_v.cpu().numpy(), (vc.astype(np.float32) * vs[..., None]).reshape(c.v.shape))
    assert c.pool.take_device_errors() == 0


@pytest.mark.parametrize("prefill,heads", [(False, 2), (True, 2), (True, 400)])
def test_append_of_unusual_rows(prefill, heads):
    """Zeros, values below the least scale, the largest finite ones, ties, infinities and NaN."""
    say("append unusual rows", prefill, heads)
    c = Case(2, [(3, 24)] if prefill else [(i, 1) for i in range(24)], (2 * heads, heads, 64))
    k, v = c.heads(c.k), c.heads(c.v)
    k[0] = 0
    v[1] = 0
    k[2], v[2] = 1e-38, -1e-42
    k[3, 0], v[3, 1] = 3.4e38, -3.4e38
    k[4] = np.float32(2.0 ** -100) * np.linspace(-1, 1, 64, dtype=np.float32)
    k[5] = np.float32(2.0 ** -101)
    k[6, 0, 3], v[7, 1, 5], k[8, 1, 63], v[9, 0, 0] = np.inf, -np.inf, np.nan, np.nan
    k[10, 0] = 127
    k[10, 0, 1:] = np.arange(63) - 31.5  # codes half way: to even
    c.upload(prefill)
    dk, dv = to_gpu(c.k), to_gpu(c.v)
    (c.pool.kv_append_prefill if prefill else c.pool.kv_append)(c.layer, dk, dv)
    c.put()
    got, want = c.cache.cpu().numpy(), c.ref.data
    split = 32 * 64
    np.testing.assert_array_equal(got[..., :split], want[..., :split])
    np.testing.assert_array_equal(np.ascontiguousarray(got[..., split:]).view(np.float32),
                                  np.ascontiguousarray(want[..., split:]).view(np.float32))


# ------------------------------------------------------------------- decode

CONTEXTS = [[1], [15, 16, 17], [63, 64, 65, 1], [300, 2, 129], [2500]]


@pytest.mark.parametrize("ctx", CONTEXTS)
@pytest.mark.parametrize("heads", HEADS)
def test_decode(heads, ctx):
    import torch

    say("decode", heads, ctx)
    c = Case(3, [(n - 1, 1) for n in ctx], heads)
    c.fill()
    c.upload(False)
    q = to_gpu(c.q)
    out = torch.full_like(q, float("nan"))
    c.pool.decode_append(c.layer, q, to_gpu(c.k), to_gpu(c.v), out, *heads)
    c.put()
    c.same_cache()
    c.check(out, "decode")
    assert c.pool.take_device_errors() == 0
    again = torch.full_like(q, float("nan"))
    c.pool.decode(c.layer, q, again, *heads)
    assert torch.equal(out, again)


@pytest.mark.parametrize("heads,ctx", [((4, 1, 64), [5000] + [1, 90, 300] * 43 + [4100, 7]),
                                       ((2, 2, 128), [700, 1, 1, 64, 65, 3000] * 11 + [1]),
                                       ((3, 1, 36), [1] * 64 + [2500] + [1] * 64),
                                       ((12, 12, 64), [1000, 16, 300, 65, 1] * 7),
                                       ((48, 24, 32), [5, 700, 80] * 43)])
def test_decode_of_many_unequal_sequences(heads, ctx):
    """More sequences than a wave has lanes, a few of them split; unsplit ones, longest first."""
    import torch

    from nitrorag_amd import _native as N

    say("decode, many sequences", heads, len(ctx))
    c = Case(41, [(n - 1, 1) for n in ctx], heads)
    c.fill()
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))
    q = to_gpu(c.q)
    c.upload(False)
    out, again, fixed = (torch.full_like(q, float("nan")) for _ in range(3))
    c.pool.decode(c.layer, q, out, *heads)
    c.check(out, "decode")
    c.pool.decode(c.layer, q, again, *heads)
    assert torch.equal(out, again)
    t, p = to_gpu(c.tables), to_gpu(np.array(ctx, np.int32) - 1)
    assert N.lib().nitro_paged_attn_decode_static(
        c.pool.handle, c.layer, q.data_ptr(), fixed.data_ptr(), t.data_ptr(), p.data_ptr(), len(ctx), c.tables.shape[1],
        max(ctx), *heads, 1, torch.cuda.current_stream().cuda_stream) == N.OK
    c.check(fixed, "static decode")
    assert c.pool.take_device_errors() == 0


@pytest.mark.parametrize("scale", [0.0, 1e-30, 30.0])
def test_decode_of_flat_and_peaked_weights(scale):
    import torch

    say("decode scale", scale)
    heads = (4, 2, 128)
    c = Case(4, [(1499, 1), (70, 1)], heads, scale=scale)
    c.fill()
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))
    c.upload(False)
    out = torch.full((2, 4 * 128), float("nan"), device="cuda")
    c.pool.decode(c.layer, to_gpu(c.q), out, *heads)
    c.check(out, f"scale {scale}")


def test_decode_weights_of_uneven_scales():
    """Values of one token a million times the others': its fixed point is the tile's, and the
    others' share of the output is held to the bound of the largest value."""
    import torch

    heads = (2, 2, 64)
    c = Case(5, [(400, 1)], heads)
    c.fill()
    c.put()
    big = c.rng.standard_normal((1, 2, 64)).astype(np.float32) * 1e6
    c.ref.put(c.layer, [c.tables[0, 3] * 16 + 5], c.rng.standard_normal((1, 2, 64)).astype(np.float32), big)
    c.cache.copy_(to_gpu(c.ref.data))
    c.upload(False)
    out = torch.full((1, 128), float("nan"), device="cuda")
    c.pool.decode(c.layer, to_gpu(c.q), out, *heads)
    c.check(out, "uneven scales")


def test_nonfinite_tokens_reach_the_queries_that_see_them():
    import torch

    heads = (4, 2, 64)
    c = Case(6, [(0, 100), (0, 40)], heads)
    k, v = c.heads(c.k), c.heads(c.v)
    k[30, 0, 5] = np.inf       # sequence 0, token 30, K/V head 0
    v[100 + 20, 1, 7] = np.nan  # sequence 1, token 20, K/V head 1
    c.q[110] = np.inf
    c.upload(True)
    out = torch.full((140, 256), 5.0, device="cuda")
    c.pool.prefill_append(c.layer, to_gpu(c.q), to_gpu(c.k), to_gpu(c.v), out, *heads)
    got = np.isnan(c.heads(out.cpu().numpy())).all(-1)
    assert (np.isnan(c.heads(out.cpu().numpy())).any(-1) == got).all()
    want = np.zeros((140, 4), bool)
    want[30:100, :2] = True
    want[120:, 2:] = True
    want[110] = True
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_scales_that_are_not_finite(which, value):
    """Either scale of a visible token (a caller's own records) makes the outputs that see it NaN."""
    import torch

    heads = (4, 2, 64)
    c = Case(15, [(0, 90)], heads)
    c.put()
    data = c.ref.data.copy()
    at = 32 * 64 + 64 * which + 4 * (37 % 16)
    data[c.tables[0, 37 // 16], c.layer, 1, at:at + 4] = np.array([value], np.float32).view(np.uint8)
    c.cache.copy_(to_gpu(data))
    c.upload(True)
    out = torch.full((90, 256), 5.0, device="cuda")
    c.pool.prefill(c.layer, to_gpu(c.q), out, *heads)
    want = np.zeros((90, 4), bool)
    want[37:, 2:] = True
    np.testing.assert_array_equal(np.isnan(c.heads(out.cpu().numpy())).all(-1), want)
    c.pool.upload_decode_batch(c.tables, [89])
    one = torch.full((1, 256), 5.0, device="cuda")
    c.pool.decode(c.layer, to_gpu(c.q[89:]), one, *heads)
    np.testing.assert_array_equal(np.isnan(c.heads(one.cpu().numpy())).all(-1), want[89:])


@pytest.mark.parametrize("q_scale,k_scale", [(1e29, 1e-29), (1e-29, 1e29), (1e36, 1e-29), (1e-29, 1e36)])
def test_scores_of_far_apart_magnitudes(q_scale, k_scale):
    """q and K of which one is near fp32's end; products up to 1e9 are one-hot weights."""
    import torch

    heads = (2, 2, 64)
    c = Case(16, [(0, 70)], heads)
    c.q *= np.float32(q_scale)
    c.k *= np.float32(k_scale)
    c.upload(True)
    out = torch.full((70, 128), float("nan"), device="cuda")
    c.pool.prefill_append(c.layer, to_gpu(c.q), to_gpu(c.k), to_gpu(c.v), out, *heads)
    c.put()
    c.check(out, "magnitudes")


# ------------------------------------------------------------------ prefill

@pytest.mark.parametrize("spans", [[(0, 1)], [(0, 16), (0, 0), (0, 17)], [(0, 200), (63, 65), (5, 1)], [(129, 70)]])
@pytest.mark.parametrize("heads", HEADS)
def test_prefill(heads, spans):
    import torch

    say("prefill", heads, spans)
    c = Case(7, spans, heads)
    c.fill()
    c.upload(True)
    q = to_gpu(c.q)
    # rows behind the last sequence's stay as they were
    out = torch.full((c.rows + 3, q.shape[1]), -7.0, device="cuda")
    c.pool.prefill_append(c.layer, q, to_gpu(c.k), to_gpu(c.v), out[:c.rows], *heads)
    c.put()
    c.same_cache()
    c.check(out[:c.rows], "prefill")
    assert (out[c.rows:] == -7).all()
    again = torch.full_like(q, float("nan"))
    c.pool.prefill(c.layer, q, again, *heads)
    assert torch.equal(out[:c.rows], again)
    assert c.pool.take_device_errors() == 0


# ----------------------------------------------------------------- together

def test_prompts_then_tokens():
    """Chunks of two prompts, then tokens of both, over two layers, as a program runs them."""
    import torch

    heads = (4, 2, 64)
    H, G, hd = heads
    say("prompts then tokens")
    rng = np.random.default_rng(8)
    import nitrorag_amd as na

    pool = na.KVPool.create_q8(40, 2, G, hd)
    ref = kv_q8.Cache(np.zeros((40, 2, G, kv_q8.record_bytes(hd)), np.uint8), hd)
    tables = rng.permutation(40).astype(np.int32).reshape(2, 20)
    cos, sin = freqs(320, hd)
    dcos, dsin = to_gpu(cos), to_gpu(sin)
    done = [0, 0]
    steps = [("prefill", [100, 37]), ("prefill", [3, 60])] + [("decode", [1, 1])] * 4 + [("prefill", [1, 90])] + [("decode", [1, 1])] * 2
    for kind, new in steps:
        pos = np.concatenate([np.arange(s, s + n) for s, n in zip(done, new)])
        seq = np.repeat([0, 1], new)
        slots = tables[seq, pos // 16] * 16 + pos % 16
        if kind == "prefill":
            pool.upload_prefill_batch(tables, done, new)
        else:
            pool.upload_decode_batch(tables, done)
        for layer in range(2):
            q, k, v = (rng.standard_normal((len(pos), n * hd)).astype(np.float32) for n in (H, G, G))
            dq, dk, dv = to_gpu(q), to_gpu(k), to_gpu(v)
            out = torch.full_like(dq, float("nan"))
            if kind == "prefill":
                pool.rope_kv_append_prefill(layer, dq, dk, dv, dcos, dsin, *heads)
                pool.prefill(layer, dq, out, *heads)
            else:
                pool.rope_kv_append(layer, dq, dk, dv, dcos, dsin, *heads)
                pool.decode(layer, dq, out, *heads)
            rq, rk = (kv_q8.rotate(x.reshape(len(pos), -1, hd), cos[pos], sin[pos]) for x in (q, k))
            ref.put(layer, slots, rk, v.reshape(len(pos), G, hd))
            for b in range(2):
                K, V = ref.values(layer, tables[b], done[b] + new[b])
                want, bound = kv_q8.attention(rq[seq == b], pos[seq == b], K, V)
                off = np.abs(out.cpu().numpy().reshape(len(pos), H, hd)[seq == b] - want) / bound
                assert off.max() <= 1, (kind, new, layer, b, off.max())
        done = [s + n for s, n in zip(done, new)]


def test_chunk_rows_as_decode_rows():
    """Rows of one sequence at consecutive positions in one decode batch (the scheduler's short
    chunks): the same cache bytes as the prefill append, whichever rows share a page."""
    import torch

    heads = (4, 2, 64)
    c = Case(9, [(10, 30)], heads)
    c.fill()
    c.pool.upload_decode_batch(np.repeat(c.tables, 30, 0), c.pos)
    q = to_gpu(c.q)
    out = torch.full_like(q, float("nan"))
    c.pool.decode_append(c.layer, q, to_gpu(c.k), to_gpu(c.v), out, *heads)
    c.put()
    c.same_cache()
    c.check(out, "chunk rows")


def test_captured_steps_replay():
    """A captured append + decode (split over workgroups) and prefill, replayed over new inputs with
    eager work between."""
    import torch

    heads = (8, 2, 128)
    c = Case(10, [(1999, 1), (70, 1), (1023, 1)], heads)
    c.fill()
    c.upload(False)
    q, k, v = to_gpu(c.q), to_gpu(c.k), to_gpu(c.v)
    out = torch.empty_like(q)
    c.pool.decode_append(c.layer, q, k, v, out, *heads)  # sizes the workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.decode_append(c.layer, q, k, v, out, *heads)
    for i in range(4):
        c.q, c.k, c.v = (c.rng.standard_normal(x.shape).astype(np.float32) for x in (c.q, c.k, c.v))
        q.copy_(to_gpu(c.q)), k.copy_(to_gpu(c.k)), v.copy_(to_gpu(c.v))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        c.put()
        c.same_cache()
        c.check(out, f"replay {i}")
        eager = torch.empty_like(out)
        c.pool.decode(c.layer, q, eager, *heads)
        assert torch.equal(eager, out)


def test_captured_decode_outlives_a_larger_launch():
    """A captured split decode keeps its workspace when a later launch of the pool needs a larger one."""
    import torch

    heads = (4, 2, 64)
    c = Case(14, [(1999, 1)], heads, spare=1000)
    c.fill()
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))
    q = to_gpu(c.q)
    out = torch.empty_like(q)
    c.upload(False)
    c.pool.decode(c.layer, q, out, *heads)
    torch.cuda.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.decode(c.layer, q, out, *heads)
    tables = np.concatenate([c.tables[:, :120]] * 8)  # fits the uploaded tables' buffer
    many = q.repeat(8, 1)
    got = torch.empty_like(many)
    c.pool.upload_decode_batch(tables, [1900] * 8)
    c.pool.decode(c.layer, many, got, *heads)
    assert torch.equal(got, got[:1].expand_as(got))
    c.upload(False)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("heads", [(4, 2, 64), (64, 64, 64)])
@pytest.mark.parametrize("rope", [False, True])
def test_captured_prefill_follows_uploads(rope, heads):
    """Captured prefill calls replayed over later batches of as many rows, cut into fewer and more chunks
    than the captured ones: each replay works on the batch uploaded last, as eager calls do."""
    import torch

    import nitrorag_amd as na

    say("captured prefill, later uploads", heads, rope)
    H, G, hd = heads
    rows, width, pages = 192, 9, 64
    rng = np.random.default_rng(21)
    batches = [(rng.permutation(pages)[:len(n) * width].astype(np.int32).reshape(len(n), width), start, n)
               for start, n in (([0, 3], [64, 128]), ([40, 16], [96, 96]), ([9, 0, 24, 79], [7, 0, 120, 65]),
                                ([70, 5], [70, 122]), ([0, 15, 30, 5, 8, 7], [1, 2, 3, 121, 1, 64]))]
    assert all(sum(n) == rows for _, _, n in batches)
    data = rng.integers(0, 256, (pages, 1, G, kv_q8.record_bytes(hd)), dtype=np.uint8)
    scales = np.abs(rng.standard_normal((pages, 1, G, 32))).astype(np.float32)
    data[..., 32 * hd:] = scales.view(np.uint8)
    clean = to_gpu(data)
    cache = clean.clone()
    pool = na.KVPool.wrap_q8(cache, hd)
    q0, k0, v = (to_gpu(rng.standard_normal((rows, n * hd)).astype(np.float32)) for n in (H, G, G))
    cos, sin = (to_gpu(x) for x in freqs(16 * width, hd))
    state = q, k, out, kr, vr = [torch.empty_like(x) for x in (q0, k0, q0, k0, v)]

    def reset():
        cache.copy_(clean), q.copy_(q0), k.copy_(k0)
        for x in (out, kr, vr):
            x.fill_(float("nan"))

    def step():
        if rope:
            pool.rope_kv_append_prefill(0, q, k, v, cos, sin, *heads)
        else:
            pool.kv_append_prefill(0, k, v)
        pool.kv_read_prefill(0, kr, vr)
        pool.prefill(0, q, out, *heads)

    pool.upload_prefill_batch(*batches[-1])  # sizes every buffer
    for captured in (0, 4):
        pool.upload_prefill_batch(*batches[captured])
        reset()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for i in (0, 1, 4, 2, 3, 0):
            pool.upload_prefill_batch(*batches[i])
            reset()
            graph.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in (cache, *state)]
            assert torch.isfinite(out).all()
            reset()
            step()
            torch.cuda.synchronize()
            for name, g, w in zip(("cache", "q", "k", "out", "read k", "read v"), got, (cache, *state)):
                assert torch.equal(g, w), f"captured {captured}, replayed over {i}: {name}"
        del graph
    assert pool.take_device_errors() == 0


@pytest.mark.parametrize("heads", [(2, 2, 64), (8, 1, 128), (100, 100, 32)])
def test_captured_decode_follows_uploads(heads):
    """A captured decode replayed over a later batch of the same tables with longer sequences (its splits
    are then longer) and over its own."""
    import torch

    say("captured decode, later uploads", heads)
    for short in (40, 700):
        c = Case(22, [(3000, 1), (2047, 1), (64, 1)], heads)
        c.fill()
        c.put()
        c.cache.copy_(to_gpu(c.ref.data))
        q = to_gpu(c.q)
        out = torch.empty_like(q)
        for pos in ([3000, 2047, 64], [short, 20, 64]):  # the workspace, then what is captured
            c.pool.upload_decode_batch(c.tables, pos)
            c.pool.decode(c.layer, q, out, *heads)
        torch.cuda.synchronize()
        first = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.pool.decode(c.layer, q, out, *heads)
        for i in range(3):
            out.fill_(float("nan"))
            c.upload(False)
            graph.replay()
            torch.cuda.synchronize()
            c.check(out, f"captured at {short}, replay {i}")
            c.pool.upload_decode_batch(c.tables, [short, 20, 64])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, first)
            c.upload(False)
            c.pool.decode(c.layer, q, out, *heads)
            c.check(out, f"eager after {i}")
        del graph


def test_on_another_stream():
    import torch

    heads = (4, 4, 64)
    c = Case(11, [(700, 1), (33, 1)], heads)
    c.fill()
    s = torch.cuda.Stream()
    q, k, v = to_gpu(c.q), to_gpu(c.k), to_gpu(c.v)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        c.upload(False)
        c.pool.decode_append(c.layer, q, k, v, out, *heads)
    s.synchronize()
    c.put()
    c.check(out, "stream")


def test_two_pools_on_two_streams():
    """Split decodes and prefills of two pools that overlap: each pool has its own workspace."""
    import torch

    heads = (8, 2, 128)
    cases = [Case(31, [(2999, 1), (1500, 1)], heads), Case(32, [(2000, 1), (2700, 1)], heads)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for c in cases:
        c.fill()
        c.put()
        c.cache.copy_(to_gpu(c.ref.data))
        c.upload(False)
        c.upload(True)
        q = to_gpu(c.q)
        outs = torch.empty_like(q), torch.empty_like(q)
        c.pool.decode(c.layer, q, outs[0], *heads)  # sizes the workspace
        c.pool.prefill(c.layer, q, outs[1], *heads)
        jobs.append((c, q, outs))
    torch.cuda.synchronize()
    want = [[o.clone() for o in outs] for _, _, outs in jobs]
    for _ in range(20):
        for (c, q, outs), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                c.pool.decode(c.layer, q, outs[0], *heads)
                c.pool.prefill(c.layer, q, outs[1], *heads)
    torch.cuda.synchronize()
    for (c, _, outs), w in zip(jobs, want):
        for o, e, what in zip(outs, w, ("decode", "prefill")):
            assert torch.equal(o, e), what
            c.check(o, what)


def test_static_decode_and_bad_pages():
    """The allocation-free form gives the uploaded form's bits; page ids outside the pool are counted
    and their keys left out; a position below 0 gives zeros."""
    import torch

    from nitrorag_amd import _native as N

    heads = (4, 2, 64)
    c = Case(12, [(1599, 1), (40, 1), (799, 1)], heads)
    c.fill()
    c.put()
    c.cache.copy_(to_gpu(c.ref.data))

    def static(tables, positions, out, limit):
        t, p, q = to_gpu(tables), to_gpu(np.asarray(positions, np.int32)), to_gpu(c.q)
        st = N.lib().nitro_paged_attn_decode_static(
            c.pool.handle, c.layer, q.data_ptr(), out.data_ptr(), t.data_ptr(), p.data_ptr(), 3, tables.shape[1], limit,
            *heads, 0, None)
        torch.cuda.synchronize()
        return st

    out = torch.full((3, 256), float("nan"), device="cuda")
    for _ in range(2):
        out.fill_(float("nan"))
        assert static(c.tables, [1599, 40, 799], out, 1600) == N.OK
        c.check(out, "static")
    say("bad pages")
    tables = c.tables.copy()
    tables[1, 2], tables[2, 7] = -1, c.cache.shape[0]
    assert static(tables, [1599, 40, 799], out, 1600) == N.OK
    assert c.pool.take_device_errors() > 0
    got = out.cpu().numpy().reshape(3, 4, 64)
    for b, gone in ((1, 2), (2, 7)):
        n = [1600, 41, 800][b]
        k, v = c.ref.values(c.layer, c.tables[b], n)
        keep = np.arange(n) // 16 != gone
        want, bound = kv_q8.attention(c.heads(c.q)[b:b + 1], [keep.sum() - 1], k[keep], v[keep])
        assert (np.abs(got[b] - want[0]) <= bound[0]).all()
    assert static(c.tables, [-1, 40, 799], out, 1600) == N.OK
    assert (out[0] == 0).all() and c.pool.take_device_errors() > 0
    assert static(c.tables, [1599, 40, 799], out, 16 * c.tables.shape[1] + 1) == N.INVALID_ARGUMENT


def test_records_past_4_gib():
    """Pages whose records lie past 2^32 bytes of the cache."""
    import torch

    import nitrorag_amd as na

    hd, G, L = 128, 8, 16
    pages = (5 << 30) // (kv_q8.record_bytes(hd) * G * L)
    say("cache of", pages, "pages")
    pool = na.KVPool.create_q8(pages, L, G, hd)
    table = np.array([[pages - 1, 3, pages - 9, pages - 2]], np.int32)
    rng = np.random.default_rng(13)
    ref = kv_q8.Cache(np.zeros((4, 1, G, kv_q8.record_bytes(hd)), np.uint8), hd)
    k, v = (rng.standard_normal((60, G * hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((60, G * hd)).astype(np.float32)
    pool.upload_prefill_batch(table, [0], [60])
    out = torch.full((60, G * hd), float("nan"), device="cuda")
    pool.prefill_append(L - 1, to_gpu(q), to_gpu(k), to_gpu(v), out, G, G, hd)
    ref.put(0, np.arange(60), k.reshape(60, G, hd), v.reshape(60, G, hd))
    K, V = ref.values(0, np.arange(4), 60)
    want, bound = kv_q8.attention(q.reshape(60, G, hd), np.arange(60), K, V)
    assert (np.abs(out.cpu().numpy().reshape(60, G, hd) - want) <= bound).all()
    pool.upload_decode_batch(table, [59])
    one = torch.full((1, G * hd), float("nan"), device="cuda")
    pool.decode(L - 1, to_gpu(q[59:]), one, G, G, hd)
    assert (np.abs(one.cpu().numpy().reshape(1, G, hd) - want[59:]) <= bound[59:]).all()
    pool.close()


def test_refusals():
    import torch

    import nitrorag_amd as na
    from nitrorag_amd import _native as N

    def refused(status, f, *a):
        with pytest.raises(N.NitroError) as e:
            f(*a)
        assert e.value.status == status, e.value

    pool = na.KVPool.create_q8(8, 2, 2, 64)
    q, k = torch.zeros((1, 256), device="cuda"), torch.zeros((1, 128), device="cuda")
    refused(N.NO_BATCH, pool.kv_append, 0, k, k)
    refused(N.NO_BATCH, pool.kv_read, 0, k, k)
    refused(N.NO_BATCH, pool.kv_read_prefill, 0, k, k)
    refused(N.NO_BATCH, pool.decode, 0, q, q, 4, 2, 64)
    refused(N.NO_BATCH, pool.prefill, 0, q, q, 4, 2, 64)
    refused(N.BAD_BLOCK_TABLE, pool.upload_decode_batch, [[8]], [0])
    pool.upload_decode_batch([[7]], [0])
    refused(N.INVALID_ARGUMENT, pool.kv_append, 2, k, k)
    refused(N.INVALID_ARGUMENT, pool.kv_read, -1, k, k)
    refused(N.INVALID_ARGUMENT, pool.decode, 0, torch.zeros((1, 128), device="cuda"), k, 4, 4, 32)  # another cut of kv_dim
    three = torch.zeros((1, 192), device="cuda")
    refused(N.UNSUPPORTED, pool.decode, 0, three, three, 3, 2, 64)
    refused(N.UNSUPPORTED, pool.data_ptrs)
    with pytest.raises(ValueError):
        pool.kv_append(0, q, q)
    with pytest.raises(TypeError):
        pool.kv_append(0, k.half(), k)
    fp32 = na.KVPool(8, 2, 128)
    fp32.upload_decode_batch([[7]], [0])
    refused(N.UNSUPPORTED, fp32.kv_read, 0, k, k)
    refused(N.UNSUPPORTED, fp32.q8_data_ptr)
    rec = na.kv_record_bytes(64)
    good = torch.zeros((2, 1, 2, rec), dtype=torch.uint8, device="cuda")
    assert na.KVPool.wrap_q8(good, 64).q8_data_ptr() == good.data_ptr()
    with pytest.raises(ValueError):
        na.KVPool.wrap_q8(good, 80)
    with pytest.raises(TypeError):
        na.KVPool.wrap_q8(good.transpose(0, 2), 64)
    with pytest.raises(TypeError):
        na.KVPool.wrap_q8(good.cpu(), 64)
    assert ctypes.c_void_p(pool.q8_data_ptr()).value % 16 == 0
