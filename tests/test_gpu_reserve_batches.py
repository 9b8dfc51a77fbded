"""Captured calls and later uploads that need more room than the captured batch: within
nitro_kvpool_reserve_batches they follow the uploads, past it they go on over the batch that
their own arrays hold."""
import numpy as np
import pytest

from gpu_helpers import to_gpu
from oracle import kv_q8

pytestmark = pytest.mark.gpu

H, G, HD, PAGES, WIDTH = 4, 2, 64, 80, 64


def make_pool(kind, rng):
    import nitrorag_amd as na

    if kind == "fp32":
        k, v = (to_gpu(rng.standard_normal((PAGES, 1, 16, G * HD)).astype(np.float32)) for _ in range(2))
        return na.KVPool.wrap(k, v)
    data = rng.integers(0, 256, (PAGES, 1, G, kv_q8.record_bytes(HD)), dtype=np.uint8)
    data[..., 32 * HD:] = np.abs(rng.standard_normal((PAGES, 1, G, 32))).astype(np.float32).view(np.uint8)
    pool = na.KVPool.wrap_q8(to_gpu(data), HD)
    pool.plain = kv_q8.Cache(data, HD)
    return pool


def tables_of(rng, n):
    """Rows of WIDTH entries; every entry is a page of the pool, 4 of each sequence's own."""
    t = rng.integers(0, PAGES, (n, WIDTH)).astype(np.int32)
    t[:, :4] = rng.permutation(PAGES)[:4 * n].reshape(n, 4)
    return t


def cut(rng, rows, chunks):
    at = np.sort(rng.choice(np.arange(1, rows), chunks - 1, replace=False))
    return np.diff(np.concatenate([[0], at, [rows]]))


def test_captured_prefill_follows_uploads_of_more_chunks():
    import torch

    rng = np.random.default_rng(51)
    pool = make_pool("q8", rng)
    rows = 160  # chunks end below position 64
    batches = []
    for chunks in (8, 17, 19, 4):
        while True:
            n = cut(rng, rows, chunks)
            if n.max() <= 60:
                break
        batches.append((tables_of(rng, chunks), [int(rng.integers(0, 64 - x + 1)) for x in n], n))
    q, k, v = (to_gpu(rng.standard_normal((rows, n * HD)).astype(np.float32)) for n in (H, G, G))
    out = torch.empty_like(q)

    def step():
        pool.kv_append_prefill(0, k, v)
        pool.prefill(0, q, out, H, G, HD)

    pool.reserve_batches(19, WIDTH, rows)
    pool.upload_prefill_batch(*batches[0])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (1, 0, 2, 3, 1):
        print("replay over", len(batches[i][2]), "chunks", flush=True)
        pool.upload_prefill_batch(*batches[i])
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(float("nan"))
        step()  # (the same rows into the same slots again)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and torch.equal(got, out)
    del graph
    assert pool.take_device_errors() == 0


def test_captured_decode_follows_uploads_after_a_larger_batch():
    import torch

    rng = np.random.default_rng(52)
    pool = make_pool("q8", rng)
    pool.reserve_batches(40, WIDTH)
    few, many = tables_of(rng, 3), rng.integers(0, PAGES, (40, WIDTH)).astype(np.int32)
    q, wide = (to_gpu(rng.standard_normal((n, H * HD)).astype(np.float32)) for n in (3, 40))
    out, other = torch.empty_like(q), torch.empty_like(wide)

    def step():
        pool.decode(0, q, out, H, G, HD)

    pool.upload_decode_batch(few, [1000, 30, 500])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for pos in ([1000, 30, 500], [5, 1023, 64], [0, 0, 0]):
        pool.upload_decode_batch(many, rng.integers(0, 1024, 40))
        pool.decode(0, wide, other, H, G, HD)
        pool.upload_decode_batch(few, pos)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(3):
            k, v = pool.plain.values(0, few[i], pos[i] + 1)
            want, bound = kv_q8.attention(q[i:i + 1].cpu().numpy().reshape(1, H, HD), [pos[i]], k, v)
            off = np.abs(out[i].cpu().numpy().reshape(1, H, HD) - want) / bound
            assert off.max() <= 1, (pos, i, off.max())
    del graph


@pytest.mark.parametrize("kind", ["fp32", "q8"])
def test_what_is_captured_keeps_its_arrays_when_an_upload_outgrows_them(kind):
    import torch

    rng = np.random.default_rng(53)
    pool = make_pool(kind, rng)
    few, many = tables_of(rng, 3), rng.integers(0, PAGES, (100, WIDTH)).astype(np.int32)
    q, rows = (to_gpu(rng.standard_normal((n, H * HD)).astype(np.float32)) for n in (3, 90))
    outs = torch.empty_like(q), torch.empty_like(rows)

    def step():
        pool.decode(0, q, outs[0], H, G, HD)
        pool.prefill(0, rows, outs[1], H, G, HD)

    pool.upload_decode_batch(few, [300, 30, 63])
    pool.upload_prefill_batch(few, [10, 0, 3], [40, 20, 30])
    step()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        if i:  # 6400 words of tables, then as many again
            pool.upload_decode_batch(many, rng.integers(0, 64, 100))
            pool.upload_prefill_batch(np.repeat(many, i, 0), np.zeros(100 * i, int), np.full(100 * i, 2))
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), i
    del graph


def test_a_batch_is_uploaded_again_where_its_arrays_moved():
    import torch

    from nitrorag_amd import _native as N

    rng = np.random.default_rng(54)
    pool = make_pool("q8", rng)
    q = to_gpu(rng.standard_normal((1, H * HD)).astype(np.float32))
    out = torch.empty_like(q)
    pool.upload_decode_batch(tables_of(rng, 1), [5])
    pool.upload_prefill_batch(tables_of(rng, 1), [5], [1])
    pool.reserve_batches(4, WIDTH, 10)  # within the room: both stay
    pool.decode(0, q, out, H, G, HD)
    pool.prefill(0, q, out, H, G, HD)
    pool.reserve_batches(100, WIDTH)
    pool.prefill(0, q, out, H, G, HD)
    for call in (pool.decode, pool.prefill):
        if call == pool.prefill:
            pool.reserve_batches(100, WIDTH, 200)
        with pytest.raises(N.NitroError) as e:
            call(0, q, out, H, G, HD)
        assert e.value.status == N.NO_BATCH
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, -1)):
        with pytest.raises(N.NitroError) as e:
            pool.reserve_batches(*bad)
        assert e.value.status == N.INVALID_ARGUMENT
