"""Forwards over 8-bit rows into a contiguous cache seen as pages, and into pages in order:
the same launches over the same values, hence the same bits."""
import numpy as np
import pytest

from test_gpu_row8_model import MODELS, model_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", sorted(MODELS))
def test_contiguous_cache(name):
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.model import ROW8

    dim, hid, L, H, G, V, S = MODELS[name]
    kv, pages = G * dim // H, S // 16
    model = na.Model(model_of(name, 8))
    caches = [torch.zeros((L, 16 * pages, kv), device="cuda") for _ in range(2)]
    paged = [torch.zeros((pages, L, 16, kv), device="cuda") for _ in range(2)]
    pools = [na.KVPool.wrap_contiguous(*caches), na.KVPool.wrap(*paged)]
    rng = np.random.default_rng(8)
    prompt, table = rng.integers(0, V, 70).astype(np.int32), np.arange(pages, dtype=np.int32)[None]
    outs = []
    for pool in pools:
        pool.upload_prefill_batch(table, [0], [70])
        got = [model.forward_prefill(pool, prompt, semantics=ROW8).cpu().numpy()]
        for pos in range(70, 76):
            pool.upload_decode_batch(table[:, :pos // 16 + 1], [pos])
            got.append(model.forward_decode_batch(pool, prompt[pos - 70:pos - 69], semantics=ROW8).cpu().numpy())
        outs.append(got)
        assert pool.take_device_errors() == 0
    for a, b in zip(*outs):
        assert np.isfinite(a).all()
        np.testing.assert_array_equal(a, b)
    for cache, pool in zip(caches, paged):
        assert torch.equal(cache[:, :76], pool.transpose(0, 1).reshape(L, 16 * pages, kv)[:, :76])
        assert (cache[:, 76:] == 0).all() and cache[:, :76].abs().sum() > 0
