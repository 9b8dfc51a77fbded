"""A pool over a borrowed 8-bit cache is one of the device that the cache lies on."""
import pytest

pytestmark = pytest.mark.gpu


def test_wrap_refuses_a_cache_of_another_device(monkeypatch):
    import torch

    import nitrorag_amd as na

    cache = torch.zeros((2, 1, 2, na.kv_record_bytes(64)), dtype=torch.uint8, device="cuda")
    na.KVPool.wrap_q8(cache, 64).close()
    # (one GPU: the other one is made current by name only, and nothing is launched)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: cache.device.index + 1)
    with pytest.raises(ValueError, match="not the current device"):
        na.KVPool.wrap_q8(cache, 64)
