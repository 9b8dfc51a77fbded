"""The server over 8-bit rows: clients' tokens are those of a scheduler that is stepped by
hand over the same prompts."""
import ctypes
import socket

import numpy as np
import pytest

from test_gpu_row8_model import MODELS, model_of, pool_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool8", [False, True])
def test_served_tokens(pool8):
    import nitrorag_amd as na
    from nitrorag_amd import _native as N
    from nitrorag_amd.model import ROW8

    name, pages, budget, made = "gqa_hd128_l2", 64, 96, 7
    model, vocab = na.Model(model_of(name, 11)), MODELS[name][5]
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (110, 1, 33)]
    prompts.append(prompts[0][:48] + [9, 8])  # shares cached pages

    sched = na.ContinuousScheduler(na.BlockManager(pages), budget, made)
    by_hand = pool_of(name, pages, pool8)
    for i, p in enumerate(prompts):
        sched.add_request(i, p)
    while sched.has_active_requests():
        sched.step(model, by_hand, ROW8)
    want = [sched.generated(i) for i in range(len(prompts))]
    assert all(len(w) == made for w in want) and len({tuple(w) for w in want}) > 1

    pool, sched = pool_of(name, pages, pool8), na.ContinuousScheduler(na.BlockManager(pages), budget, made)
    server = ctypes.c_void_p()
    N.call("nitro_server_create", sched.handle, model.handle, pool.handle, ROW8, 256, ctypes.byref(server))
    clients = []
    for p in prompts:
        a, b = socket.socketpair()
        b.sendall(np.asarray([len(p)] + p, np.int32).tobytes())
        N.call("nitro_server_accept_fd", server, a.detach(), ctypes.byref(ctypes.c_int32()))
        clients.append(b)
    active = ctypes.c_int32(1)
    for _ in range(100):
        if not active.value:
            break
        N.call("nitro_server_step", server, None, ctypes.byref(active))
    assert not active.value
    for b, tokens in zip(clients, want):
        b.settimeout(10)
        data = b""
        while chunk := b.recv(1 << 16):  # (the server closes a connection after its last token)
            data += chunk
        b.close()
        assert np.frombuffer(data, np.int32).tolist() == list(tokens)
    N.call("nitro_server_destroy", server)
    assert pool.take_device_errors() == 0
