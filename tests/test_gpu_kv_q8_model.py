"""Model forwards and the scheduler over an 8-bit K/V pool.

The oracle model appends the values that 8 bits hold.  The GPU's K and V rows differ
from the oracle's by fp32 rounding, 1e-6 or so relative, so about one code in 4000
(2 * 127 * 1e-6) is rounded to the neighbour: a whole step in 1/4000 of the values,
where holding them in 8 bits at all moves every value by 0.29 steps rms.  So what
those neighbours may move a logit by is about sqrt(1/4000) / 0.29 = 5% of what the
quantisation itself moves it by, which the fp32 oracle shows; a quarter of the
largest such move is allowed here on top of the logits' bar."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOGIT_ATOL, LOGIT_RTOL = 2e-3, 1e-3

MODELS = {
    # name: (dim, hidden, layers, heads, kv heads, vocab, seq_len)
    "mha_hd64_l3": (256, 512, 3, 4, 4, 1000, 256),
    "gqa_hd128_l2": (512, 1024, 2, 4, 2, 700, 200),
    "gqa_hd96_l2": (384, 512, 2, 4, 2, 400, 160),
}


def say(*a):
    print(*a, flush=True)


class Both:
    """The oracle model with K and V held in 8 bits, and in fp32, over pools of their own."""

    def __init__(self, blob, pages):
        from oracle import attn, kv_q8
        from oracle import model as om

        self.models = [om.OracleModel(blob), om.OracleModel(blob)]
        self.models[0]._attn = kv_q8.HeldAttention(attn, self.models[0].n_kv_heads)
        shape = (pages, self.models[0].n_layers, 16, self.models[0].kv_dim)
        self.pools = [(np.zeros(shape, np.float32), np.zeros(shape, np.float32)) for _ in range(2)]

    def run(self, name, *a, **kw):
        """(logits held in 8 bits, how far fp32's are at most)."""
        got = [getattr(m, name)(k, v, *a, **kw) for m, (k, v) in zip(self.models, self.pools)]
        got = [g if g.ndim == 2 else g[None, :] for g in got]
        return got[0], np.abs(got[0] - got[1]).max()


def check(got, want, moved, what):
    off = np.abs(got - want) - LOGIT_RTOL * np.abs(want) - LOGIT_ATOL
    assert moved > 0.0 and off.max() <= 0.25 * moved, (what, off.max(), moved)


@pytest.mark.parametrize("bulk", [False, True])
@pytest.mark.parametrize("name", sorted(MODELS))
def test_forwards(name, bulk):
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.model import FULL_ROWS, LAST_BLOCK, synthetic_model_file
    from oracle import model as om

    say("8-bit pool:", name, "bulk" if bulk else "full rows")
    dim, hid, L, H, G, V, S = MODELS[name]
    blob = om.scale_residual_outputs(synthetic_model_file(dim, hid, L, H, G, V, S, seed=len(name)), 8.0)
    model, both, sem = na.Model(blob), Both(blob, 96), LAST_BLOCK if bulk else FULL_ROWS
    pool = na.KVPool.create_q8(96, L, G, dim // H)
    bm = na.BlockManager(96)
    rng = np.random.default_rng(21)
    seqs = [na.Sequence(i) for i in range(7)]
    for i, s in enumerate(seqs):
        n = 70 if i == 0 else int(rng.integers(1, 30))
        toks = rng.integers(0, V, n).astype(np.int32)
        for t in toks:
            s.allocate_next_token(int(t), bm)
        table = na.pack_block_tables([s])
        pool.upload_prefill_batch(table, [0], [n])
        got = model.forward_prefill(pool, toks, semantics=sem).cpu().numpy()
        want, moved = both.run("forward_prefill_chunk", table[0], 0, toks, bulk=bulk)
        if n > 1:
            check(got, want, moved, f"prefill {n}")
    for nb in (7, 3, 1, 7):
        toks = rng.integers(0, V, nb).astype(np.int32)
        pos = [s.logical_token_count for s in seqs[:nb]]
        for s, t in zip(seqs, toks):
            s.allocate_next_token(int(t), bm)
        tables = na.pack_block_tables(seqs[:nb])
        pool.upload_decode_batch(tables, pos)
        got = model.forward_decode_batch(pool, toks, semantics=sem).cpu().numpy()
        want, moved = both.run("forward_decode_batch", tables, pos, toks, bulk=bulk)
        check(got, want, moved, f"decode {nb}")
    torch.cuda.synchronize()
    assert pool.take_device_errors() == 0


def test_scheduler_over_an_8_bit_pool():
    """Long and short prompts (the latter's chunks run as decode rows) through the scheduler: each
    token it generates is the largest logit of the same sequence's own forwards, or within what
    neighbouring codes may move a logit of it."""
    import nitrorag_amd as na
    from nitrorag_amd.model import FULL_ROWS, synthetic_model_file
    from oracle import model as om

    dim, hid, L, H, G, V, S = MODELS["gqa_hd128_l2"]
    blob = om.scale_residual_outputs(synthetic_model_file(dim, hid, L, H, G, V, S, seed=3), 8.0)
    model = na.Model(blob)
    pool = na.KVPool.create_q8(64, L, G, dim // H)
    bm = na.BlockManager(64)
    S_ = na.ContinuousScheduler(bm, 96, 6)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, V, n).tolist() for n in (120, 20, 45)]
    prompts.append(prompts[0][:64] + [5, 6, 7])  # shares cached pages
    for i, p in enumerate(prompts):
        S_.add_request(i, p)
    while S_.has_active_requests():
        S_.step(model, pool, FULL_ROWS)
    assert pool.take_device_errors() == 0
    for i, p in enumerate(prompts):
        both = Both(blob, 16)
        table = np.arange(16, dtype=np.int32)
        made = S_.generated(i)
        assert len(made) == 6
        for step, token in enumerate(made):
            if step == 0:
                want, moved = both.run("forward_prefill_chunk", table, 0, p, bulk=False)
            else:
                want, moved = both.run("forward_decode_batch", table[None], [len(p) + step - 1], [made[step - 1]], bulk=False)
            best = want[0].max()
            assert best - want[0][token] <= 0.5 * moved + 2 * (LOGIT_ATOL + LOGIT_RTOL * abs(best)), (i, step)


def test_pools_a_model_refuses():
    import nitrorag_amd as na
    from nitrorag_amd import _native as N
    from nitrorag_amd.model import synthetic_model_file

    model = na.Model(synthetic_model_file(256, 512, 2, 4, 4, 300, 64))
    for layers, heads, hd in ((1, 4, 64), (2, 8, 32), (2, 2, 128)):
        pool = na.KVPool.create_q8(8, layers, heads, hd)
        pool.upload_decode_batch([[0]], [0])
        with pytest.raises(N.NitroError) as e:
            model.forward_decode_batch(pool, [1])
        assert e.value.status == N.INVALID_ARGUMENT
        S = na.ContinuousScheduler(na.BlockManager(8), 32, 4)
        S.add_request(0, [1, 2, 3])
        with pytest.raises(N.NitroError) as e:
            S.step(model, pool)
        assert e.value.status == N.INVALID_ARGUMENT
