"""Model forwards, the scheduler and the server with what the products read held in 8
bits (ROW8).

Against the same chain of public operators, each of which is tested for itself
(test_gpu_row8.py and the attention's tests): the launches are the same, so the residual
stream has the same bits and the logits only the final norm's and classifier's rounding
between them.  (A model over rows held in 8 bits is no smooth function of its inputs: a
relative difference of 1e-6 moves a few codes to their neighbours, and one such code a
logit by as much as holding all rows does.  A reference with sums in another order says
little about it.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOGIT_ATOL, LOGIT_RTOL = 2e-3, 1e-3
CHUNK_AS_DECODE = 32  # rows up to which a scheduler's chunk rides in the decode batch

MODELS = {
    # name: (dim, hidden, layers, heads, kv heads, vocab, seq_len); widths of whole column tiles, so
    # that wq, wk and wv in one matrix are the same launch as the model's group of three
    "mha_hd64_l3": (256, 512, 3, 4, 4, 1000, 256),
    "gqa_hd128_l2": (512, 1024, 2, 4, 2, 700, 200),
    "gqa_hd96_l2": (768, 544, 2, 8, 4, 400, 160),
}


class Chain:
    """A model's forward from public operators, over a pool."""

    def __init__(self, blob, pool):
        import torch

        import nitrorag_amd as na
        from oracle import model as om

        self.m, self.pool, self.na = om.OracleModel(blob), pool, na
        m = self.m

        def dev(a):
            return torch.from_numpy(np.array(a, copy=True)).cuda()

        def blocks(w, n):
            return w.reshape(-1, n // 32, 36)

        self.layers = []
        for l in range(m.n_layers):
            qkv = np.concatenate([blocks(w[l], m.dim) for w in (m.wq, m.wk, m.wv)])
            self.layers.append((dev(m.rms_att[l]), na.Q8Weights(dev(qkv)), na.Q8Weights(dev(blocks(m.wo[l], m.dim))),
                                dev(m.rms_ffn[l]), na.Q8Weights(dev(blocks(m.w1[l], m.dim)), dev(blocks(m.w3[l], m.dim))),
                                na.Q8Weights(dev(blocks(m.w2[l], m.hidden)))))
        self.emb, self.freq = dev(m.emb), (dev(m.freq_real), dev(m.freq_imag))

    def run(self, tokens, prefill):
        """The residual stream after the layers; rows [0, prefill) are the pool's prefill
        batch, the others its decode batch."""
        import torch

        m, na, pool, rows = self.m, self.na, self.pool, len(tokens)
        shape = (m.n_heads, m.n_kv_heads, m.head_size)
        x = self.emb[torch.from_numpy(np.asarray(tokens, np.int64)).cuda()].contiguous()
        scales = torch.empty(rows, device="cuda")
        c, hc = (torch.empty((rows, n), dtype=torch.int8, device="cuda") for n in (m.dim, m.hidden))
        out, hb = (torch.empty((rows, n), device="cuda") for n in (m.dim + 2 * m.kv_dim, m.hidden))
        for l, (att, wqkv, wo, ffn, w13, w2) in enumerate(self.layers):
            na.rms_norm_row8(x, att, c, scales)
            wqkv.matmul(c, scales, out)
            q, k, v = (t.contiguous() for t in out.split([m.dim, m.kv_dim, m.kv_dim], 1))
            got = torch.empty_like(q)
            if prefill:
                pool.rope_kv_append_prefill(l, q[:prefill], k[:prefill], v[:prefill], *self.freq, *shape)
            if prefill < rows:
                pool.rope_kv_append(l, q[prefill:], k[prefill:], v[prefill:], *self.freq, *shape)
            if prefill:
                pool.prefill(l, q[:prefill], got[:prefill], *shape)
            if prefill < rows:
                pool.decode(l, q[prefill:], got[prefill:], *shape)
            na.row8_quantize(got, c, scales)
            wo.matmul(c, scales, x, residual=x)
            na.rms_norm_row8(x, ffn, c, scales)
            w13.matmul(c, scales, hb, activation="silu")
            na.row8_quantize(hb, hc, scales)
            w2.matmul(hc, scales, x, residual=x)
        return x.cpu().numpy()

    def logits(self, x):
        x, w = x.astype(np.float64), self.m.emb.astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * self.m.rms_final.astype(np.float64)
        return x @ w.T


def check(got, want, what):
    off = np.abs(got - want) - LOGIT_RTOL * np.abs(want) - LOGIT_ATOL
    assert got.shape == want.shape and off.max() <= 0, (what, off.max())


def model_of(name, seed):
    from nitrorag_amd.model import synthetic_model_file
    from oracle import model as om

    dim, hid, L, H, G, V, S = MODELS[name]
    return om.scale_residual_outputs(synthetic_model_file(dim, hid, L, H, G, V, S, seed=seed), 8.0)


def pool_of(name, pages, pool8):
    import torch

    import nitrorag_amd as na

    dim, hid, L, H, G, V, S = MODELS[name]
    if pool8:
        return na.KVPool.create_q8(pages, L, G, dim // H)
    k = torch.zeros((pages, L, 16, G * dim // H), device="cuda")
    return na.KVPool.wrap(k, torch.zeros_like(k))


@pytest.mark.parametrize("pool8", [False, True])
@pytest.mark.parametrize("name", sorted(MODELS))
def test_forwards(name, pool8):
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.model import ROW8

    dim, hid, L, H, G, V, S = MODELS[name]
    blob = model_of(name, len(name))
    model, pool = na.Model(blob), pool_of(name, 96, pool8)
    chain = Chain(blob, pool_of(name, 96, pool8))
    bm = na.BlockManager(96)
    rng = np.random.default_rng(21)
    seqs = [na.Sequence(i) for i in range(20)]
    for group in ([0], [1], range(2, 9), range(9, 20)):
        lens = [70 if i == 0 else int(rng.integers(1, 30)) for i in group]
        toks = rng.integers(0, V, sum(lens)).astype(np.int32)
        at = 0
        for i, n in zip(group, lens):
            for t in toks[at:at + n]:
                seqs[i].allocate_next_token(int(t), bm)
            at += n
        tables = na.pack_block_tables([seqs[i] for i in group])
        for p in (pool, chain.pool):
            p.upload_prefill_batch(tables, [0] * len(lens), lens)
        got = model.forward_prefill(pool, toks, semantics=ROW8).cpu().numpy()
        check(got, chain.logits(chain.run(toks, len(toks))[np.cumsum(lens) - 1]), f"prefill {lens}")
    for nb in (20, 3, 1, 17):
        toks = rng.integers(0, V, nb).astype(np.int32)
        pos = [s.logical_token_count for s in seqs[:nb]]
        for s, t in zip(seqs, toks):
            s.allocate_next_token(int(t), bm)
        for p in (pool, chain.pool):
            p.upload_decode_batch(na.pack_block_tables(seqs[:nb]), pos)
        got = model.forward_decode_batch(pool, toks, semantics=ROW8).cpu().numpy()
        check(got, chain.logits(chain.run(toks, 0)), f"decode {nb}")
    torch.cuda.synchronize()
    assert pool.take_device_errors() == 0


def test_semantics_side_by_side():
    """Forwards of the three semantics in any order give what each gives alone."""
    import nitrorag_amd as na
    from nitrorag_amd.model import FULL_ROWS, LAST_BLOCK, ROW8

    name = "gqa_hd128_l2"
    blob, V = model_of(name, 5), MODELS[name][5]
    rng = np.random.default_rng(0)
    tokens = rng.integers(0, V, 60).astype(np.int32)
    table = np.arange(4, dtype=np.int32)[None]

    def forward(model, semantics, n):
        pool = pool_of(name, 4, False)
        pool.upload_prefill_batch(table, [0], [n])
        return model.forward_prefill(pool, tokens[:n], semantics=semantics).cpu().numpy()

    alone = {(s, n): forward(na.Model(blob), s, n) for s in (FULL_ROWS, LAST_BLOCK, ROW8) for n in (3, 20, 60)}
    model = na.Model(blob)
    for s, n in ((ROW8, 3), (FULL_ROWS, 20), (ROW8, 20), (LAST_BLOCK, 60), (ROW8, 60), (FULL_ROWS, 60), (FULL_ROWS, 3), (ROW8, 3), (LAST_BLOCK, 3)):
        np.testing.assert_array_equal(forward(model, s, n), alone[s, n], f"{s} {n}")


def test_captured_decode():
    """A captured decode step, replayed over new positions, gives the eager step's logits."""
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.model import ROW8

    name = "mha_hd64_l3"
    blob, V = model_of(name, 6), MODELS[name][5]
    rng = np.random.default_rng(1)
    tables = np.arange(20, dtype=np.int32).reshape(4, 5)
    tokens = rng.integers(0, V, 4).astype(np.int32)
    outs = []
    for captured in (False, True):
        model, pool = na.Model(blob), pool_of(name, 20, False)
        pool.upload_prefill_batch(tables, [0] * 4, [9] * 4)
        model.forward_prefill(pool, np.tile(tokens, 9), semantics=ROW8)
        logits, got, graph = torch.empty((4, V), device="cuda"), [], None
        for step in range(4):
            pool.upload_decode_batch(tables, [9 + step] * 4)
            if captured and step == 1:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    model.forward_decode_batch(pool, tokens, logits, ROW8)
            if graph:
                graph.replay()
            else:
                model.forward_decode_batch(pool, tokens, logits, ROW8)
            torch.cuda.synchronize()
            got.append(logits.cpu().numpy())
        outs.append(got)
        assert pool.take_device_errors() == 0
    for step, (a, b) in enumerate(zip(*outs)):
        np.testing.assert_array_equal(a, b, f"step {step}")


def tables_of(words):
    """{request id: block table} from a scheduler's state words."""
    at, tables = 0, {}

    def vector():
        nonlocal at
        n = words[at]
        at += 1 + n
        return words[at - n:at]

    vector(), vector()
    n, at = words[at], at + 1
    for _ in range(n):
        rid = words[at]
        at += 5
        vector()
        at += 3
        vector()
        tables[rid] = vector()
    return tables


@pytest.mark.parametrize("pool8", [False, True])
def test_scheduler(pool8):
    """Steps of long and short chunks (the latter's rows ride in the decode batch) with decode
    rows, beside the same steps planned, run through the chain and committed."""
    import nitrorag_amd as na
    from nitrorag_amd.model import ROW8

    name = "gqa_hd128_l2"
    blob, V = model_of(name, 3), MODELS[name][5]
    model, pool, chain = na.Model(blob), pool_of(name, 64, pool8), Chain(blob, pool_of(name, 64, pool8))
    scheds = [na.ContinuousScheduler(na.BlockManager(64), 96, 6) for _ in range(2)]
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, V, n).tolist() for n in (120, 20, 45)]
    prompts.append(prompts[0][:64] + [5, 6, 7])  # shares cached pages
    for s in scheds:
        for i, p in enumerate(prompts):
            s.add_request(i, p)
    kinds = set()
    while scheds[0].has_active_requests():
        scheds[0].step(model, pool, ROW8)
        got = scheds[0].last_logits()
        plan = scheds[1].plan()
        rid, start, P, finishes = plan.prefill_id, plan.prefill_start, plan.prefill_length, plan.prefill_finishes
        ids, tokens, positions = plan.decode_ids, plan.decode_tokens, plan.decode_positions
        tables = tables_of(scheds[1].state_words())
        rows = ([prompts[rid][start + i] for i in range(P)] if P else []) + list(tokens)
        as_decode = P <= CHUNK_AS_DECODE
        batch = ([(tables[rid], start + i) for i in range(P)] if as_decode else []) + [(tables[i], p) for i, p in zip(ids, positions)]
        if batch:
            wide = max(p // 16 + 1 for _, p in batch)
            packed = np.zeros((len(batch), wide), np.int32)
            for r, (t, p) in enumerate(batch):
                packed[r, :p // 16 + 1] = t[:p // 16 + 1]
            chain.pool.upload_decode_batch(packed, [p for _, p in batch])
        if P and not as_decode:
            chain.pool.upload_prefill_batch(np.array([tables[rid]], np.int32), [start], [P])
        kinds.add((P > 0, as_decode, len(tokens) > 0))
        want = np.zeros((0, V))
        if rows:
            x = chain.run(rows, 0 if as_decode else P)
            want = chain.logits(x[P - 1 if finishes else P:])
        if len(want):
            check(got, want, plan)
        chosen = [int(r.argmax()) if r.max() > 0 else 0 for r in got]
        scheds[1].commit(chosen[0] if finishes else 0, chosen[1:] if finishes else chosen)
    assert [scheds[0].generated(i) for i in range(4)] == [scheds[1].generated(i) for i in range(4)]
    assert {(True, False, False), (True, True, True), (False, True, True)} <= kinds, kinds
    assert pool.take_device_errors() == 0


def test_row8_of_other_entry_points():
    """A server takes ROW8; the product alone does not, and no entry takes a fourth semantics."""
    import ctypes

    import torch

    import nitrorag_amd as na
    from nitrorag_amd import _native as N
    from nitrorag_amd.model import ROW8

    name = "mha_hd64_l3"
    model, pool = na.Model(model_of(name, 2)), pool_of(name, 8, False)
    sched = na.ContinuousScheduler(na.BlockManager(8), 32, 4)
    server = ctypes.c_void_p()
    N.call("nitro_server_create", sched._h, model.handle, pool.handle, ROW8, 64, ctypes.byref(server))
    N.call("nitro_server_destroy", server)
    with pytest.raises(na.NitroError):
        N.call("nitro_server_create", sched._h, model.handle, pool.handle, 3, 64, ctypes.byref(server))
    pool.upload_decode_batch([[0]], [0])
    with pytest.raises(na.NitroError):
        model.forward_decode_batch(pool, [1], semantics=3)
    pool.upload_prefill_batch([[0]], [0], [2])
    with pytest.raises(na.NitroError):
        model.forward_prefill(pool, [1, 2], semantics=3)
    sched.add_request(0, [1, 2, 3])
    with pytest.raises(na.NitroError):
        sched.step(model, pool, 3)
    w = torch.zeros(8 * 36, dtype=torch.uint8, device="cuda")
    with pytest.raises(na.NitroError):
        na.q8_matmul(w, torch.zeros((1, 32), device="cuda"), torch.zeros((1, 8), device="cuda"), ROW8)
