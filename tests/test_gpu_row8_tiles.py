"""Products of 8-bit rows through every kernel they can take (row8_tiles.py), whole outputs
against 64 bits; a matrix past 4 GiB; wq, wk and wv in one launch through each kernel."""
import numpy as np
import pytest

import row8_forms as forms
from gpu_helpers import to_gpu
from row8_tiles import CASES, GROUPS
from test_gpu_row8_model import Chain, check as check_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    yield
    torch.cuda.synchronize()


def sums(q, s, codes, scales):
    """(p, bound) of forms.product before the epilogue, in 64 bits on the GPU: a block's sum is
    exact, an fma for each block and the joins of up to 16 waves round by half a step of at
    most sum_j |ws_j * block_j|, the row's scale once."""
    import torch

    xs = scales.double()[:, None]
    p = torch.zeros((len(codes), len(q)), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(p)
    for j in range(q.shape[1]):
        block = codes[:, 32 * j:32 * j + 32].double().contiguous() @ q[:, j].double().t().contiguous()
        block *= s[:, j].double()
        p += block
        mag += block.abs_()
    return p * xs, mag * xs * forms.EPS32 * (q.shape[1] + 16 + 1)


def product(mats, codes, scales, bias, residual, activation):
    """forms.product of one matrix with relu and of a pair with silu, on the GPU (its
    derivation of the bound holds here)."""
    import torch

    parts = []
    for i, (q, s) in enumerate(mats):
        p, e = sums(q, s, codes, scales)
        p += bias.double()[i * len(q):(i + 1) * len(q)]
        parts.append((p, e + forms.EPS32 * (p.abs() + e)))
    p, e = parts[0]
    e = e * 1.13
    if activation == "relu":
        y = p.clamp(min=0.0)
    else:
        y = p / (1 + torch.exp(-p))
        e = e + 16 * forms.EPS32 * (1 + p.abs()) * y.abs() + 1e-35
    if len(parts) > 1:
        up, e_up = parts[1]
        e = e * (up.abs() + e_up) + e_up * y.abs() + forms.EPS32 * (y * up).abs()
        y = y * up
    y = y + residual.double()
    e = e + forms.EPS32 * (y.abs() + e)
    return y, e + forms.EPS32 * y.abs()


def held_rows(rng, rows, n):
    """Codes and scales of normal rows, held by the operator that test_gpu_row8.py tests."""
    import torch

    import nitrorag_amd as na

    codes, scales = torch.empty((rows, n), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    na.row8_quantize(to_gpu(rng.standard_normal((rows, n)).astype(np.float32)), codes, scales)
    return codes, scales


def test_the_64_bit_form():
    """On the GPU it is the numpy form."""
    rng = np.random.default_rng(0)
    codes, scales = held_rows(rng, 9, 160)
    for gated, activation in ((False, "relu"), (True, "silu")):
        mats = [forms.matrix(rng, 37, 160)[1:] for _ in range(1 + gated)]
        bias, residual = rng.standard_normal(37 * len(mats)).astype(np.float32), rng.standard_normal((9, 37)).astype(np.float32)
        got = product([(to_gpu(q), to_gpu(s)) for q, s in mats], codes, scales, to_gpu(bias), to_gpu(residual), activation)
        want = forms.product(mats, codes.cpu().numpy(), scales.cpu().numpy(), bias, residual, activation)
        for g, w in zip(got, want):
            np.testing.assert_allclose(g.cpu().numpy(), w, rtol=1e-9, atol=1e-14)


@pytest.mark.parametrize("gated,tile,rows,n,d", [(*key, *shape) for key in sorted(CASES) for shape in CASES[key]])
def test_every_kernel(gated, tile, rows, n, d):
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.row8 import product_tile

    assert product_tile(rows, n, d, gated=gated) == tile
    rng = np.random.default_rng(rows + n + d)
    codes, scales = held_rows(rng, rows, n)
    mats = [forms.matrix(rng, d, n) for _ in range(1 + gated)]
    bias = to_gpu(rng.standard_normal(d * len(mats)).astype(np.float32))
    residual = to_gpu(rng.standard_normal((rows, d)).astype(np.float32))
    buf = torch.full(((rows + 1) * d,), 5.0, device="cuda")
    out = buf[:rows * d].view(rows, d)
    activation = "silu" if gated else "relu"
    na.Q8Weights(*(to_gpu(m[0]) for m in mats)).matmul(codes, scales, out, bias=bias, residual=residual, activation=activation)
    torch.cuda.synchronize()
    want, bound = product([(to_gpu(q), to_gpu(s)) for _, q, s in mats], codes, scales, bias, residual, activation)
    over = (out.double() - want).abs() - bound
    worst = np.unravel_index(over.argmax().item(), over.shape)
    assert over[worst].item() <= 0, (worst, out[worst].item(), want[worst].item(), bound[worst].item())
    assert torch.isfinite(out).all() and (buf[rows * d:] == 5).all()


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_matrix_past_4_gib(gated, rows):
    """A matrix whose blocks, and their copy, pass 2^32 bytes: columns of all of it."""
    import torch

    import nitrorag_amd as na

    n, d = 65536, 60017
    gen = torch.Generator(device="cuda").manual_seed(rows)
    w = torch.randint(0, 256, (d, n // 32, 36), dtype=torch.uint8, device="cuda", generator=gen)
    w[..., :4] = torch.tensor([1 / (127 * 256.0)], device="cuda").view(torch.uint8)
    assert w.numel() > 1 << 32
    weights = na.Q8Weights(w, w) if gated else na.Q8Weights(w)
    codes, scales = held_rows(np.random.default_rng(rows), rows, n)
    out = torch.full((rows, d), float("nan"), device="cuda")
    weights.matmul(codes, scales, out)
    cols = torch.cat([torch.arange(0, d, 1009), torch.arange(d - 40, d)]).cuda()
    some = torch.stack([w[c] for c in cols.tolist()])
    q, s = some[..., 4:].contiguous().view(torch.int8), some[..., :4].contiguous().view(torch.float32)[..., 0]
    p, bound = sums(q, s, codes, scales)
    if gated:  # p * p, each factor off by the bound
        bound = 2 * p.abs() * bound + bound * bound + forms.EPS32 * p * p
        p = p * p
    bound = bound + 2 * forms.EPS32 * p.abs()
    assert ((out[:, cols].double() - p).abs() <= bound).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("rows,dim,kv,heads,kv_heads", [shape for tile in sorted(GROUPS) for shape in GROUPS[tile]])
def test_wq_wk_wv_in_one_launch(rows, dim, kv, heads, kv_heads):
    """A layer's prompt.  Its K and V lie in the pool as their products left them (the rotation
    is by no angle): each against 64 bits over the rows that the norm holds.  Q by what follows
    it, against the chain over wq, wk and wv as one matrix, which sums in the same order."""
    import torch

    import nitrorag_amd as na
    from nitrorag_amd.model import ROW8, synthetic_model_file
    from oracle.model import scale_residual_outputs

    seq_len, vocab, head = 128, max(rows, 64), dim // heads
    blob = scale_residual_outputs(synthetic_model_file(dim, 64, 1, heads, kv_heads, vocab, seq_len, seed=rows), 8.0)
    blob = np.frombuffer(bytes(blob), np.uint8).copy()
    freq = blob[-4 * seq_len * head:].view(np.float32)  # cosines, then sines
    freq[:freq.size // 2], freq[freq.size // 2:] = 1, 0
    lens = [min(100, rows - at) for at in range(0, rows, 100)]
    tables = (np.arange(7 * len(lens), dtype=np.int32)[::-1].copy()).reshape(-1, 7)
    shape = (7 * len(lens), 1, 16, kv)
    caches = [[torch.full(shape, 7.0, device="cuda") for _ in range(2)] for _ in range(2)]
    pools = [na.KVPool.wrap(*c) for c in caches]
    for p in pools:
        p.upload_prefill_batch(tables, [0] * len(lens), lens)
    rng = np.random.default_rng(rows)
    tokens = rng.permutation(vocab)[:rows].astype(np.int32)
    chain = Chain(blob, pools[1])
    got = na.Model(blob).forward_prefill(pools[0], tokens, semantics=ROW8).cpu().numpy()
    check_logits(got, chain.logits(chain.run(tokens, rows)[np.cumsum(lens) - 1]), "logits")

    m = chain.m
    codes, scales = torch.empty((rows, dim), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    na.rms_norm_row8(to_gpu(m.emb[tokens]), to_gpu(m.rms_att[0]), codes, scales)
    at = np.concatenate([np.arange(n) for n in lens])
    seq = np.repeat(np.arange(len(lens)), lens)
    page, slot = tables[seq, at // 16], at % 16
    for w, held, other in zip((m.wk[0], m.wv[0]), *caches):
        w = np.frombuffer(bytes(w), np.uint8).reshape(kv, dim // 32, 36)
        q, s = w[..., 4:].copy().view(np.int8), w[..., :4].copy().view(np.float32)[..., 0]
        p, bound = sums(to_gpu(q), to_gpu(s), codes, scales)
        rows_held = held[to_gpu(page).long(), 0, to_gpu(slot).long()]
        assert ((rows_held.double() - p).abs() <= bound + forms.EPS32 * p.abs()).all()
        assert torch.equal(held, other)  # the bits of the chain's, and nothing else written
