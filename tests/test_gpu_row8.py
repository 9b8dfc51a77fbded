"""Rows held in 8 bits on the GPU: the norm, quantising and reading back bit for bit
against their definition, products within what fp32 sums may leave of the 64-bit result."""
import numpy as np
import pytest

import row8_forms as forms
from gpu_helpers import to_gpu

pytestmark = pytest.mark.gpu

# one group of four or less, the borders of the kernels' widths, odd ones, past all registers
WIDTHS = [1, 3, 4, 31, 64, 255, 256, 257, 768, 1024, 1025, 2049, 4096, 4099, 5003, 8192, 8195, 11008, 16385, 32768, 32769, 40001, 65536, 65539]


@pytest.fixture(scope="module", autouse=True)
def gpu():
    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import nitrorag_amd  # noqa: F401
    yield
    torch.cuda.synchronize()


def held_on_gpu(call, rows, n, offset=0):
    """codes and scales that call(codes, scales) writes, with untouched bytes around them."""
    import torch

    codes = torch.full((rows * n + 64,), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((rows + 2,), 55.0, device="cuda")
    call(codes[16 + offset:16 + offset + rows * n].view(rows, n), scales[1:1 + rows])
    torch.cuda.synchronize()
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    assert (c[:16 + offset] == 77).all() and (c[16 + offset + rows * n:] == 77).all() and s[0] == 55 and s[-1] == 55
    return c[16 + offset:16 + offset + rows * n].reshape(rows, n), s[1:-1]


def rows_of(rng, rows, n):
    return (rng.standard_normal((rows, n)) * np.exp(rng.uniform(-8, 8, (rows, 1)))).astype(np.float32)


def same(got, want, what):
    codes, scales = want
    np.testing.assert_array_equal(got[1], scales, what)
    np.testing.assert_array_equal(got[0], codes, what)


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5])
def test_quantize_and_read(rows, n):
    import torch

    import nitrorag_amd as na

    x = rows_of(np.random.default_rng(n + rows), rows, n)
    got = held_on_gpu(lambda c, s: na.row8_quantize(to_gpu(x), c, s), rows, n)
    same(got, forms.hold(x), f"{rows} x {n}")
    back = torch.full((rows * n + 2,), 9.0, device="cuda")
    na.row8_read(to_gpu(got[0]), to_gpu(got[1]), back[1:-1].view(rows, n))
    back = back.cpu().numpy()
    assert back[0] == 9 and back[-1] == 9
    np.testing.assert_array_equal(back[1:-1].reshape(rows, n), got[0].astype(np.float32) * got[1][:, None])


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("form", ["plain", "residual", "sum", "sum over x", "sum over residual"])
def test_rms_norm(form, n):
    import nitrorag_amd as na

    rng = np.random.default_rng(n)
    rows = 3 if n > 3000 else 300 if n == 1025 else 7
    x, res = rows_of(rng, rows, n), rows_of(rng, rows, n) if form != "plain" else None
    weight = rng.uniform(-1.5, 1.5, n).astype(np.float32)
    dx, dres = to_gpu(x), None if res is None else to_gpu(res)
    total = {"sum": to_gpu(np.full_like(x, 3)), "sum over x": dx, "sum over residual": dres}.get(form)
    got = held_on_gpu(lambda c, s: na.rms_norm_row8(dx, to_gpu(weight), c, s, residual=dres, sum=total), rows, n)
    h, y = forms.normed(x, weight, res)
    same(got, forms.hold(y), f"{form} {n}")
    if total is not None:
        np.testing.assert_array_equal(total.cpu().numpy(), h)


def test_rows_of_many():
    """More rows than a launch's first workgroups, and 16-wave workgroups' other form."""
    import nitrorag_amd as na

    rng = np.random.default_rng(5)
    for rows, n in ((3001, 768), (1000, 1500), (300, 6000), (257, 4096)):
        x, weight = rows_of(rng, rows, n), rng.uniform(0.5, 1.5, n).astype(np.float32)
        got = held_on_gpu(lambda c, s: na.rms_norm_row8(to_gpu(x), to_gpu(weight), c, s), rows, n)
        same(got, forms.hold(forms.normed(x, weight)[1]), f"{rows} x {n}")


@pytest.mark.parametrize("n,offset", [(768, 1), (4096, 3), (5003, 2), (70000, 1)])
def test_rows_that_begin_anywhere(n, offset):
    """x, weight and codes that start at odd elements."""
    import torch

    import nitrorag_amd as na

    rng = np.random.default_rng(n)
    x, weight = rows_of(rng, 4, n), rng.uniform(0.5, 1.5, n).astype(np.float32)
    dx = torch.zeros(4 * n + offset, device="cuda")
    dw = torch.zeros(n + offset, device="cuda")
    dx[offset:], dw[offset:] = to_gpu(x).flatten(), to_gpu(weight)
    got = held_on_gpu(lambda c, s: na.rms_norm_row8(dx[offset:].view(4, n), dw[offset:], c, s), 4, n, offset)
    same(got, forms.hold(forms.normed(x, weight)[1]), f"{n} + {offset}")


@pytest.mark.parametrize("n", [5, 768, 4099, 65539])
def test_rows_without_numbers(n):
    """Zero rows, rows below 2^-100, rows with an infinity or a NaN: the others are as without them."""
    import nitrorag_amd as na

    x = rows_of(np.random.default_rng(n), 8, n)
    x[1] = 0
    x[2] = 1e-31
    x[3] *= 0
    x[3, n - 1] = 2.0 ** -100
    x[4, n // 2] = np.inf
    x[5, 0] = -np.inf
    x[6, n - 1] = np.nan
    got = held_on_gpu(lambda c, s: na.row8_quantize(to_gpu(x), c, s), 8, n)
    same(got, forms.hold(x), f"{n}")
    assert got[1][1] == 0 and got[1][2] == 0 and got[1][3] > 0 and np.isnan(got[1][4:7]).all()
    weight = np.ones(n, np.float32)
    got = held_on_gpu(lambda c, s: na.rms_norm_row8(to_gpu(x), to_gpu(weight), c, s), 8, n)
    same(got, forms.hold(forms.normed(x, weight)[1]), f"{n} normed")
    assert np.isnan(got[1][4:7]).all() and np.isfinite(got[1][[0, 1, 2, 3, 7]]).all()


def test_norm_of_large_and_small_rows():
    """Squares past fp32's range, a sum that overflows, a large eps."""
    import nitrorag_amd as na

    n = 1000
    x = rows_of(np.random.default_rng(1), 4, n)
    x[0] *= np.float32(1e30) / np.abs(x[0]).max()
    x[1] *= np.float32(1e-30) / np.abs(x[1]).max()
    x[2, 7] = 3e38
    res = np.zeros_like(x)
    res[2, 7] = 3e38
    weight = np.full(n, 2.0, np.float32)
    for eps in (1e-5, 1e-30, 3.0):
        got = held_on_gpu(lambda c, s: na.rms_norm_row8(to_gpu(x), to_gpu(weight), c, s, residual=to_gpu(res), eps=eps), 4, n)
        with np.errstate(over="ignore"):
            same(got, forms.hold(forms.normed(x, weight, res, eps)[1]), f"eps {eps}")
        assert np.isnan(got[1][2]) and np.isfinite(got[1][[0, 1, 3]]).all()


# ------------------------------------------------------------------ products

SHAPES = [
    # rows, n, d: one block and one output, odd block counts, rows about the 16- and 64-row
    # tiles, outputs that fill no tile, many tiles
    (1, 32, 1), (1, 4096, 1003), (3, 96, 17), (15, 768, 64), (16, 2048, 768), (17, 1056, 100), (33, 32, 33),
    (64, 11008, 40), (65, 64, 16), (77, 1056, 1003), (128, 96, 128), (129, 160, 129), (300, 768, 515), (257, 32, 65),
    (1030, 96, 4100), (700, 416, 6100), (2051, 32, 2080)]


def check(out, want, what):
    y, bound = want
    assert out.shape == y.shape
    assert np.isfinite(out).all(), what
    over = np.abs(out.astype(np.float64) - y) - bound
    worst = np.unravel_index(over.argmax(), over.shape)
    assert over[worst] <= 0, f"{what}: {out[worst]} for {y[worst]} at {worst}, allowed {bound[worst]}"


def product_case(seed, rows, n, d, gated=False):
    rng = np.random.default_rng(seed)
    codes, scales = forms.hold(rng.standard_normal((rows, n)).astype(np.float32))
    mats = [forms.matrix(rng, d, n) for _ in range(2 if gated else 1)]
    bias = rng.standard_normal(d * len(mats)).astype(np.float32)
    residual = (3 * rng.standard_normal((rows, d))).astype(np.float32)
    return codes, scales, mats, bias, residual


def on_gpu(mats, codes, scales, **kw):
    import torch

    import nitrorag_amd as na

    weights = na.Q8Weights(*(to_gpu(m[0]) for m in mats))
    assert weights.d == mats[0][0].shape[0] and weights.n == codes.shape[1]
    out = torch.full((len(codes), weights.d), float("nan"), device="cuda")
    kw = {k: to_gpu(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    weights.matmul(to_gpu(codes), to_gpu(scales), out, **kw)
    torch.cuda.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("rows,n,d", SHAPES)
def test_product(rows, n, d):
    codes, scales, mats, bias, residual = product_case(rows + n + d, rows, n, d)
    forms_of = [(q, s) for _, q, s in mats]
    check(on_gpu(mats, codes, scales), forms.product(forms_of, codes, scales), "product")
    check(on_gpu(mats, codes, scales, bias=bias, residual=residual, activation="relu"),
          forms.product(forms_of, codes, scales, bias, residual, "relu"), "bias, relu, residual")


@pytest.mark.parametrize("rows,n,d", SHAPES)
def test_gated_product(rows, n, d):
    codes, scales, mats, bias, residual = product_case(rows * 3 + n + d, rows, n, d, gated=True)
    forms_of = [(q, s) for _, q, s in mats]
    check(on_gpu(mats, codes, scales, activation="silu"), forms.product(forms_of, codes, scales, activation="silu"), "gated")
    check(on_gpu(mats, codes, scales, bias=bias, residual=residual, activation="gelu"),
          forms.product(forms_of, codes, scales, bias, residual, "gelu"), "gated with bias and residual")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows,d", [(2, 50), (40, 70), (150, 200), (1100, 4000)])
def test_activations(rows, d, activation, gated):
    codes, scales, mats, bias, _ = product_case(rows, rows, 64, d, gated)
    bias[::7] *= 2.5
    check(on_gpu(mats, codes, scales, bias=bias, activation=activation),
          forms.product([(q, s) for _, q, s in mats], codes, scales, bias, None, activation), activation)


@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [1, 40, 1100])
def test_activations_of_any_number(rows, activation):
    """Rows of zeros leave the bias alone in front of the activation."""
    row = np.array([0, 1e-38, 1e-30, 1e-4, 1, 5, 9, 13, 20, 60, 88, 89, 100, 104, 200, 1e4, 1e10, 1e19, 1e20, 1e30, 3e38, np.inf], np.float32)
    bias = np.tile(np.concatenate([row, -row, [np.nan]]).astype(np.float32), 90 if rows > 1000 else 2)
    w, q, s = forms.matrix(np.random.default_rng(rows), len(bias), 64)
    codes, scales = np.zeros((rows, 64), np.int8), np.zeros(rows, np.float32)
    got = on_gpu([(w, q, s)], codes, scales, bias=bias, activation=activation)
    with np.errstate(all="ignore"):
        want, bound = forms.product([(q, s)], codes[:1], scales[:1], bias, None, activation)
        finite = np.isfinite(want[0])
        over = np.abs(got[:, finite] - want[0, finite]) > bound[0, finite]
    assert not over.any(), (got[:, finite][over][:4], np.broadcast_to(bias[finite], over.shape)[over][:4])
    if activation != "relu":  # from 20 on exp(-p) is nothing next to 1: the roundings alone
        large = finite & (bias >= 20)
        assert (np.abs(got[:, large] - bias[large].astype(np.float64)) <= 16 * forms.EPS32 * bias[large].astype(np.float64)).all()
    np.testing.assert_array_equal(got[:, ~finite], np.broadcast_to(want[0, ~finite], (rows, (~finite).sum())))


@pytest.mark.parametrize("rows", [1, 20, 100, 1100])
def test_residual_in_place_and_rows_behind(rows):
    import torch

    import nitrorag_amd as na

    d = 4001
    codes, scales, mats, bias, residual = product_case(rows, rows, 128, d)
    buf = torch.full(((rows + 1) * d,), 5.0, device="cuda")
    out = buf[:rows * d].view(rows, d)
    out.copy_(to_gpu(residual))
    na.Q8Weights(to_gpu(mats[0][0])).matmul(to_gpu(codes), to_gpu(scales), out, residual=out)
    check(out.cpu().numpy(), forms.product([mats[0][1:]], codes, scales, None, residual), "in place")
    assert (buf[rows * d:] == 5).all()


@pytest.mark.parametrize("rows", [4, 40, 200, 1100])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_without_numbers_stay_alone(rows, gated):
    """A row whose scale is NaN gives NaN, a zero row the bias; other rows keep their bits."""
    import torch

    d = 4000 if rows > 1000 else 300
    codes, scales, mats, bias, _ = product_case(rows, rows, 96, d, gated)
    whole = on_gpu(mats, codes, scales, bias=bias, activation="silu")
    codes[1], scales[1] = 0, np.nan
    codes[2], scales[2] = 0, 0
    got = on_gpu(mats, codes, scales, bias=bias, activation="silu")
    assert np.isnan(got[1]).all()
    keep = [r for r in range(rows) if r not in (1, 2)]
    np.testing.assert_array_equal(got[keep], whole[keep])
    want, bound = forms.product([(q, s) for _, q, s in mats], codes[2:3], scales[2:3], bias, None, "silu")
    assert (np.abs(got[2] - want[0]) <= bound[0]).all()
    assert not torch.isnan(to_gpu(got[keep])).any()


def test_extreme_codes():
    """Every code at its limit: the largest sums a block can have (-128 in the weights too)."""
    for rows in (1, 50, 200):
        n, d = 352, 48
        rng = np.random.default_rng(rows)
        codes = np.where(rng.random((rows, n)) < 0.5, 127, -127).astype(np.int8)
        codes[0] = 127
        scales = np.full(rows, 1 / 127, np.float32)
        w, q, s = forms.matrix(rng, d, n)
        q[:] = np.where(rng.random(q.shape) < 0.5, 127, -128)
        q[0] = -128
        w[..., 4:] = q.view(np.uint8)
        check(on_gpu([(w, q, s)], codes, scales), forms.product([(q, s)], codes, scales), f"{rows} rows")


@pytest.mark.parametrize("rows", [1, 24, 90, 1100])
def test_same_bits_every_time(rows):
    codes, scales, mats, bias, residual = product_case(rows, rows, 1024, 4000 if rows > 1000 else 500, True)
    kw = dict(bias=bias, residual=residual, activation="gelu_tanh")
    first = on_gpu(mats, codes, scales, **kw)
    for _ in range(3):
        np.testing.assert_array_equal(on_gpu(mats, codes, scales, **kw), first)


def test_matrix_past_4_gib_of_codes():
    """Rows and weights whose bytes pass 2^31 and 2^32."""
    import torch

    import nitrorag_amd as na

    n, rows = 65536, 66000
    codes = torch.zeros((rows, n), dtype=torch.int8, device="cuda")
    scales = torch.ones(rows, device="cuda")
    last = torch.randint(-127, 128, (n,), device="cuda", dtype=torch.int8)
    codes[-1], codes[40000] = last, last
    w, q, s = forms.matrix(np.random.default_rng(0), 16, n)
    out = torch.empty((rows, 16), device="cuda")
    na.Q8Weights(to_gpu(w)).matmul(codes, scales, out)
    want, bound = forms.product([(q, s)], last.cpu().numpy()[None], np.ones(1))
    for r in (rows - 1, 40000):
        assert (np.abs(out[r].cpu().numpy() - want[0]) <= bound[0]).all()
    assert (out[:40000] == 0).all() and (out[40001:-1] == 0).all()
    del codes
    x = torch.empty((rows, n), device="cuda")
    x.zero_()[-1] = last.float()
    held = torch.empty((rows, n), dtype=torch.int8, device="cuda")
    na.row8_quantize(x, held, scales)
    top = last.abs().max().item()
    assert scales[-1].item() == np.float32(top) / np.float32(127) and (scales[:-1] == 0).all()
    na.row8_read(held, scales, x)
    assert (x[-1] - last.float()).abs().max().item() <= 0.5001 * top / 127 and (x[0] == 0).all()


def test_more_rows_than_a_launch_takes():
    """Rows past 2^20 (products), 2^21 (norm, quantising) and 2^25 (reading) in one call."""
    import torch

    import nitrorag_amd as na

    rng = np.random.default_rng(9)
    rows, n = (1 << 25) + 9, 1
    x = rng.standard_normal((rows, n)).astype(np.float32)
    codes, scales = held_on_gpu(lambda c, s: na.row8_quantize(to_gpu(x), c, s), rows, n)
    np.testing.assert_array_equal(codes, 127 * np.sign(x))
    np.testing.assert_array_equal(scales, np.abs(x[:, 0]) / np.float32(127))
    back = torch.empty((rows, n), device="cuda")
    na.row8_read(to_gpu(codes), to_gpu(scales), back)
    np.testing.assert_array_equal(back.cpu().numpy(), codes * scales[:, None])

    rows, n = (1 << 21) + 5, 3
    x, add = (rng.standard_normal((rows, n)).astype(np.float32) for _ in range(2))
    weight, h = rng.uniform(0.5, 1.5, n).astype(np.float32), torch.empty((rows, n), device="cuda")
    codes, scales = held_on_gpu(lambda c, s: na.rms_norm_row8(to_gpu(x), to_gpu(weight), c, s, residual=to_gpu(add), sum=h), rows, n)
    want, y = forms.normed(x, weight, add)
    np.testing.assert_array_equal(h.cpu().numpy(), want)
    top = np.abs(y).max(1)
    np.testing.assert_array_equal(scales, top / np.float32(127))
    np.testing.assert_array_equal(codes, np.rint(y.astype(np.float64) * (np.float32(127) / top)[:, None]))

    rows, n, d = (1 << 20) + 77, 32, 17
    codes, scales = rng.integers(-127, 128, (rows, n)).astype(np.int8), rng.uniform(0.5, 1.5, rows).astype(np.float32)
    residual, mats = rng.standard_normal((rows, d)).astype(np.float32), [forms.matrix(rng, d, n) for _ in range(2)]
    for pair in (mats[:1], mats):
        out = to_gpu(residual)
        na.Q8Weights(*(to_gpu(m[0]) for m in pair)).matmul(to_gpu(codes), to_gpu(scales), out, residual=out, activation="relu")
        check(out.cpu().numpy(), forms.product([m[1:] for m in pair], codes, scales, None, residual, "relu"), f"{len(pair)}")


# ----------------------------------------------------- together, streams, graphs

class Layer:
    """The half of a layer after attention, as a model runs it: the attention's product has
    been added to the stream; norm, gated product, its rows held, w2 added to the stream."""

    def __init__(self, rng, rows, dim, hidden):
        import torch

        import nitrorag_amd as na

        self.na, self.rows = na, rows
        self.up, self.gate, self.down = forms.matrix(rng, hidden, dim), forms.matrix(rng, hidden, dim), forms.matrix(rng, dim, hidden)
        self.w13, self.w2 = na.Q8Weights(to_gpu(self.gate[0]), to_gpu(self.up[0])), na.Q8Weights(to_gpu(self.down[0]))
        self.weight = rng.uniform(0.5, 1.5, dim).astype(np.float32)
        self.dweight = to_gpu(self.weight)
        self.x, self.o = torch.empty((rows, dim), device="cuda"), torch.empty((rows, dim), device="cuda")
        self.hb = torch.empty((rows, hidden), device="cuda")
        self.c, self.s = torch.empty((rows, dim), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        self.hc, self.hs = torch.empty((rows, hidden), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")

    def run(self):
        self.na.rms_norm_row8(self.o, self.dweight, self.c, self.s, residual=self.x, sum=self.x)
        self.w13.matmul(self.c, self.s, self.hb, activation="silu")
        self.na.row8_quantize(self.hb, self.hc, self.hs)
        self.w2.matmul(self.hc, self.hs, self.x, residual=self.x)

    def check(self, x, o):
        """Each step against 64 bits over what the step before it left."""
        h, y = forms.normed(o, self.weight, x)
        c, s = forms.hold(y)
        same((self.c.cpu().numpy(), self.s.cpu().numpy()), (c, s), "norm")
        hb = self.hb.cpu().numpy()
        check(hb, forms.product([self.gate[1:], self.up[1:]], c, s, activation="silu"), "gated")
        hc, hs = forms.hold(hb)
        same((self.hc.cpu().numpy(), self.hs.cpu().numpy()), (hc, hs), "hb")
        check(self.x.cpu().numpy(), forms.product([self.down[1:]], hc, hs, None, h), "w2")

    def fill(self, rng):
        x, o = (rng.standard_normal(tuple(self.x.shape)).astype(np.float32) for _ in range(2))
        self.x.copy_(to_gpu(x))
        self.o.copy_(to_gpu(o))
        return x, o


@pytest.mark.parametrize("rows", [1, 6, 40, 150])
def test_a_layer(rows):
    import torch

    rng = np.random.default_rng(rows)
    layer = Layer(rng, rows, 256, 704)
    given = layer.fill(rng)
    layer.run()
    torch.cuda.synchronize()
    layer.check(*given)


@pytest.mark.parametrize("rows", [1, 40, 150])
def test_a_captured_layer(rows):
    import torch

    rng = np.random.default_rng(rows)
    layer = Layer(rng, rows, 256, 704)
    layer.fill(rng)
    layer.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    for _ in range(3):
        given = layer.fill(rng)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        layer.check(*given)


def test_two_streams():
    import torch

    rng = np.random.default_rng(3)
    layers = [Layer(rng, rows, 256, 704) for rows in (8, 100)]
    streams = [torch.cuda.Stream() for _ in layers]
    given = [layer.fill(rng) for layer in layers]
    torch.cuda.synchronize()
    for layer, stream in zip(layers, streams):
        with torch.cuda.stream(stream):
            layer.run()
    torch.cuda.synchronize()
    for layer, g in zip(layers, given):
        layer.check(*g)


# ------------------------------------------------------------------- refusals

def test_refusals():
    import torch

    import nitrorag_amd as na

    w = torch.zeros((8, 2, 36), dtype=torch.uint8, device="cuda")
    weights = na.Q8Weights(w)
    codes, scales = torch.zeros((3, 64), dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    out = torch.zeros((3, 8), device="cuda")
    weights.matmul(codes, scales, out)
    bad = [
        (codes[:, :32].contiguous(), scales, out, {}), (codes, scales[:2], out, {}), (codes, scales, out[:2], {}),
        (codes, scales, out, {"bias": out[0, :7].contiguous()}), (codes, scales, out, {"residual": out[:2]}),
        (codes, scales, out, {"activation": "tanh"}), (codes[0], scales, out, {})]
    for c, s, o, kw in bad:
        with pytest.raises(na.NitroError):
            weights.matmul(c, s, o, **kw)
    odd = torch.zeros(3 * 64 + 8, dtype=torch.int8, device="cuda")[8:].view(3, 64)
    with pytest.raises(na.NitroError):
        weights.matmul(odd, scales, out)
    for c, s, o in ((codes.float(), scales, out), (codes, scales.double(), out), (codes, scales, out.t()), (codes.cpu(), scales, out),
                    (codes, scales, out.cpu()), (codes, scales, None), (codes, None, out)):
        with pytest.raises(TypeError):
            weights.matmul(c, s, o)
    for wrong in (w.view(-1), w[:, :, :35].contiguous(), torch.zeros((0, 36), dtype=torch.uint8, device="cuda")):
        with pytest.raises(na.NitroError):
            na.Q8Weights(wrong)
    with pytest.raises(na.NitroError):
        na.Q8Weights(w, w[:4])
    for wrong in (w.cpu(), w.view(torch.int8), None):
        with pytest.raises(TypeError):
            na.Q8Weights(wrong)
    x = torch.zeros((3, 64), device="cuda")
    with pytest.raises(na.NitroError):
        na.rms_norm_row8(x, x[0, :60].contiguous(), codes, scales)
    with pytest.raises(na.NitroError):
        na.rms_norm_row8(x, x[0], codes, scales, eps=0.0)
    with pytest.raises(na.NitroError):
        na.row8_quantize(x[:2], codes, scales)
    with pytest.raises(TypeError):
        na.row8_read(codes, scales, x.half())
    torch.cuda.synchronize()


@pytest.mark.parametrize("which", ["x", "weight", "codes", "scales", "residual", "sum"])
def test_norm_refuses_each_tensor(which):
    """Of another shape, type, layout or place, or none where one is needed."""
    import torch

    import nitrorag_amd as na

    x = torch.zeros((3, 64), device="cuda")
    good = {"x": x, "weight": x[0], "codes": torch.zeros((3, 64), dtype=torch.int8, device="cuda"),
            "scales": torch.zeros(3, device="cuda"), "residual": x, "sum": x}
    na.rms_norm_row8(**good)
    t = good[which]
    shapes = [t[:-1].contiguous(), t[None], t.new_zeros(0)]
    for wrong in shapes:
        with pytest.raises(na.NitroError):
            na.rms_norm_row8(**{**good, which: wrong})
    strided = t.new_zeros((*t.shape, 2))[..., 0]
    for wrong in [t.cpu(), t.double(), strided, t.cpu().numpy(), 3] + [None] * (which not in ("residual", "sum")):
        with pytest.raises(TypeError):
            na.rms_norm_row8(**{**good, which: wrong})
    if which in ("x", "codes", "scales"):
        given = {"x": x, "codes": good["codes"], "scales": good["scales"]}
        for call in (na.row8_quantize, na.row8_read):
            for wrong in shapes:
                with pytest.raises(na.NitroError):
                    call(**{**given, which: wrong})
            for wrong in (t.cpu(), strided, None):
                with pytest.raises(TypeError):
                    call(**{**given, which: wrong})
