"""Rows of 2^30 entries, the longest there are: held and normed bit for bit against their
definition, read back, multiplied; norm and holding also at a ragged end, one entry less."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LONGEST = 1 << 30
CHUNK = 1 << 25


@pytest.fixture(scope="module", autouse=True)
def gpu():
    import torch

    assert torch.cuda.is_available(), "GPU tests need a GPU"
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def held(codes, scales, y_of, n):
    """codes and scales are those of the row whose chunks y_of(at, to) gives."""
    import torch

    top = max(y_of(at, min(at + CHUNK, n)).abs().max().item() for at in range(0, n, CHUNK))
    assert scales.item() == np.float32(top) / np.float32(127)
    inv = float(np.float32(127) / np.float32(top))
    for at in range(0, n, CHUNK):
        to = min(at + CHUNK, n)
        assert torch.equal(codes[0, at:to], torch.round(y_of(at, to).double() * inv).to(torch.int8)), at


@pytest.mark.parametrize("n", [LONGEST, LONGEST - 1])
def test_longest_row(n):
    import torch

    import nitrorag_amd as na

    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((1, n), device="cuda", generator=gen)
    codes, scales = torch.empty((1, n), dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    print(f"row of {n}", flush=True)
    na.row8_quantize(x, codes, scales)
    held(codes, scales, lambda at, to: x[0, at:to], n)
    back = torch.empty_like(x)
    na.row8_read(codes, scales, back)
    for at in range(0, n, CHUNK):
        assert torch.equal(back[0, at:at + CHUNK], codes[0, at:at + CHUNK].float() * scales)

    weight = torch.rand(n, device="cuda", generator=gen).add_(0.5)
    print("norm", flush=True)
    na.rms_norm_row8(x, weight, codes, scales, residual=back, sum=back)
    back2 = torch.empty((1, n), device="cuda")  # (what the residual was)
    again = torch.empty((1, n), dtype=torch.int8, device="cuda")
    again_scale = torch.empty(1, device="cuda")
    na.row8_quantize(x, again, again_scale)
    na.row8_read(again, again_scale, back2)
    total = 0.0
    for at in range(0, n, CHUNK):
        h = x[0, at:at + CHUNK] + back2[0, at:at + CHUNK]
        assert torch.equal(back[0, at:at + CHUNK], h)
        total += (h.double() * h.double()).sum().item()
    r = 1 / np.sqrt(total / n + 1e-5)
    held(codes, scales, lambda at, to: (back[0, at:to].double() * r * weight[at:to].double()).float(), n)


def test_product_of_the_longest_row():
    """Zeros but for four blocks, the first and the last of the row among them: exact sums."""
    import torch

    import nitrorag_amd as na

    nb, d = LONGEST // 32, 3
    places = [0, 1, nb // 2 + 7, nb - 1]
    rng = np.random.default_rng(1)
    w = torch.zeros((d, nb, 36), dtype=torch.uint8, device="cuda")
    codes, scales = torch.zeros((1, LONGEST), dtype=torch.int8, device="cuda"), torch.full((1,), 0.5, device="cuda")
    want = np.zeros(d)
    for j in places:
        x, q = rng.integers(-127, 128, 32).astype(np.int8), rng.integers(-127, 128, (d, 32)).astype(np.int8)
        codes[0, 32 * j:32 * j + 32] = torch.from_numpy(x).cuda()
        w[:, j, 4:] = torch.from_numpy(q.view(np.uint8)).cuda()
        w[:, j, :4] = torch.tensor([2.0], device="cuda").view(torch.uint8)
        want += q.astype(np.float64) @ x.astype(np.float64)
    out = torch.empty((1, d), device="cuda")
    print("product of the longest row", flush=True)
    na.Q8Weights(w).matmul(codes, scales, out)
    assert out[0].tolist() == want.tolist()
