"""Sizes past the C ABI's 32 bits are refused where Python hands them over (no GPU, no memory:
tensors without data that say they are on the current device)."""
import pytest
import torch

from nitrorag_amd import _native as N
from nitrorag_amd import row8

WRAP = 1 << 32  # what a 32-bit argument takes for 0


class OnDevice(torch.Tensor):
    is_cuda = True

    def get_device(self):
        return 0


def tensor(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta").as_subclass(OnDevice)


@pytest.fixture
def calls(monkeypatch):
    """Device 0 is the current one; what reaches the library is noted, not launched."""
    noted = []

    def call(name, *args):
        if name != "nitro_q8_weights_destroy":
            noted.append((name, *args))

    monkeypatch.setattr(row8, "_bound", (torch.int8, torch.float32, lambda: 0, lambda dev: 0))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(N, "call", call)
    return noted


def entries(rows, n):
    """The calls over rows x n, by name."""
    codes, scales, x = tensor(rows, n, dtype=torch.int8), tensor(rows), tensor(rows, n)
    return {"rms_norm_row8": lambda: row8.rms_norm_row8(x, tensor(n), codes, scales),
            "row8_quantize": lambda: row8.row8_quantize(x, codes, scales),
            "row8_read": lambda: row8.row8_read(codes, scales, x)}


@pytest.mark.parametrize("rows,n", [(1, WRAP + 64), (3, 1 << 31), (WRAP + 5, 32), (1 << 31, 1), (WRAP + 1, 1 << 28)])
@pytest.mark.parametrize("entry", ["rms_norm_row8", "row8_quantize", "row8_read"])
def test_rows_past_32_bits_are_refused(calls, entry, rows, n):
    with pytest.raises(N.NitroError) as e:
        entries(rows, n)[entry]()
    assert e.value.status == N.UNSUPPORTED and not calls


@pytest.mark.parametrize("rows,n", [(1, 1), ((1 << 31) - 1, 1), (1, 1 << 30), (1, (1 << 31) - 1)])
@pytest.mark.parametrize("entry", ["rms_norm_row8", "row8_quantize", "row8_read"])
def test_sizes_of_32_bits_arrive_as_they_are(calls, entry, rows, n):
    entries(rows, n)[entry]()
    assert len(calls) == 1 and calls[0][-3:-1] == (rows, n)


@pytest.mark.parametrize("blocks,d", [(WRAP // 32 + 2, 1), (1, WRAP + 8), ((1 << 25) + 1, 1), (1, (1 << 29) + 1)])
def test_matrices_past_the_limits_are_refused(calls, blocks, d):
    with pytest.raises(N.NitroError) as e:
        row8.Q8Weights(tensor(d, blocks, 36, dtype=torch.uint8))
    assert e.value.status == N.UNSUPPORTED and not calls


def test_product_of_rows_past_32_bits_is_refused(calls):
    weights = row8.Q8Weights(tensor(1 << 29, 1, 36, dtype=torch.uint8))
    assert calls.pop()[3:5] == (32, 1 << 29)
    weights = row8.Q8Weights(tensor(8, 2, 36, dtype=torch.uint8))
    calls.clear()

    def product(rows):
        weights.matmul(tensor(rows, 64, dtype=torch.int8), tensor(rows), tensor(rows, 8))

    for rows in (1 << 31, WRAP + 3):
        with pytest.raises(N.NitroError) as e:
            product(rows)
        assert e.value.status == N.UNSUPPORTED and not calls
    product((1 << 31) - 1)
    assert calls[0][7] == (1 << 31) - 1
