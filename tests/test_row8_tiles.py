"""Which kernel takes a product of 8-bit rows (nitro_row8_tile), and that the shapes the
GPU tests run take every one of them.  Needs no GPU."""
import math
import random

import pytest

from nitrorag_amd import _native as N
from nitrorag_amd.row8 import product_tile
from row8_tiles import CASES, GROUPS, blocks_of_a_step, variant


@pytest.mark.parametrize("gated,tile", sorted(CASES))
def test_shapes_take_their_kernel(gated, tile):
    steps, ragged = [], False
    for rows, n, d in CASES[gated, tile]:
        assert product_tile(rows, n, d, gated=gated) == tile, (rows, n, d)
        steps.append(math.ceil(n / 32 / blocks_of_a_step(tile)))
        columns = tile[1] // 2 if gated else tile[1]
        ragged = ragged or rows % tile[0] and d % columns
    assert max(steps) > 2 and ragged
    if tile[2] == 1:
        assert {s % 2 for s in steps if s > 2} == {0, 1} and any(n // 32 % blocks_of_a_step(tile) for _, n, _ in CASES[gated, tile])


@pytest.mark.parametrize("tile", sorted(GROUPS))
def test_groups_take_their_kernel(tile):
    for rows, dim, kv, _, _ in GROUPS[tile]:
        assert product_tile(rows, dim, dim, kv) == tile, (rows, dim, kv)
        # the same over one matrix of all their rows: the same order of sums
        assert product_tile(rows, dim, dim + 2 * kv) == tile, (rows, dim, kv)


def test_no_product_takes_another_kernel():
    tested = {variant(gated, rows, tile) for (gated, tile), shapes in CASES.items() for rows, _, _ in shapes}
    grouped = {variant(False, rows, tile) for tile, shapes in GROUPS.items() for rows, *_ in shapes}
    rng = random.Random(17)

    def size(low, high):
        return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))

    met, met_grouped = set(), set()
    for _ in range(40000):
        rows, n, gated = size(1, 1 << 20), 32 * size(1, 1024), rng.random() < 0.5
        met.add(variant(gated, rows, product_tile(rows, n, size(1, 1 << 17), gated=gated)))
        dim, kv = 32 * size(2, 512), 32 * size(1, 512)
        met_grouped.add(variant(False, rows, product_tile(rows, dim, dim, kv)))
    assert met <= tested and tested <= met, met ^ tested
    # (16 x 32 x 4 for up to 8 rows is taken by groups past 6000 columns only; as a product
    # of its own it is tested above)
    assert {v for v in met_grouped if v[1] != (16, 32, 4)} <= grouped, met_grouped - grouped


def test_largest_sizes_have_a_kernel():
    limit = (1 << 31) - 1
    for rows, n, d in ((limit, 32, 1), (1, 1 << 30, 1), (1, 32, 1 << 29), (64, 32, 1 << 29), (limit, 1 << 30, 64)):
        assert product_tile(rows, n, d)[0] >= 16


@pytest.mark.parametrize("change,status", [
    ({0: 0}, N.INVALID_ARGUMENT), ({0: -1}, N.INVALID_ARGUMENT), ({1: 0}, N.INVALID_ARGUMENT), ({1: 48}, N.INVALID_ARGUMENT),
    ({2: 0}, N.INVALID_ARGUMENT), ({3: -32}, N.INVALID_ARGUMENT), ({3: 32, 4: 1}, N.INVALID_ARGUMENT), ({5: None}, N.INVALID_ARGUMENT),
    ({1: (1 << 30) + 32}, N.UNSUPPORTED), ({2: (1 << 29) + 1}, N.UNSUPPORTED), ({3: (1 << 29) + 1}, N.UNSUPPORTED)])
def test_tile_refuses(change, status):
    import ctypes

    args = [4, 64, 8, 0, 0, (ctypes.c_int32 * 3)()]
    for i, v in change.items():
        args[i] = v
    with pytest.raises(N.NitroError) as e:
        N.call("nitro_row8_tile", *args)
    assert e.value.status == status


def test_binding_refuses_sizes_past_32_bits():
    for args in ((1 << 32, 32, 8), (1, 1 << 32, 8), (1, 32, (1 << 32) + 8), (1, 32, 8, 1 << 32)):
        with pytest.raises(N.NitroError):
            product_tile(*args)
