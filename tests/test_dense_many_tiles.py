"""Sizes at which a block of the dense kernels does several rows or tiles: rings that wrap, barriers in
their second phase, both halves of tensor memory, sums over many rows."""
import pytest
import torch

import test_block_norm as norms
import test_int8_product as products
from conftest import import_package

import_package()

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SMS = 148


def ceil_div(n, m):
    return -(-n // m)


def tiles(sizes, channels):
    """(rows of a tile, tiles) of a product on the tensor cores, by the rule that picks its kernel: the
    rounds of 148 SMs at 23, 35 or 44 a tile of 64, 128 or 256 rows, a group's last tile half empty."""
    rows, experts = sum(sizes), len(sizes)
    groups, best = min(experts, rows), None
    assert rows > 8 and ceil_div(rows, experts) > 2
    for tile, cost in ((64, 23), (128, 35), (256, 44)):
        n = ceil_div(rows, tile) if experts == 1 else ceil_div(2 * rows + groups * tile, 2 * tile)
        total = ceil_div(n * ceil_div(channels, 128), SMS) * cost
        if best is None or total < best[0]:
            best = total, tile
    return best[1], sum(ceil_div(n, best[1]) for n in sizes) * ceil_div(channels, 128)


RAGGED = [0, 700, 1, 130, 0, 0, 900, 257, 64, 512]
MANY = [(i * 7) % 41 for i in range(64)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,channels,inner,tile", [([500], 4096, 640, 128), ([1100], 4090, 1040, 128), ([2500], 4100, 1040, 256),
                                                       ([2500], 4100, 130, 256), (MANY, 520, 1040, 64), (RAGGED, 1400, 400, 128),
                                                       (RAGGED, 4100, 528, 256), ([640] * 3 + [5, 0, 1290], 2600, 2064, 256)])
def test_products_of_several_tiles_a_block(sizes, channels, inner, tile, dtype):
    chosen, n = tiles(sizes, channels)
    assert chosen == tile and (n > SMS or sizes == [500])
    products.check(sizes, channels, inner, dtype, bias=True)


@gpu
def test_one_group_of_all_rows():
    """The rule goes by the average: here one expert has every row, and its tiles are many rounds."""
    products.check([0] * 15 + [3000], 1030, 272, BF16)


@gpu
@pytest.mark.parametrize("columns,rows", [(264, 12007), (1000, 6007), (1024, 6007), (2048, 3001), (4096, 3001), (8192, 2001), (1207, 6007), (5001, 2001)])
@pytest.mark.parametrize("dtype,residual,kind,gate", [(BF16, BF16, "rms", "element"), (F32, F32, "layer", "element"), (F16, F32, "layer", "row"),
                                                      (F16, F16, "rms", "none")])
def test_norms_of_several_rows_a_block(columns, rows, dtype, residual, kind, gate):
    norms.check(rows, columns, dtype, residual, kind=kind, gate=gate, activation="silu")


@gpu
@pytest.mark.parametrize("columns", [16, 48, 120, 256])
def test_norms_of_several_rows_a_lane(columns):
    norms.check(60013, columns, BF16, kind="rms", activation="silu")
    norms.check(60013, columns, F32, kind="layer", gate="row")
