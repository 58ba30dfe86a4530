"""Products of 4-bit floats by groups whose offsets run backwards (ruyamd_mul_mxfp4).

Groups then overlap: a column of two groups is of either, and has to be one of the two, element by element. As
launches are made for as many columns as the product has, kernels on tiles may leave some out where groups have
more; the generic kernel leaves out none. What is not written keeps a NaN, which no product here has.
"""
import numpy as np
import pytest
import torch

import grouped_reference as R
from test_gpu_mxfp4 import COL, TYPES, announce, context, name_of, params_of, random_held  # noqa: F401  (context: a fixture)
from ruy_amd import api

pytestmark = pytest.mark.gpu

TILES = [(16, 16, 0), (64, 64, 0), (64, 64, 1), (128, 128, 0), (128, 128, 1), (256, 128, 0), (256, 256, 0)]


def share_written(context, dst_type, m, n, k, offsets):  # noqa: F811
    """Makes a call, checks what it wrote; which part of the columns that any group has that is."""
    rng = np.random.default_rng(n)
    announce("backwards", name_of(dst_type), m, n, k, offsets)
    lhs, rhs = random_held(rng, m, k, count=len(offsets) - 1), random_held(rng, n, k)
    y = torch.full((n, m), float("nan"), dtype=R.TORCH[dst_type], device="cuda")
    table = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params_of(dst_type), context, api.Matrix(dst_type, y, api.Layout(m, n, m, COL)),
                  api.Groups(table, len(offsets) - 1))
    x, right = rhs.values(), torch.zeros_like(y, dtype=torch.bool)
    covered = torch.zeros(n, dtype=torch.bool, device="cuda")
    for i, (begin, end) in enumerate(R.held_ranges(offsets, n)):
        covered[begin:end] = True
        if begin < end:
            # (Sums of these are exact in fp32, in any order.)
            right[begin:end] |= y[begin:end] == R.rounded(x[begin:end] @ lhs.values(i).t().contiguous(), dst_type)
    written = ~torch.isnan(y)
    assert not written[~covered].any()
    assert right[written].all(), "%d wrong" % (written & ~right).sum().item()
    return written[covered].float().mean().item()


BACKWARDS = [(130, 40, 512, [0, 30, 10, 40, 40]), (300, 300, 1024, [-5, 200, 50, 309, 300]), (70, 100, 544, [60, 0, 100, 20, 20])]


def enough(tile, n, offsets):
    """Whether a launch makes all of the groups' tiles: it is made for n // columns of a tile + groups of these, which is enough for
    groups that do not overlap. (The streaming kernel's have 16 columns or 32. The second case above has 29 lots of 16, of which 22 are
    made, or 15 of 32, of which 13 are; 8 of 64, 4 of 128 and 2 of 256 are all made.)"""
    counts = [end - begin for begin, end in R.held_ranges(offsets, n)]
    return all(sum(-(-c // t) for c in counts) <= n // t + len(counts) for t in ((16, 32) if tile[1] == 16 else tile[1:2]))


@pytest.mark.parametrize("dst_type", TYPES, ids=name_of)
@pytest.mark.parametrize("m,n,k,offsets", BACKWARDS)
def test_the_generic_kernel_writes_all_columns(context, dst_type, m, n, k, offsets):  # noqa: F811
    context.force_generic_kernel(True)
    try:
        assert share_written(context, dst_type, m, n, k, offsets) == 1
        assert context.last_kernel_name() == "generic"
    finally:
        context.force_generic_kernel(False)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k,offsets", BACKWARDS)
def test_tiles_write_all_columns_where_they_are_enough(context, tile, m, n, k, offsets):  # noqa: F811
    context.force_tile(*tile)
    try:
        for dst_type in TYPES:
            share = share_written(context, dst_type, m, n, k, offsets)
            assert share == 1 if enough(tile, n, offsets) else share > 0.5
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("tile", TILES)
def test_tiles_that_are_too_few(context, tile):  # noqa: F811
    """Three groups that each have all 2000 columns, and a launch for 2000 // tile + 5 lots of them: as all tiles have the same rows and
    no column is in more than three, a third of these lots' columns is written at least. With the last of each group, which are shorter,
    among them: of 16 columns 130 lots, 2080 / 6000 = 0.346; of 32 64 and 3 of 16, 0.349; of 64 33 and 3 of 16, 0.36; of 128 17 and 3 of 80,
    0.40; of 256 9 and 3 of 208, 0.48."""
    context.force_tile(*tile)
    try:
        assert share_written(context, TYPES[0], 256, 2000, 512, [0, 2000, 0, 2000, 0, 2000]) >= 0.34
    finally:
        context.force_tile(0, 0)
