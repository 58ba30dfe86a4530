"""Grouped products (ruyamd_mul_grouped, ruyamd_mul_grouped_depth, ruyamd_mul_int4) of strides and sizes at and beyond
what offsets of 32 bits and single launches hold. Whole numbers: every result is the exact one."""
import sys

import pytest
import torch

import grouped_reference as R
from grouped_reference import COL, ROW, Buffer
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

name_of = S.DTYPE_NAMES.get


def announce(*what):
    print("[case]", *what, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def context():
    ctx = api.Context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


def needs(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < (gigabytes + 4) << 30:
        pytest.skip("needs %d GB of device memory" % gigabytes)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def groups_of(bounds):
    return api.Groups(torch.tensor(bounds, dtype=torch.int32, device="cuda"), len(bounds) - 1)


def far_rows(type_, rows, cols, pitch, seed):
    """rows x cols whole numbers, `pitch` values from a row to the next; what lies between is not written."""
    flat = torch.empty((rows - 1) * pitch + cols, dtype=R.TORCH[type_], device="cuda")
    view = torch.as_strided(flat, (rows, cols), (pitch, 1))
    view.copy_(R.whole_numbers(generator(seed), (rows, cols), 3))
    return flat, view


# The runs of a tile begin up to (rows of the tile - 1) pitches behind its first. 2^31 bytes are 255 pitches of 4 210 752 values
# of 16 bits and 127 of 8 454 660, and pitches above 8 388 480 values are not for tiles; of 32 bits 127 of 4 227 330 and
# 4 194 176.
@pytest.mark.parametrize("type_", [S.BF16, S.F16], ids=name_of)
@pytest.mark.parametrize("pitch", [4210744, 4210752, 4210760, 5242880, 8388480, 8388488])
@pytest.mark.parametrize("tile", [(256, 256), (256, 128), (128, 128), (0, 0)], ids=str)
def test_rows_of_a_tile_beyond_2_31_bytes(context, type_, pitch, tile):
    rows, k, other = 300, 136, 264
    needs(rows * pitch * 2 >> 30)
    flat, far = far_rows(type_, rows, k, pitch, 1)
    near = R.whole_numbers(generator(2), (2, k, other), 3)
    context.force_tile(*tile)
    try:
        announce("far rows", name_of(type_), pitch, tile)
        # As weights by rows.
        x, y = Buffer(type_, k, other, COL).set(near[0]), Buffer(S.F32, rows, other, COL)
        api.mul_grouped(api.Matrix(type_, flat, api.Layout(rows, k, pitch, ROW)), x.matrix(), groups_of([0, other]),
                        api.MulParams(S.F32, S.F32), context, y.matrix())
        assert torch.equal(y.view().double(), far.double() @ near[0])
        # As tokens by columns, in groups that begin inside a tile and end with one.
        w, y = Buffer(type_, other, k, ROW, count=2), Buffer(S.F32, other, rows, COL)
        for i in range(2):
            w.set(near[i].t(), i)
        api.mul_grouped(w.matrix(), api.Matrix(type_, flat, api.Layout(k, rows, pitch, COL)), groups_of([0, 5, rows]),
                        api.MulParams(S.F32, S.F32), context, y.matrix())
        tokens = far.double().t().contiguous()
        for i, at in enumerate((slice(0, 5), slice(5, rows))):
            assert torch.equal(y.view()[:, at].double(), near[i].t().contiguous() @ tokens[:, at])
    finally:
        context.force_tile()


@pytest.mark.parametrize("pitch", [4194176, 4194180])
def test_rows_of_a_tile_beyond_2_31_bytes_of_fp32(context, pitch):
    rows, k, n = 300, 100, 264
    needs(rows * pitch * 4 >> 30)
    flat, far = far_rows(S.F32, rows, k, pitch, 3)
    x = R.whole_numbers(generator(4), (k, n), 3)
    for tile in ((128, 128), (64, 64), (0, 0)):
        context.force_tile(*tile)
        try:
            announce("far rows", "f32", pitch, tile)
            rhs, y = Buffer(S.F32, k, n, COL).set(x), Buffer(S.F32, rows, n, COL)
            api.mul_grouped(api.Matrix(S.F32, flat, api.Layout(rows, k, pitch, ROW)), rhs.matrix(), groups_of([0, n]),
                            api.MulParams(S.F32, S.F32), context, y.matrix())
            assert torch.equal(y.view().double(), far.double() @ x)
        finally:
            context.force_tile()
