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


@pytest.mark.parametrize("type_", [S.BF16, S.F16, S.F32], ids=name_of)
def test_depth_positions_beyond_2_31_bytes(context, type_):
    """The gradient of a bias, a product with a column of ones: one value behind the other over all of the depth. (Groups at
    the end of it, of less than 16 bytes too: what is in front of them belongs to none.)"""
    size = 4 if type_ == S.F32 else 2
    m, depth = 16 // size, 2 ** 31 // size + 1000
    needs(depth * (m + 1) * size >> 30)
    lhs = torch.empty(depth, m, dtype=R.TORCH[type_], device="cuda")
    ones = torch.empty(depth, dtype=R.TORCH[type_], device="cuda")
    tail = 3000
    first = depth - tail
    lhs[first:] = R.whole_numbers(generator(5), (tail, m), 3).to(R.TORCH[type_])
    # (No ones, for what a position read elsewhere would bring to differ.)
    ones[first:] = R.whole_numbers(generator(6), (tail,), 3).to(R.TORCH[type_])
    for bounds in ([0, 100, 100, 1990, tail], [5, 1999, 2001, 2005, 2900], [tail - 74, tail - 3, tail - 2, tail - 1, tail]):
        announce("far depth", name_of(type_), depth, bounds)
        dst = Buffer(S.F32, m, 1, ROW, count=4)
        api.mul_grouped_depth(api.Matrix(type_, lhs, api.Layout(m, depth, m, COL)),
                              api.Matrix(type_, ones, api.Layout(depth, 1, 1, ROW)), groups_of([first + b for b in bounds]),
                              api.MulParams(S.F32, S.F32), context, dst.matrix())
        assert context.last_kernel_name() == "grouped_mfma"
        for i, (begin, end) in enumerate(zip(bounds, bounds[1:])):
            want = (lhs[first + begin:first + end].double() * ones[first + begin:first + end, None].double()).sum(0)
            assert torch.equal(dst.view(i)[:, 0].double(), want)
        # The other way round: the ones as the only row of lhs, which then is the side along which dst is contiguous.
        dst = Buffer(S.F32, 1, m, COL, count=4)
        api.mul_grouped_depth(api.Matrix(type_, ones, api.Layout(1, depth, 1, COL)),
                              api.Matrix(type_, lhs, api.Layout(depth, m, m, ROW)), groups_of([first + b for b in bounds]),
                              api.MulParams(S.F32, S.F32), context, dst.matrix())
        assert context.last_kernel_name() == "grouped_mfma"
        for i, (begin, end) in enumerate(zip(bounds, bounds[1:])):
            want = (lhs[first + begin:first + end].double() * ones[first + begin:first + end, None].double()).sum(0)
            assert torch.equal(dst.view(i)[0].double(), want)


# 2^20 rows by 1024 columns, a column to each group: more workgroups than 2^32 threads make, streaming and on 64x64 tiles. (One
# group's weights begin a little behind another's: 1024 matrices of their own would be 64 GB.)
MANY_ROWS, MANY_GROUPS = 1 << 20, 1024


def check_columns(dst, values_of, x):
    y = dst.view()
    assert torch.isfinite(y).all()
    for i in list(range(0, MANY_GROUPS, 61)) + [MANY_GROUPS - 1]:
        assert torch.equal(y[:, i].double(), values_of(i) @ x[:, i])


@pytest.mark.parametrize("tile", [(0, 0), (64, 64)], ids=str)
def test_more_tiles_than_one_launch_takes(context, tile):
    needs(8)
    m, k, n, apart = MANY_ROWS, 32, MANY_GROUPS, 8
    flat = R.whole_numbers(generator(7), (m * k + n * apart,), 3).to(torch.bfloat16)
    x = R.whole_numbers(generator(8), (k, n), 2)  # (sums of up to 192: bfloat16 has them all)
    rhs, dst = Buffer(S.BF16, k, n, COL).set(x), Buffer(S.BF16, m, n, COL)
    context.force_tile(*tile)
    try:
        announce("more tiles than one launch takes", tile)
        groups = groups_of(list(range(n + 1)))
        groups.matrix_stride = apart
        api.mul_grouped(api.Matrix(S.BF16, flat, api.Layout(m, k, k, ROW)), rhs.matrix(), groups,
                        api.MulParams(S.F32, S.BF16), context, dst.matrix())
        assert context.last_kernel_name() == "grouped_mfma"
    finally:
        context.force_tile()
    check_columns(dst, lambda i: flat[i * apart:i * apart + m * k].view(m, k).double(), x)


def test_more_4_bit_rows_than_one_launch_takes(context):
    needs(8)
    m, k, n = MANY_ROWS, 32, MANY_GROUPS
    data = torch.randint(256, (m * k // 2 + n,), generator=generator(9), device="cuda", dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-2, 1, (m + n,), generator=generator(10), device="cuda").float())
    x = R.whole_numbers(generator(11), (k, n), 1)
    rhs, dst = Buffer(S.BF16, k, n, COL).set(x), Buffer(S.BF16, m, n, COL)
    weights = api.Int4Matrix(m, k, 32, data, scales, S.F32, matrix_bytes=1, scales_matrix_stride=1)
    announce("more 4-bit rows than one launch takes")
    api.mul_int4(weights, rhs.matrix(), api.MulParams(S.F32, S.BF16), context, dst.matrix(), groups_of(list(range(n + 1))))
    assert context.last_kernel_name() == "generic"

    def values_of(i):
        return R.int4_values(data[i:i + m * k // 2].view(m, k // 2), scales[i:i + m, None], None, m, k, 32)

    check_columns(dst, values_of, x)  # (sums of up to 256 times the scale)


def test_as_many_groups_as_a_call_may_have(context):
    """65536 groups, most of them empty, some with several columns or depth positions, in every kind of kernel."""
    m, k, n, count, apart = 24, 64, 3000, 65536, 8
    rng = torch.Generator().manual_seed(12)
    ends = torch.sort(torch.randint(0, n + 1, (count - 1,), generator=rng)).values
    ends = (ends // 40 * 40).tolist()  # (75 groups of 40, far apart)
    bounds = [0] + ends + [n]
    groups = groups_of(bounds)
    full = [(i, b, e) for i, (b, e) in enumerate(zip(bounds, bounds[1:])) if b < e]
    assert len(full) >= 70
    x = R.whole_numbers(generator(13), (k, n), 3)
    rhs = Buffer(S.BF16, k, n, COL).set(x)
    groups.matrix_stride = apart
    flat = R.whole_numbers(generator(14), (m * k + count * apart,), 3).to(torch.bfloat16)
    dst = Buffer(S.F32, m, n, COL)
    for tile in ((0, 0), (64, 64), (256, 256)):
        context.force_tile(*tile)
        try:
            announce("many groups", tile)
            api.mul_grouped(api.Matrix(S.BF16, flat, api.Layout(m, k, k, ROW)), rhs.matrix(), groups,
                            api.MulParams(S.F32, S.F32), context, dst.matrix())
            assert context.last_kernel_name() == ("grouped_mfma" if tile[0] else "grouped_stream")
        finally:
            context.force_tile()
        for i, begin, end in full:
            w = flat[i * apart:i * apart + m * k].view(m, k).double()
            assert torch.equal(dst.view()[:, begin:end].double(), w @ x[:, begin:end])
        dst.flat.fill_(float("nan"))
    announce("many groups, 4 bits")
    data = torch.randint(256, (m * k // 2 + count,), generator=generator(15), device="cuda", dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-2, 3, (m * 2 + count,), generator=generator(16), device="cuda").float())
    weights = api.Int4Matrix(m, k, 32, data, scales, S.F32, matrix_bytes=1, scales_matrix_stride=1)
    api.mul_int4(weights, rhs.matrix(), api.MulParams(S.F32, S.F32), context, dst.matrix(), groups)
    assert context.last_kernel_name() == "int4_stream"
    for i, begin, end in full:
        w = R.int4_values(data[i:i + m * k // 2].view(m, k // 2), scales[i:i + 2 * m].view(m, 2), None, m, k, 32)
        assert torch.equal(dst.view()[:, begin:end].double(), w @ x[:, begin:end])
    announce("many groups, depth")
    dy = R.whole_numbers(generator(17), (m, n), 3)
    grad = Buffer(S.F32, m, 16, ROW, count=count)
    by_rows = Buffer(S.BF16, n, 16, ROW).set(x[:16].t())
    groups.matrix_stride = 0
    api.mul_grouped_depth(Buffer(S.BF16, m, n, COL).set(dy).matrix(), by_rows.matrix(), groups,
                          api.MulParams(S.F32, S.F32), context, grad.matrix())
    assert context.last_kernel_name() == "grouped_mfma"
    got = grad.flat[:count * m * 16].view(count, m, 16)
    for i, begin, end in full:
        assert torch.equal(got[i].double(), dy[:, begin:end].contiguous() @ x[:16, begin:end].t().contiguous())
    empty = torch.ones(count, dtype=torch.bool, device="cuda")
    empty[[i for i, _, _ in full]] = False
    assert (got[empty] == 0).all()
