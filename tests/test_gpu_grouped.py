"""Products for layers of experts (ruyamd_mul_grouped, ruyamd_mul_grouped_depth,
ruyamd_mul_int4) against their definitions in 64 bits.

Most problems have small whole numbers for values, and powers of two for scales:
every product and every sum is then exact in fp32 whatever its order, and the
result must be the exact one, rounded once to the destination's type. Problems of
normally distributed values are held to the bound of an fp32 sum in any order
(grouped_reference.error_bound).
"""
import ctypes as C
import sys

import numpy as np
import pytest
import torch

import grouped_reference as R
from grouped_reference import COL, ROW, Buffer
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

TYPES = [S.BF16, S.F16, S.F32]
name_of = S.DTYPE_NAMES.get
KERNELS = ["generic", "chosen"]


def announce(*what):
    print("[case]", *what, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def context():
    ctx = api.Context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


@pytest.fixture(params=KERNELS)
def kernel(request, context):
    context.force_generic_kernel(request.param == "generic")
    yield request.param
    context.force_generic_kernel(False)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def exactly(want, dst_type):
    return R.rounded(want, dst_type)


def check(got, want, dst_type, bound=None):
    if bound is None:
        wrong = got != exactly(want, dst_type)
        assert not wrong.any().item(), "%d wrong, the first at %s" % (wrong.sum().item(), wrong.nonzero()[0].tolist())
        return
    error = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (error <= bound).all(), "%.3g times the bound" % (error / bound).max().item()


def params_of(dst_type, bias=None, low=None, high=None):
    p = api.MulParams(S.F32, dst_type)
    p.set_bias(bias)
    if low is not None:
        p.set_clamp_min(low)
    if high is not None:
        p.set_clamp_max(high)
    return p


def run_columns(context, type_, dst_type, m, k, n, offsets, orders=(ROW, COL, COL), pads=(0, 0, 0), shift=0, gap=0,
                bias=False, low=None, high=None, seed=0, whole=True, call=api.mul_grouped):
    """One ruyamd_mul_grouped call, checked with everything around it."""
    g, count = generator(seed), len(offsets) - 1
    announce("columns", name_of(type_), name_of(dst_type), m, k, n, list(map(int, offsets))[:70], orders, pads, shift, gap)
    lhs = Buffer(type_, m, k, orders[0], pads[0], shift, count, gap)
    rhs = Buffer(type_, k, n, orders[1], pads[1], shift)
    dst = Buffer(dst_type, m, n, orders[2], pads[2], shift, fill=-77.0)
    weights = []
    for i in range(count):
        w = R.whole_numbers(g, (m, k), 3) if whole else torch.randn(m, k, generator=g, device="cuda").double()
        lhs.set(w, i)
        weights.append(lhs.view(i).double())
    x = R.whole_numbers(g, (k, n), 3) if whole else torch.randn(k, n, generator=g, device="cuda").double()
    x = rhs.set(x).view().double()
    b = None
    if bias:  # (with room between one group's and the next one's)
        b = R.whole_numbers(g, (count, m + 3), 9).float()
    table = torch.tensor(np.asarray(offsets, dtype=np.int32), device="cuda")
    before = dst.flat.clone()
    call(lhs.matrix(), rhs.matrix(), api.Groups(table, count, lhs.matrix_stride, m + 3 if bias else 0),
         params_of(dst_type, b, low, high), context, dst.matrix())
    got = dst.view()
    written = torch.zeros(n, dtype=torch.bool, device="cuda")
    for i, (begin, end) in enumerate(R.held_ranges(offsets, n)):
        if begin == end:
            continue
        written[begin:end] = True
        want = weights[i] @ x[:, begin:end]
        bound = None
        if not whole:
            bound = R.error_bound(weights[i].abs() @ x[:, begin:end].abs() + (b[i, :m, None].abs() if bias else 0), k,
                                  want, dst_type)
        if bias:
            want = want + b[i, :m, None].double()
        if low is not None or high is not None:
            want = R.clamp(want, -np.inf if low is None else low, np.inf if high is None else high)
        check(got[:, begin:end], want, dst_type, bound)
    assert dst.untouched(before, lambda i: (slice(None), written))


def run_depth(context, type_, dst_type, m, n, depth, offsets, orders=(COL, ROW, ROW), pads=(0, 0, 0), shift=0, gap=0,
              low=None, seed=0, whole=True):
    """One ruyamd_mul_grouped_depth call."""
    g, count = generator(seed), len(offsets) - 1
    announce("depth", name_of(type_), name_of(dst_type), m, n, depth, list(map(int, offsets))[:70], orders, pads, shift, gap)
    lhs = Buffer(type_, m, depth, orders[0], pads[0], shift)
    rhs = Buffer(type_, depth, n, orders[1], pads[1], shift)
    dst = Buffer(dst_type, m, n, orders[2], pads[2], shift, count, gap, fill=-77.0)
    make = (lambda *s: R.whole_numbers(g, s, 3)) if whole else (
        lambda *s: torch.randn(*s, generator=g, device="cuda").double())
    a, b = lhs.set(make(m, depth)).view().double(), rhs.set(make(depth, n)).view().double()
    table = torch.tensor(np.asarray(offsets, dtype=np.int32), device="cuda")
    before = dst.flat.clone()
    api.mul_grouped_depth(lhs.matrix(), rhs.matrix(), api.Groups(table, count, dst.matrix_stride),
                          params_of(dst_type, None, low), context, dst.matrix())
    for i, (begin, end) in enumerate(R.held_ranges(offsets, depth)):
        # (Contiguous: products of transposed views are left to no library here.)
        want = a[:, begin:end].contiguous() @ b[begin:end].contiguous()
        bound = None
        if not whole:
            bound = R.error_bound(a[:, begin:end].abs().contiguous() @ b[begin:end].abs().contiguous(), end - begin, want,
                                  dst_type)
        if low is not None:
            want = R.clamp(want, low, np.inf)
        check(dst.view(i), want, dst_type, bound)
    assert dst.untouched(before, lambda i: (slice(None), slice(None)))


def run_int4(context, type_, dst_type, m, k, n, group_size, offsets=None, scale_type=S.F16, zeros=True, rhs_order=COL,
             dst_order=COL, pads=(0, 0, 0, 0), shift=0, bias=False, low=None, high=None, seed=0, whole=True, values=None):
    """One ruyamd_mul_int4 call. pads: bytes between rows of 4-bit values, values
    between rows of scales, of rhs and of dst; shift: bytes in front of the data."""
    g, count = generator(seed), len(offsets) - 1 if offsets is not None else 1
    groups = -(-k // group_size)
    announce("int4", name_of(type_), name_of(dst_type), m, k, n, group_size, name_of(scale_type), zeros,
             None if offsets is None else list(map(int, offsets))[:70], rhs_order, dst_order, pads, shift)
    row_bytes, stride = (k + 1) // 2 + pads[0], groups + pads[1]
    gap = 7 if pads[0] else 0
    data = torch.randint(256, (shift + count * (m * row_bytes + gap),), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand(count, m, stride, generator=g, device="cuda").double() + 0.5
    if whole:
        scales = torch.exp2(torch.randint(-2, 3, scales.shape, generator=g, device="cuda").double())
    scales = scales.to(R.TORCH[scale_type])
    zero_points = torch.randint(16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    rhs = Buffer(type_, k, n, rhs_order, pads[2], shift % 2)
    dst = Buffer(dst_type, m, n, dst_order, pads[3], shift % 2, fill=-77.0)
    x = R.whole_numbers(g, (k, n), 3) if whole else torch.randn(k, n, generator=g, device="cuda").double()
    if values is not None:
        x = values(x)
    x = rhs.set(x).view().double()
    b = R.whole_numbers(g, (count, m), 9).float() if bias else None
    weights = api.Int4Matrix(m, k, group_size, data.data_ptr() + shift, scales, scale_type, zero_points,
                             row_bytes if pads[0] else 0, stride if pads[1] else 0,
                             m * row_bytes + gap if gap else 0, 0)
    table = None
    if offsets is not None:
        table = torch.tensor(np.asarray(offsets, dtype=np.int32), device="cuda")
    before = dst.flat.clone()
    api.mul_int4(weights, rhs.matrix(), params_of(dst_type, b, low, high), context, dst.matrix(),
                 None if table is None else api.Groups(table, count))
    written = torch.zeros(n, dtype=torch.bool, device="cuda")
    for i, (begin, end) in enumerate(R.held_ranges(offsets, n) if offsets is not None else [(0, n)]):
        if begin == end:
            continue
        written[begin:end] = True
        at = shift + i * (m * row_bytes + gap)
        w = R.int4_values(data[at:at + m * row_bytes].view(m, row_bytes), scales[i],
                          zero_points[i] if zeros else None, m, k, group_size)
        want = w @ x[:, begin:end]
        bound = None
        if not whole:
            # (Kernels may form the sums of q * x and of x apart: q and a zero point are
            # 15 at most, shifted by 16 31.)
            largest = 48 * scales[i].double()[:, torch.arange(k, device="cuda") // group_size]
            bound = R.error_bound(largest @ x[:, begin:end].abs() + (b[i, :, None].abs() if bias else 0), k + 2 * groups,
                                  want, dst_type)
        if bias:
            want = want + b[i, :, None].double()
        if low is not None or high is not None:
            want = R.clamp(want, -np.inf if low is None else low, np.inf if high is None else high)
        if values is not None:  # (infinities and NaN: where and which they are)
            check_special(dst.view()[:, begin:end].double(), want, bound)
        else:
            check(dst.view()[:, begin:end], want, dst_type, bound)
    assert dst.untouched(before, lambda i: (slice(None), written))


def check_special(got, want, bound=None):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(torch.isinf(got), infinite)
    assert torch.equal(got[infinite], want[infinite])
    fine = torch.isfinite(want)
    if bound is None:
        assert torch.equal(got[fine], want[fine])
    else:
        assert ((got - want).abs()[fine] <= bound[fine]).all()


# ---- Columns dealt to groups ----

@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(a, b, d) for a in (ROW, COL) for b in (ROW, COL) for d in (ROW, COL)], ids=str)
def test_columns_orders_and_small_sizes(context, kernel, type_, orders):
    rng = np.random.default_rng(1)
    for m, k, n, count in [(1, 1, 1, 1), (3, 0, 5, 2), (5, 2, 9, 3), (16, 32, 16, 2), (17, 33, 40, 5), (64, 64, 64, 1),
                           (130, 100, 70, 7)]:
        offsets = R.random_offsets(rng, count, n)
        run_columns(context, type_, type_, m, k, n, offsets, orders, bias=True, low=-20.0, high=30.0, seed=m)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(ROW, COL, COL), (COL, COL, COL), (ROW, ROW, ROW)], ids=str)
def test_columns_strides_and_alignment(context, kernel, type_, orders):
    rng = np.random.default_rng(2)
    for m, k, n, pads, shift, gap in [(48, 72, 33, (1, 3, 5), 1, 0), (40, 64, 130, (8, 8, 8), 8, 16),
                                      (129, 257, 50, (2, 2, 2), 2, 3), (200, 130, 300, (0, 7, 0), 0, 1)]:
        run_columns(context, type_, S.F32, m, k, n, R.random_offsets(rng, 6, n), orders, pads, shift, gap, seed=k)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("m,k,n,count", [(256, 512, 3, 8), (515, 771, 40, 3), (384, 640, 300, 2), (300, 200, 1000, 70),
                                         (1030, 520, 700, 4), (512, 256, 2100, 5)])
def test_columns_of_every_size(context, kernel, type_, m, k, n, count):
    rng = np.random.default_rng(3)
    for orders in [(ROW, COL, COL), (COL, COL, COL)]:
        run_columns(context, type_, type_, m, k, n, R.random_offsets(rng, count, n), orders, bias=True, low=0.0)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("dst_f32", [False, True])
@pytest.mark.parametrize("m,k,n,count", [(200, 2048, 9, 4), (256, 1111, 600, 3)])
def test_columns_of_ordinary_values(context, kernel, type_, dst_f32, m, k, n, count):
    rng = np.random.default_rng(4)
    for orders in [(ROW, COL, COL), (COL, COL, COL)]:
        run_columns(context, type_, S.F32 if dst_f32 else type_, m, k, n, R.random_offsets(rng, count, n), orders,
                    bias=True, whole=False)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_columns_no_group_and_offsets_out_of_range(context, kernel, type_):
    """Columns in front of the first group and behind the last stay as they are;
    offsets outside the matrix or running backwards are held to it."""
    for m, k, n in [(70, 64, 40), (300, 128, 400)]:
        for offsets in ([n // 4, n // 4, n // 2, n - 5], [0, 0, 0], [n, n, n, n], [-50, n // 2, 2 ** 31 - 1],
                        [n // 2, n // 4, n // 4 + 3, 2, n // 4]):
            run_columns(context, type_, type_, m, k, n, offsets, bias=True)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_columns_one_token_to_each_of_many_groups(context, kernel, type_):
    for n, count in [(1, 200), (64, 64), (130, 700)]:
        offsets = np.minimum(np.arange(count + 1) * n // min(n, count), n)
        run_columns(context, type_, type_, 48, 96, n, offsets)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("n", [6, 300])
def test_columns_values_that_are_not_finite(context, kernel, type_, n):
    """They reach the rows and columns they belong to and no others, and do not
    come in from beside the matrices (whose surroundings are NaN here)."""
    g = generator(5)
    for k in (64, 100, 131):
        lhs, rhs = Buffer(type_, 150, k, ROW, 5, 3, 2, 4), Buffer(type_, k, n, COL, 3, 5)
        dst = Buffer(type_, 150, n, COL, fill=-77.0)
        for i in range(2):
            lhs.set(R.whole_numbers(g, (150, k), 3), i)
        rhs.set(R.whole_numbers(g, (k, n), 3))
        lhs.view(1)[7, 1] = float("inf")
        rhs.view()[k - 1, 4] = float("-inf")
        rhs.view()[0, 2] = float("nan")
        cut = n // 2
        table = torch.tensor([0, cut, n], dtype=torch.int32, device="cuda")
        announce("not finite", name_of(type_), k, n)
        api.mul_grouped(lhs.matrix(), rhs.matrix(), api.Groups(table, 2, lhs.matrix_stride), params_of(type_), context,
                        dst.matrix())
        for i, at in enumerate((slice(0, cut), slice(cut, n))):
            want = lhs.view(i).double() @ rhs.view()[:, at].double()
            check_special(dst.view()[:, at].double(), exactly(want, type_).double())


# ---- Depth dealt to groups ----

@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(a, b, d) for a in (ROW, COL) for b in (ROW, COL) for d in (ROW, COL)], ids=str)
def test_depth_orders_and_small_sizes(context, kernel, type_, orders):
    rng = np.random.default_rng(6)
    for m, n, depth, count in [(1, 1, 1, 1), (3, 5, 0, 2), (16, 16, 9, 4), (33, 70, 100, 5), (130, 100, 300, 3)]:
        run_depth(context, type_, S.F32, m, n, depth, R.random_offsets(rng, count, depth), orders, low=-15.0)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(COL, ROW, ROW), (COL, ROW, COL), (ROW, COL, ROW)], ids=str)
def test_depth_strides_and_alignment(context, kernel, type_, orders):
    rng = np.random.default_rng(7)
    for m, n, depth, pads, shift, gap in [(48, 72, 33, (1, 3, 5), 1, 0), (40, 64, 130, (8, 8, 8), 8, 16),
                                          (129, 257, 500, (2, 2, 2), 2, 3), (200, 130, 300, (0, 7, 0), 0, 1)]:
        run_depth(context, type_, type_, m, n, depth, R.random_offsets(rng, 6, depth), orders, pads, shift, gap)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("m,n,depth,count", [(256, 512, 3, 8), (515, 771, 400, 9), (300, 200, 1000, 70),
                                             (1030, 520, 700, 4)])
def test_depth_of_every_size(context, kernel, type_, m, n, depth, count):
    rng = np.random.default_rng(8)
    run_depth(context, type_, type_, m, n, depth, R.random_offsets(rng, count, depth))
    run_depth(context, type_, S.F32, m, n, depth, R.random_offsets(rng, count, depth))


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_depth_of_ordinary_values(context, kernel, type_):
    rng = np.random.default_rng(9)
    run_depth(context, type_, S.F32, 256, 300, 2500, R.random_offsets(rng, 4, 2500), whole=False)
    run_depth(context, type_, type_, 130, 264, 700, R.random_offsets(rng, 2, 700), whole=False)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_depth_no_group_and_offsets_out_of_range(context, kernel, type_):
    for offsets in ([20, 20, 60, 90], [0, 0, 0], [-5, 50, 2 ** 31 - 1], [60, 30, 33, 31, 100]):
        run_depth(context, type_, type_, 70, 90, 100, offsets)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_depth_values_that_are_not_finite_stay_in_their_group(context, kernel, type_):
    g = generator(10)
    lhs, rhs = Buffer(type_, 140, 90, COL, 3, 1), Buffer(type_, 90, 135, ROW, 5, 1)
    dst = Buffer(type_, 140, 135, ROW, 0, 0, 3, fill=-77.0)
    lhs.set(R.whole_numbers(g, (140, 90), 3))
    rhs.set(R.whole_numbers(g, (90, 135), 3))
    lhs.view()[3, 31] = float("inf")   # behind the end of group 0,
    rhs.view()[29, 7] = float("nan")   # in its last place,
    rhs.view()[89, 100] = float("-inf")
    bounds = [0, 30, 31, 90]           # in groups of 30, 1 and 59
    table = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    announce("depth, not finite", name_of(type_))
    api.mul_grouped_depth(lhs.matrix(), rhs.matrix(), api.Groups(table, 3, dst.matrix_stride), params_of(type_), context,
                          dst.matrix())
    for i in range(3):
        at = slice(bounds[i], bounds[i + 1])
        want = lhs.view()[:, at].double().contiguous() @ rhs.view()[at].double().contiguous()
        check_special(dst.view(i).double(), exactly(want, type_).double())


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_gradients_are_the_products_derivative(context, kernel, type_):
    """sum(c * (W x)) is linear in W and in x: a step along any direction changes
    it by that direction's product with the gradients. Whole numbers, so exactly."""
    g = generator(11)
    m, k, n, bounds = 96, 130, 75, [0, 30, 30, 75]
    table = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    groups = api.Groups(table, 3)

    def forward(w, x):
        y = Buffer(S.F32, m, n, COL)
        lhs = Buffer(type_, m, k, ROW, count=3)
        for i in range(3):
            lhs.set(w[i], i)
        api.mul_grouped(lhs.matrix(), Buffer(type_, k, n, COL).set(x).matrix(), groups, params_of(S.F32), context, y.matrix())
        return y.view().double()

    w, dw = R.whole_numbers(g, (3, m, k), 2), R.whole_numbers(g, (3, m, k), 1)
    x, dx = R.whole_numbers(g, (k, n), 2), R.whole_numbers(g, (k, n), 1)
    c = R.whole_numbers(g, (m, n), 2)
    weights = Buffer(type_, m, k, ROW, count=3)
    for i in range(3):
        weights.set(w[i], i)
    cotangent = Buffer(type_, m, n, COL).set(c)
    grad_x, grad_w = Buffer(S.F32, k, n, COL), Buffer(S.F32, m, k, ROW, count=3)
    transposed = weights.matrix()
    transposed.layout = api.Layout(k, m, weights.stride, COL)
    api.mul_grouped(transposed, cotangent.matrix(), groups, params_of(S.F32), context, grad_x.matrix())
    by_rows = Buffer(type_, n, k, ROW).set(x.t())
    api.mul_grouped_depth(cotangent.matrix(), by_rows.matrix(), groups, params_of(S.F32), context, grad_w.matrix())
    difference = (c * (forward(w, x + dx) - forward(w, x - dx))).sum() / 2
    assert difference == (grad_x.view().double() * dx).sum()
    difference = (c * (forward(w + dw, x) - forward(w - dw, x))).sum() / 2
    assert difference == sum((grad_w.view(i).double() * dw[i]).sum() for i in range(3))
    # The bias's gradient: the columns of every group added up.
    ones, grad_b = Buffer(type_, n, 1, ROW).set(torch.ones(n, 1)), Buffer(S.F32, m, 1, ROW, count=3)
    api.mul_grouped_depth(cotangent.matrix(), ones.matrix(), groups, params_of(S.F32), context, grad_b.matrix())
    for i in range(3):
        assert torch.equal(grad_b.view(i)[:, 0].double(), c[:, bounds[i]:bounds[i + 1]].sum(1))


# ---- 4-bit weights ----

@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group_size", [32, 64, 96, 128, 256, 4096])
def test_int4_group_sizes(context, kernel, type_, zeros, group_size):
    for m, k, n in [(48, 512, 1), (33, 300, 3), (20, 1000, 16), (64, 2048, 5)]:
        run_int4(context, type_, type_, m, k, n, group_size, zeros=zeros, bias=True, low=-300.0, high=500.0, seed=k)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("scale_type", TYPES, ids=name_of)
def test_int4_small_and_odd_sizes(context, kernel, type_, scale_type):
    for m, k, n in [(1, 1, 1), (2, 2, 2), (3, 31, 4), (5, 33, 1), (16, 0, 3), (17, 63, 17), (40, 127, 2), (100, 129, 33),
                    (15, 257, 48), (31, 1027, 65), (130, 255, 100)]:
        run_int4(context, type_, S.F32, m, k, n, 32, scale_type=scale_type, seed=m)
        run_int4(context, type_, type_, m, k, n, 5000, scale_type=scale_type, zeros=False, seed=m)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_int4_strides_orders_and_alignment(context, kernel, type_):
    for m, k, n, group_size, pads, shift in [(50, 256, 3, 32, (1, 1, 1, 1), 1), (50, 250, 20, 64, (6, 2, 6, 3), 2),
                                             (64, 512, 8, 128, (16, 4, 8, 8), 16), (40, 511, 35, 32, (3, 0, 1, 0), 5)]:
        for rhs_order, dst_order in [(COL, COL), (ROW, ROW), (ROW, COL), (COL, ROW)]:
            run_int4(context, type_, type_, m, k, n, group_size, rhs_order=rhs_order, dst_order=dst_order, pads=pads,
                     shift=shift)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("group_size", [32, 128])
def test_int4_with_experts(context, kernel, type_, group_size):
    rng = np.random.default_rng(12)
    for m, k, n, count in [(64, 256, 1, 8), (70, 384, 32, 64), (40, 200, 100, 3), (130, 512, 65, 130), (32, 128, 300, 2)]:
        run_int4(context, type_, type_, m, k, n, group_size, R.random_offsets(rng, count, n), bias=True)
    run_int4(context, type_, type_, 48, 128, 40, group_size, [5, 5, 20, 30], pads=(3, 1, 1, 1), shift=1)
    run_int4(context, type_, type_, 48, 128, 40, group_size, [30, 10, 13, 2, 9])


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k,n,group_size", [(512, 4096, 1, 128), (96, 2051, 3, 32), (200, 8192, 40, 64)])
def test_int4_ordinary_values(context, kernel, type_, zeros, m, k, n, group_size):
    run_int4(context, type_, S.F32, m, k, n, group_size, zeros=zeros, scale_type=type_, whole=False)
    run_int4(context, type_, type_, m, k, n, group_size, zeros=zeros, scale_type=S.F32, whole=False, bias=True)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n", [1, 4, 20])
def test_int4_values_that_are_not_finite(context, kernel, type_, zeros, n):
    """An infinity in a column becomes an infinity of the weight's sign or, met by
    a weight of zero, NaN; other columns are what they would be without it."""
    def values(x):
        x = x.clone()
        x[100, 0] = float("inf")
        if n > 1:
            x[3, n - 1] = float("-inf")
        if n > 4:
            x[200, 2] = float("nan")
            x[0, 7], x[-1, 7] = float("inf"), float("-inf")
        return x
    run_int4(context, type_, S.F32, 64, 256, n, 64, zeros=zeros, values=values)
    run_int4(context, type_, S.F32, 33, 211, n, 32, zeros=zeros, values=values)


# ---- Calls ----

def small_call(context, type_=S.BF16, n=8):
    """Objects of a good call, to be spoilt: lhs, rhs, groups, params, dst."""
    lhs, rhs, dst = Buffer(type_, 32, 64, ROW, count=2), Buffer(type_, 64, n, COL), Buffer(type_, 32, n, COL)
    table = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
    return lhs, rhs, api.Groups(table, 2), params_of(type_), dst


def refused(context, code, call, *args):
    with pytest.raises(api.RuyAmdError) as e:
        call(*args)
    assert e.value.code == code, str(e.value)


def test_refusals_of_grouped_products(context):
    def attempt(code, change, call=api.mul_grouped):
        lhs, rhs, groups, params, dst = small_call(context)
        o = {"lhs": lhs.matrix(), "rhs": rhs.matrix(), "groups": groups, "params": params, "dst": dst.matrix()}
        o["keep"] = (lhs, rhs, dst)
        change(o)
        refused(context, code, call, o["lhs"], o["rhs"], o["groups"], o["params"], context, o["dst"])

    def setting(which, **fields):
        def change(o):
            for name, value in fields.items():
                setattr(o[which], name, value)
        return change

    def layout(which, *args):
        return lambda o: setattr(o[which], "layout", api.Layout(*args))

    def dst_type(o):
        o["dst"].dtype = S.F16
        o["params"] = params_of(S.F16)

    def bias(o):
        o["bias"] = torch.zeros(64, device="cuda")
        o["params"].set_bias(o["bias"])

    def bias_by_columns(o):
        bias(o)
        o["params"].set_channel_dimension(api.ChannelDimension.kCol)

    invalid, unsupported = S.E_INVALID, S.E_UNSUPPORTED
    attempt(invalid, lambda o: o.update(groups=None))
    attempt(invalid, layout("lhs", 32, 63, 64, ROW))
    attempt(invalid, layout("rhs", 64, 9, 64, COL))
    attempt(invalid, layout("dst", 31, 8, 32, COL))
    attempt(invalid, layout("lhs", 32, 64, 63, ROW))
    attempt(invalid, layout("rhs", 64, -1, 64, COL))
    attempt(invalid, layout("dst", 32, 8, 32, 2))
    attempt(invalid, setting("lhs", data=None))
    attempt(invalid, setting("rhs", zero_point=3))
    attempt(invalid, lambda o: setattr(o["rhs"], "data", o["rhs"].data + 1))
    attempt(unsupported, setting("lhs", dtype=S.F16))
    attempt(unsupported, setting("rhs", dtype=S.I8))
    attempt(unsupported, dst_type)
    attempt(unsupported, setting("rhs", data=np.zeros(64 * 8, np.int16)))
    attempt(invalid, setting("groups", count=0))
    attempt(invalid, setting("groups", count=65537))
    attempt(invalid, setting("groups", matrix_stride=-1))
    attempt(invalid, setting("groups", offsets=None))
    attempt(unsupported, setting("groups", offsets=np.zeros(3, np.int32)))
    attempt(unsupported, bias_by_columns)
    attempt(unsupported, lambda o: o["params"].set_bias(np.zeros(64, np.float32)))
    attempt(invalid, lambda o: o["params"].set_clamp_min(float("nan")))
    attempt(unsupported, lambda o: setattr(o["params"], "accum_dtype", S.F64))
    attempt(invalid, lambda o: setattr(o["params"], "_mf", 1 << 30))
    # The depth dealt to groups: dst holds the matrices.
    def depth(o):
        o["lhs"].layout, o["rhs"].layout = api.Layout(16, 8, 16, COL), api.Layout(8, 16, 16, ROW)
        o["dst"].layout = api.Layout(16, 8, 16, COL)
    attempt(invalid, depth, api.mul_grouped_depth)
    def depth_bias(o):
        depth(o)
        o["dst"].layout = api.Layout(16, 16, 16, COL)
        bias(o)
    attempt(unsupported, depth_bias, api.mul_grouped_depth)
    # A good call still goes through afterwards, and ruyamd_mul knows the new types no more than before.
    lhs, rhs, groups, params, dst = small_call(context)
    api.mul_grouped(lhs.matrix(), rhs.matrix(), groups, params, context, dst.matrix())
    refused(context, invalid, api.mul, lhs.matrix(), rhs.matrix(), params, context, dst.matrix())
    context.set_runtime_enabled_paths(api.Path.kStandardCpp)
    try:
        refused(context, S.E_NO_PATH, api.mul_grouped, lhs.matrix(), rhs.matrix(), groups, params, context, dst.matrix())
    finally:
        context.set_runtime_enabled_paths(api.Path.kNone)


def test_refusals_of_int4_products(context):
    def attempt(code, groups=None, **fields):
        _, rhs, _, params, dst = small_call(context)
        data = torch.zeros(32 * 32, dtype=torch.uint8, device="cuda")
        scales = torch.ones(32 * 2, dtype=torch.bfloat16, device="cuda")
        w = api.Int4Matrix(32, 64, 32, data, scales, S.BF16)
        for name, value in fields.items():
            setattr(w, name, value)
        if code is None:
            api.mul_int4(w, rhs.matrix(), params, context, dst.matrix(), groups)
        else:
            refused(context, code, api.mul_int4, w, rhs.matrix(), params, context, dst.matrix(), groups)

    attempt(None)
    attempt(None, group_size=65)  # (at least cols: one scale to a row)
    for fields in [dict(group_size=0), dict(group_size=48), dict(group_size=-32), dict(rows=31), dict(cols=62),
                   dict(rows=-1), dict(row_bytes=31), dict(row_bytes=-32), dict(scale_stride=1), dict(matrix_bytes=-1),
                   dict(scales_matrix_stride=-1), dict(data=None), dict(scales=None)]:
        attempt(S.E_INVALID, **fields)
    for fields in [dict(scale_dtype=S.I8), dict(data=np.zeros(1024, np.uint8)), dict(scales=np.zeros(64, np.int16)),
                   dict(zero_points=np.zeros(64, np.uint8))]:
        attempt(S.E_UNSUPPORTED, **fields)
    attempt(S.E_INVALID, groups=api.Groups(None, 1))
    assert api.lib.ruyamd_mul_int4(None, None, None, None, None, None) == S.E_INVALID
    assert api.lib.ruyamd_mul_int4(context._h, None, None, None, None, None) == S.E_INVALID
    assert api.lib.ruyamd_mul_grouped(None, None, None, None, None, None) == S.E_INVALID
    assert api.lib.ruyamd_mul_grouped_depth(context._h, None, None, None, None, None) == S.E_INVALID


def test_nothing_to_write(context):
    for m, n in [(0, 5), (5, 0)]:
        run_columns(context, S.BF16, S.BF16, m, 16, n, [0, n])
        run_depth(context, S.BF16, S.BF16, m, n, 16, [0, 16])
        run_int4(context, S.BF16, S.BF16, m, 64, n, 32)


def test_calls_on_another_stream_and_without_waiting(context):
    """Calls go to the context's stream, in order with the work that fills their
    operands there, and the same object is used call after call."""
    stream = torch.cuda.Stream()
    other = api.Context()
    other.set_stream(stream.cuda_stream)
    other.set_synchronous(False)
    g = generator(13)
    m, k, n = 512, 768, 24
    w = R.whole_numbers(g, (4, m, k), 3)
    xs = [R.whole_numbers(g, (k, n), 3) for _ in range(4)]
    lhs, rhs = Buffer(S.F16, m, k, ROW, count=4), Buffer(S.F16, k, n, COL)
    dsts = [Buffer(S.F32, m, n, COL) for _ in xs]
    for i in range(4):
        lhs.set(w[i], i)
    tables = [torch.tensor(t, dtype=torch.int32, device="cuda")
              for t in ([0, 24, 24, 24, 24], [0, 1, 2, 3, 24], [0, 0, 0, 0, 24], [0, 6, 12, 18, 24])]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for x, table, dst in zip(xs, tables, dsts):
            rhs.set(x)
            api.mul_grouped(lhs.matrix(), rhs.matrix(), api.Groups(table, 4), params_of(S.F32), other, dst.matrix())
    stream.synchronize()
    for x, table, dst in zip(xs, tables, dsts):
        bounds = table.tolist()
        for i in range(4):
            at = slice(bounds[i], bounds[i + 1])
            assert torch.equal(dst.view()[:, at].double(), w[i] @ x[:, at])
    other.close()


def test_recorded_calls_follow_the_offsets(context):
    """A graph of all three calls replayed with other operands and other groups."""
    g = generator(14)
    m, k, n = 256, 384, 40
    lhs, rhs, dst = Buffer(S.BF16, m, k, ROW, count=3), Buffer(S.BF16, k, n, COL), Buffer(S.F32, m, n, COL)
    dw = Buffer(S.F32, m, k, ROW, count=3)
    dy, by_rows = Buffer(S.BF16, m, n, COL), Buffer(S.BF16, n, k, ROW)
    data = torch.randint(256, (3, m, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.ones(3, m, k // 64, device="cuda")
    int4, dst4 = api.Int4Matrix(m, k, 64, data, scales, S.F32), Buffer(S.F32, m, n, COL)
    table = torch.tensor([0, 10, 20, 40], dtype=torch.int32, device="cuda")
    groups = api.Groups(table, 3)
    side = torch.cuda.Stream()
    other = api.Context()
    other.set_stream(side.cuda_stream)
    other.set_synchronous(False)

    def calls():
        api.mul_grouped(lhs.matrix(), rhs.matrix(), groups, params_of(S.F32), other, dst.matrix())
        api.mul_grouped_depth(dy.matrix(), by_rows.matrix(), groups, params_of(S.F32), other, dw.matrix())
        api.mul_int4(int4, rhs.matrix(), params_of(S.F32), other, dst4.matrix(), groups)

    for i in range(3):
        lhs.set(R.whole_numbers(g, (m, k), 3), i)
    rhs.set(R.whole_numbers(g, (k, n), 3))
    dy.set(R.whole_numbers(g, (m, n), 3))
    by_rows.set(R.whole_numbers(g, (n, k), 3))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for bounds in ([0, 10, 20, 40], [0, 0, 40, 40], [3, 4, 4, 9], [0, 13, 26, 39]):
        table.copy_(torch.tensor(bounds, dtype=torch.int32))
        x, c, xt = R.whole_numbers(g, (k, n), 3), R.whole_numbers(g, (m, n), 3), R.whole_numbers(g, (n, k), 3)
        rhs.set(x)
        dy.set(c)
        by_rows.set(xt)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(3):
            at = slice(bounds[i], bounds[i + 1])
            assert torch.equal(dst.view()[:, at].double(), lhs.view(i).double() @ x[:, at])
            assert torch.equal(dw.view(i).double(), c[:, at].contiguous() @ xt[at].contiguous())
            w = R.int4_values(data[i], scales[i], None, m, k, 64)
            assert torch.equal(dst4.view()[:, at].double(), w @ x[:, at])
    del graph
    other.close()


def test_the_ctypes_path_makes_the_same_calls(context, monkeypatch):
    for native in (api.native, None):
        monkeypatch.setattr(api, "native", native)
        run_columns(context, S.BF16, S.F32, 40, 64, 20, [0, 7, 20], bias=True)
        run_depth(context, S.F16, S.F16, 40, 64, 20, [0, 7, 20])
        run_int4(context, S.F32, S.F32, 40, 64, 20, 32, [0, 7, 20])


def test_offsets_of_values_beyond_32_bits(context, kernel):
    """The last group's matrix and rows lie more than 2^32 bytes behind the first's."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    m, k, n, count = 64, 128, 20, 3
    far = (1 << 31) + 64  # values
    g = generator(15)
    flat = torch.zeros(2 * far + m * k, dtype=torch.bfloat16, device="cuda")
    w = R.whole_numbers(g, (count, m, k), 3)
    for i in range(count):
        flat[i * far:i * far + m * k] = w[i].flatten().to(torch.bfloat16)
    rhs, dst = Buffer(S.BF16, k, n, COL), Buffer(S.F32, m, n, COL)
    x = R.whole_numbers(g, (k, n), 3)
    rhs.set(x)
    table = torch.tensor([0, 5, 9, 20], dtype=torch.int32, device="cuda")
    lhs = api.Matrix(S.BF16, flat, api.Layout(m, k, k, ROW))
    announce("far matrices")
    api.mul_grouped(lhs, rhs.matrix(), api.Groups(table, count, far), params_of(S.F32), context, dst.matrix())
    for i, at in enumerate((slice(0, 5), slice(5, 9), slice(9, 20))):
        assert torch.equal(dst.view()[:, at].double(), w[i] @ x[:, at])
    # Long strides: a row (a column) of 2^27 values and more to the next.
    stride = (1 << 27) + 8
    tall = torch.as_strided(flat, (30, k), (stride, 1))
    tall.copy_(R.whole_numbers(g, (30, k), 3))
    lhs = api.Matrix(S.BF16, flat, api.Layout(30, k, stride, ROW))
    one = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    dst = Buffer(S.F32, 30, n, COL)
    api.mul_grouped(lhs, rhs.matrix(), api.Groups(one, 1), params_of(S.F32), context, dst.matrix())
    assert torch.equal(dst.view().double(), tall.double() @ x)
    far_columns = api.Matrix(S.BF16, flat, api.Layout(k, 30, stride, COL))
    lhs, dst = Buffer(S.BF16, m, k, ROW).set(w[0]), Buffer(S.F32, m, 30, COL)
    one = torch.tensor([0, 30], dtype=torch.int32, device="cuda")
    api.mul_grouped(lhs.matrix(), far_columns, api.Groups(one, 1), params_of(S.F32), context, dst.matrix())
    assert torch.equal(dst.view().double(), w[0] @ tall.double().t().contiguous())
    by_rows = api.Matrix(S.BF16, flat, api.Layout(30, k, stride, ROW))
    c = R.whole_numbers(g, (m, 30), 3)
    dy, dw = Buffer(S.BF16, m, 30, COL).set(c), Buffer(S.F32, m, k, ROW)
    api.mul_grouped_depth(dy.matrix(), by_rows, api.Groups(one, 1), params_of(S.F32), context, dw.matrix())
    assert torch.equal(dw.view().double(), c @ tall.double())
    # 4-bit rows and matrices as far apart.
    data = flat.view(torch.uint8)
    scales = torch.ones(2, m, 1, device="cuda")
    q = torch.randint(256, (2, m, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    for i in range(2):
        data[i * 2 * far:i * 2 * far + m * k // 2] = q[i].flatten()
    int4 = api.Int4Matrix(m, k, 128, data, scales, S.F32, matrix_bytes=2 * far)
    table = torch.tensor([0, 5, 20], dtype=torch.int32, device="cuda")
    dst = Buffer(S.F32, m, n, COL)
    api.mul_int4(int4, rhs.matrix(), params_of(S.F32), context, dst.matrix(), api.Groups(table, 2))
    for i, at in enumerate((slice(0, 5), slice(5, 20))):
        assert torch.equal(dst.view()[:, at].double(), R.int4_values(q[i], scales[i], None, m, k, 128) @ x[:, at])


# --- Every kernel, wherever the rules that choose would draw their lines -----

TILES = [(64, 64), (128, 128), (256, 128), (256, 256)]


@pytest.fixture(params=TILES, ids=str)
def tile(request, context):
    context.force_tile(*request.param)
    yield request.param
    context.force_tile()


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(a, b, d) for a in (ROW, COL) for b in (ROW, COL) for d in (ROW, COL)], ids=str)
def test_every_tile_with_columns(context, tile, type_, orders):
    """Depths of one step and less, of as many as a workgroup has buffers for, and of
    more; groups that are empty, of one column, of more than a tile."""
    for m, k, n in [(8, 8, 8), (264, 64, 72), (136, 128, 296), (520, 200, 560), (312, 712, 40)]:
        offsets = [0, n // 8, n // 8, n // 8 + 1, n // 4, n]
        run_columns(context, type_, type_, m, k, n, offsets, orders, bias=True, low=-50.0, seed=m)
        assert context.last_kernel_name() == "grouped_mfma"


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("orders", [(a, b, d) for a in (ROW, COL) for b in (ROW, COL) for d in (ROW, COL)], ids=str)
def test_every_tile_with_depth(context, tile, type_, orders):
    for m, n, depth in [(8, 8, 8), (264, 72, 64), (136, 520, 360), (560, 312, 1000)]:
        offsets = [0, depth // 8, depth // 8, depth // 8 + 1, depth // 4, depth]
        run_depth(context, type_, S.F32, m, n, depth, offsets, orders, seed=m)
        assert context.last_kernel_name() == "grouped_mfma"


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_every_tile_with_ordinary_values(context, tile, type_):
    run_columns(context, type_, type_, 520, 1032, 600, [0, 5, 300, 600], bias=True, whole=False)
    run_depth(context, type_, type_, 264, 520, 1500, [0, 333, 334, 1500], whole=False)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_kernels_are_the_ones_meant(context, type_):
    run_columns(context, type_, type_, 256, 512, 8, [0, 3, 3, 8])
    assert context.last_kernel_name() == "grouped_stream"
    # All columns in one of many groups: several workgroups read its weights.
    run_columns(context, type_, type_, 80, 520, 60, [0] * 7 + [60] * 14)
    assert context.last_kernel_name() == "grouped_stream"
    # Tokens slab by slab.
    run_columns(context, type_, type_, 80, 9000, 20, [0, 20])
    assert context.last_kernel_name() == "grouped_stream"
    run_columns(context, type_, type_, 80, 9000, 9, [0, 9])
    assert context.last_kernel_name() == "grouped_stream"
    run_columns(context, type_, type_, 256, 512, 400, [0, 30, 30, 400])
    assert context.last_kernel_name() == "grouped_mfma"
    run_columns(context, type_, type_, 40, 17, 3, [0, 3])
    assert context.last_kernel_name() in ("generic", "grouped_mfma")
    run_columns(context, type_, type_, 40, 2, 3, [0, 3])
    assert context.last_kernel_name() == "generic"
    run_depth(context, type_, type_, 256, 512, 400, [0, 30, 30, 400])
    assert context.last_kernel_name() == "grouped_mfma"


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
def test_int4_where_something_does_not_fit_into_lds(context, type_, zeros):
    # More scales than there is room for, with and without a whole last group.
    for k in (70016, 131072 + 5):
        run_int4(context, type_, S.F32, 20, k, 2, 32, zeros=zeros, scale_type=S.F32)
        assert context.last_kernel_name() == "int4_stream"
    # Tokens that do not lie side by side: some of them, or none, fit.
    run_int4(context, type_, S.F32, 20, 9000, 12, 128, zeros=zeros, rhs_order=ROW)
    assert context.last_kernel_name() == "int4_stream"
    run_int4(context, type_, S.F32, 20, 70016, 2, 64, zeros=zeros, rhs_order=ROW)
    assert context.last_kernel_name() == "generic"
    # Slab by slab, with experts and a depth that ends inside a slab.
    run_int4(context, type_, S.F32, 50, 4105, 90, 128, offsets=[0, 1, 1, 50, 90], zeros=zeros)
    assert context.last_kernel_name() == "int4_stream"
