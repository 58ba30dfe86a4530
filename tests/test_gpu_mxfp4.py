"""Microscaled 4-bit floating point (ruyamd_quantize_mxfp4, ruyamd_dequantize_mxfp4,
ruyamd_mul_mxfp4) against its definition.

Numbers and scales have to be the definition's, bit for bit. Products of blocks with scales near 1
are exact in fp32 whatever the order of their sums: products of two values are multiples of 1/4 up to 36,
with two scales of 1/2 to 2 multiples of 1/16 up to 144, and 7281 of these stay below 2^24 of
these sixteenths. Others are held to the bound of an fp32 sum (grouped_reference.error_bound).
"""
import numpy as np
import pytest
import torch

import grouped_reference as R
import mxfp4_reference as Q
from grouped_reference import COL, ROW, Buffer
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

TYPES = [S.BF16, S.F16, S.F32]
name_of = S.DTYPE_NAMES.get


def announce(*what):
    print("[case]", *what, flush=True)


@pytest.fixture(scope="module")
def context():
    ctx = api.Context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


@pytest.fixture(params=["generic", "chosen"])
def kernel(request, context):
    context.force_generic_kernel(request.param == "generic")
    yield request.param
    context.force_generic_kernel(False)


class Held:
    """`count` matrices of 4-bit values in device memory: pads and gaps (bytes) of data and scales
    filled with 0xff, `shift` bytes in front."""

    def __init__(self, rows, cols, pad=0, scale_pad=0, shift=0, count=1, gap=0):
        self.rows, self.cols, self.shift, self.count = rows, cols, shift, count
        self.row_bytes, self.scale_stride = (cols + 1) // 2 + pad, -(-cols // 32) + scale_pad
        self.matrix_bytes, self.scales_matrix_stride = rows * self.row_bytes + gap, rows * self.scale_stride + gap
        self.data = torch.full((shift + count * self.matrix_bytes + 1,), 255, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((shift + count * self.scales_matrix_stride + 1,), 255, dtype=torch.uint8, device="cuda")

    def parts(self, i=0):
        data = torch.as_strided(self.data, (self.rows, (self.cols + 1) // 2), (self.row_bytes, 1), self.shift + i * self.matrix_bytes)
        scales = torch.as_strided(self.scales, (self.rows, -(-self.cols // 32)), (self.scale_stride, 1),
                                  self.shift + i * self.scales_matrix_stride)
        return data, scales

    def set(self, numbers, scales, i=0):
        data, s = self.parts(i)
        data.copy_(torch.from_numpy(Q.pack(numbers)))
        s.copy_(torch.from_numpy(scales))
        return self

    def matrix(self):
        return api.MxFp4Matrix(self.rows, self.cols, self.data.data_ptr() + self.shift, self.scales.data_ptr() + self.shift,
                               self.row_bytes, self.scale_stride, self.matrix_bytes, self.scales_matrix_stride)

    def values(self, i=0):
        """float64 on the device."""
        data, scales = (t.cpu().numpy() for t in self.parts(i))
        return torch.from_numpy(Q.values(Q.unpack(data, self.cols), scales)).cuda()

    def check(self, numbers, scales):
        """That these are what it has, and its pads are as they were."""
        data, s = (t.cpu().numpy() for t in self.parts())
        assert (s == scales).all(), "%d scales" % (s != scales).sum()
        want = Q.pack(numbers)
        assert (data == want).all(), "%d bytes, the first at %s" % ((data != want).sum(), np.argwhere(data != want)[0])
        rest_d, rest_s = self.data.clone(), self.scales.clone()
        for flat, part in ((rest_d, self.parts()[0]), (rest_s, self.parts()[1])):
            torch.as_strided(flat, part.shape, part.stride(), part.storage_offset()).fill_(255)
            assert (flat == 255).all()


def spread_values(rng, rows, cols, type_):
    """Values of all magnitudes that the type has, zeros of both signs, ties, subnormal ones."""
    low, high = {S.F32: (-149, 127), S.BF16: (-133, 127), S.F16: (-24, 15)}[type_]
    exponent = rng.integers(low, high, (rows, -(-cols // 32))).repeat(32, axis=1)[:, :cols] - rng.integers(0, 6, (rows, cols))
    mantissa = rng.choice([1, 1.25, 1.5, 1.75, 1.125, 1.875], (rows, cols)) * rng.choice([-1, 1], (rows, cols))
    x = np.ldexp(mantissa, exponent)
    x[rng.random((rows, cols)) < 0.1] = 0.0
    x[rng.random((rows, cols)) < 0.1] = -0.0
    return x


CONVERTED = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 7), (4, 64), (7, 515), (3, 2048), (2, 4104), (300, 2051), (40, 8192), (1, 16384),
             # Several rows to a wave, and just not; rows that end in a unit, alone in a segment or not.
             (700, 3), (701, 8), (333, 12), (515, 63), (1000, 96), (130, 129), (257, 250), (65, 256), (300, 257), (4100, 300), (5000, 600),
             (4200, 1025), (2100, 2050), (4099, 770)]


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("rows,cols", CONVERTED)
def test_quantize_and_back(context, kernel, type_, rows, cols):
    announce("quantize", name_of(type_), rows, cols)
    rng = np.random.default_rng(rows * cols)
    for order, pad, shift, q_pad, s_pad in [(ROW, 0, 0, 0, 0), (ROW, 3, 1, 1, 2), (COL, 1, 0, 16, 0)]:
        for make in (lambda: rng.standard_normal((rows, cols)), lambda: spread_values(rng, rows, cols, type_)):
            src = Buffer(type_, rows, cols, order, pad, shift).set(torch.from_numpy(make()))
            x = src.view().double().cpu().numpy()
            numbers, scales = Q.quantize(x)
            held = Held(rows, cols, q_pad, s_pad, shift)
            api.quantize_mxfp4(src.matrix(), context, held.matrix())
            held.check(numbers, scales)
            dst = Buffer(type_, rows, cols, order, pad + 1, shift, fill=-77.0)
            before = dst.flat.clone()
            api.dequantize_mxfp4(held.matrix(), context, dst.matrix())
            want = R.rounded(torch.from_numpy(Q.values(numbers, scales)).cuda(), type_)
            assert torch.equal(dst.view(), want)
            assert dst.untouched(before, lambda i: (slice(None), slice(None)))


@pytest.mark.parametrize("type_", [S.BF16, S.F16], ids=name_of)
def test_quantize_of_every_16_bit_value(context, type_):
    """Every value of the type as the largest of its block, and beside one 1, 2, 4, 8 and 16 times as large."""
    bits = np.arange(65536, dtype=np.uint16).view(np.int16)
    every = torch.from_numpy(bits).view(R.TORCH[type_]).double().numpy()
    for times in (1, 2, 4, 8, 16):
        largest = every * times
        x = np.zeros((65536, 32))
        x[:, 5], x[:, 30] = every, largest
        src = Buffer(type_, 65536, 32).set(torch.from_numpy(x))
        x = src.view().double().cpu().numpy()  # (a product may have gone to infinity)
        numbers, scales = Q.quantize(x)
        held = Held(65536, 32)
        api.quantize_mxfp4(src.matrix(), context, held.matrix())
        held.check(numbers, scales)


def test_quantize_next_to_every_tie(context, kernel):
    """fp32 values at and one step to either side of each border, for scales over the whole range."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    rows = []
    for e in list(range(-149, -100)) + list(range(-100, 126, 5)) + [125]:
        with np.errstate(over="ignore", under="ignore"):
            at = np.ldexp(borders, e).astype(np.float32)
        near = np.concatenate([at, np.nextafter(at, np.float32(np.inf)), np.nextafter(at, np.float32(0))])
        rows.append(np.concatenate([near, -near[:4], np.ldexp(np.float32([7.5]), e)]))
    x = np.stack(rows).astype(np.float64)
    x[~np.isfinite(x)] = 0.0
    src = Buffer(S.F32, *x.shape).set(torch.from_numpy(x))
    x = src.view().double().cpu().numpy()
    numbers, scales = Q.quantize(x)
    held = Held(*x.shape)
    api.quantize_mxfp4(src.matrix(), context, held.matrix())
    held.check(numbers, scales)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_blocks_that_are_not_finite(context, kernel, type_):
    x = torch.randn(6, 100, device="cuda")
    x[0, 3], x[1, 40], x[2, 99], x[3, 64] = float("inf"), float("-inf"), float("nan"), float("-nan")
    src = Buffer(type_, 6, 100).set(x)
    numbers, scales = Q.quantize(src.view().double().cpu().numpy())
    assert (scales == 255).sum() == 4
    held = Held(6, 100)
    api.quantize_mxfp4(src.matrix(), context, held.matrix())
    held.check(numbers, scales)
    dst = Buffer(type_, 6, 100)
    api.dequantize_mxfp4(held.matrix(), context, dst.matrix())
    assert torch.equal(torch.isnan(dst.view()).cpu(), torch.from_numpy(np.isnan(Q.values(numbers, scales))))


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_dequantize_of_every_number_and_scale(context, kernel, type_):
    numbers = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    held = Held(256, 32).set(numbers, scales)
    dst = Buffer(type_, 256, 32)
    api.dequantize_mxfp4(held.matrix(), context, dst.matrix())
    want = torch.from_numpy(Q.values(numbers, scales)).to(R.TORCH[type_]).cuda()
    got = dst.view()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(9, 8, 7), want.nan_to_num(9, 8, 7))


@pytest.mark.parametrize("tokens,top,cols", [(1, 8, 2048), (40, 2, 515), (300, 4, 4096), (9, 3, 33), (500, 3, 100), (333, 2, 7), (70, 5, 255)])
def test_quantize_into_places(context, kernel, tokens, top, cols):
    rng = np.random.default_rng(cols)
    n = tokens * top + 2
    places = rng.permutation(n)[:tokens * top].reshape(tokens, top)
    places = np.where(rng.random(places.shape) < 0.2, rng.choice([-1, n, 2 ** 31 - 1], size=places.shape), places)
    src = Buffer(S.BF16, tokens, cols, ROW, 1).set(torch.from_numpy(rng.standard_normal((tokens, cols))))
    numbers, scales = Q.quantize(src.view().double().cpu().numpy())
    held = Held(n, cols, 2, 1)
    routing = api.Routing(tokens, top, 1, None, torch.tensor(places.astype(np.int32), device="cuda"))
    api.quantize_mxfp4(src.matrix(), context, held.matrix(), routing)
    data, s = (t.cpu().numpy() for t in held.parts())
    want_data, want_s = np.full_like(data, 255), np.full_like(s, 255)
    for t in range(tokens):
        for p in places[t]:
            if 0 <= p < n:
                want_data[p], want_s[p] = Q.pack(numbers[t:t + 1])[0], scales[t]
    assert (data == want_data).all() and (s == want_s).all()


# ---- Products ----

def params_of(dst_type, bias=None, low=None, high=None):
    p = api.MulParams(S.F32, dst_type)
    p.set_bias(bias)
    if low is not None:
        p.set_clamp_min(low)
    if high is not None:
        p.set_clamp_max(high)
    return p


def random_held(rng, rows, cols, pad=0, scale_pad=0, shift=0, count=1, gap=0, low=126, high=128):
    held = Held(rows, cols, pad, scale_pad, shift, count, gap)
    for i in range(count):
        held.set(rng.integers(0, 16, (rows, cols), dtype=np.uint8), rng.integers(low, high + 1, (rows, -(-cols // 32))).astype(np.uint8), i)
    if cols % 2:
        for i in range(count):  # the unused half of a last byte may be anything
            held.parts(i)[0][:, -1] |= 0x70
    return held


def run_mul(context, dst_type, m, n, k, offsets=None, pads=(0, 0, 0, 0), shift=0, gap=0, dst_order=COL, dst_pad=0, bias=False,
            low=None, high=None, seed=0, scales=(126, 128)):
    """One ruyamd_mul_mxfp4 call, checked with everything around it. pads: of rows and scales of lhs and of rhs."""
    rng, count = np.random.default_rng(seed), 1 if offsets is None else len(offsets) - 1
    announce("mxfp4", name_of(dst_type), m, n, k, None if offsets is None else list(map(int, offsets))[:70], pads, shift, gap, dst_order)
    lhs = random_held(rng, m, k, pads[0], pads[1], shift, count, gap, *scales)
    rhs = random_held(rng, n, k, pads[2], pads[3], shift, low=scales[0], high=scales[1])
    dst = Buffer(dst_type, m, n, dst_order, dst_pad, shift % 2, fill=-77.0)
    b = torch.from_numpy(rng.integers(-9, 10, (count, m + 3))).float().cuda() if bias else None
    table = None if offsets is None else torch.tensor(np.asarray(offsets, dtype=np.int32), device="cuda")
    before = dst.flat.clone()
    api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params_of(dst_type, b, low, high), context, dst.matrix(),
                  None if table is None else api.Groups(table, count, 0, m + 3 if bias else 0))
    x, exact = rhs.values(), scales == (126, 128) and k <= 7281
    written = torch.zeros(n, dtype=torch.bool, device="cuda")
    # (A column of two groups, as offsets that run backwards have them, is of either.)
    right = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    for i, (begin, end) in enumerate(R.held_ranges(offsets, n) if offsets is not None else [(0, n)]):
        if begin == end:
            continue
        written[begin:end] = True
        w = lhs.values(i)
        part = x[begin:end].t().contiguous()
        want = w @ part
        bound = None
        if bias:
            want = want + b[i, :m, None].double()
        if not exact:  # (what is rounded to dst's type has the bias in it: half a step of the whole)
            bound = R.error_bound(w.abs() @ part.abs() + (b[i, :m, None].abs() if bias else 0), k, want, dst_type)
        if low is not None or high is not None:
            want = R.clamp(want, -np.inf if low is None else low, np.inf if high is None else high)
        got = dst.view()[:, begin:end]
        right[:, begin:end] |= got == R.rounded(want, dst_type) if exact else (got.double() - want).abs() <= bound
    if offsets is not None and (np.diff(offsets) < 0).any():
        # (Groups that overlap have more columns than the product, for whose number calls are made: some may be left out.)
        right |= dst.view() == -77
    wrong = ~right[:, written]
    assert not wrong.any().item(), "%d wrong, the first at %s" % (wrong.sum().item(), wrong.nonzero()[0].tolist())
    assert dst.untouched(before, lambda i: (slice(None), written))


# m, n, k: few columns and many; depths of one block, below one, of several steps and a bit more, odd ones.
SIZES = [(1, 1, 1), (3, 2, 31), (16, 1, 32), (17, 1, 33), (33, 5, 64), (64, 16, 512), (100, 17, 515), (256, 32, 2048), (1000, 3, 2051),
         (130, 33, 1056), (64, 64, 256), (129, 127, 224), (300, 200, 1000), (256, 256, 768), (515, 300, 2880), (70, 700, 4096),
         (260, 270, 65), (2048, 1, 2048), (300, 40, 95)]


@pytest.mark.parametrize("dst_type", TYPES, ids=name_of)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(context, kernel, dst_type, m, n, k):
    run_mul(context, dst_type, m, n, k)
    run_mul(context, dst_type, m, n, k, None, (1, 1, 3, 2), 1, 0, COL, 3, True, -20.0, 300.0, seed=1)
    run_mul(context, dst_type, m, n, k, None, (16, 4, 32, 0), 0, 0, ROW, 1, True, 0.0, seed=2)


OFFSETS = {
    "even": lambda n: np.linspace(0, n, 6).astype(int),
    "with empty ones": lambda n: np.array([0, 0, n // 3, n // 3, n // 3 + 1, n, n]),
    "not all columns": lambda n: np.array([n // 4, n // 2, n // 2, n - 1]),
    "one": lambda n: np.array([0, n]),
    "outside and backwards": lambda n: np.array([-5, n // 2, n // 4, n + 9, n]),
    "many": lambda n: R.random_offsets(np.random.default_rng(3), 100, n),
}


@pytest.mark.parametrize("kind", list(OFFSETS))
@pytest.mark.parametrize("dst_type", TYPES, ids=name_of)
@pytest.mark.parametrize("m,n,k", [(40, 7, 64), (64, 32, 513), (200, 150, 1024), (300, 700, 288), (129, 1000, 96)])
def test_products_by_groups(context, kernel, dst_type, m, n, k, kind):
    offsets = OFFSETS[kind](n)
    run_mul(context, dst_type, m, n, k, offsets)
    run_mul(context, dst_type, m, n, k, offsets, (1, 2, 0, 3), 1, 5, COL, 2, True, 0.0, seed=1)
    run_mul(context, dst_type, m, n, k, offsets, (16, 0, 16, 0), 0, 48, ROW, 0, True, seed=2)


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("k", [32, 64, 224, 256, 288, 480, 512, 544, 768, 1024, 1040, 1333, 2016])
def test_every_tile_at_every_end_of_the_depth(context, tile, k):
    """One, two and more steps and pairs of steps, whole and cut short; both ways into LDS."""
    context.force_tile(tile, tile)
    try:
        run_mul(context, S.BF16, 300, 290, k)
        assert context.last_kernel_name() == "mxfp4_mfma"
        run_mul(context, S.F32, 270, 300, k, np.array([0, 33, 33, 200, 300]), (16 - (k + 1) // 2 % 16, 3, 16 - (k + 1) // 2 % 16, 1), 0, 16,
                COL, 0, True, 0.0, seed=1)
        run_mul(context, S.F16, 257, 513, k, None, (1, 0, 3, 0), 1, seed=2)
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("tile", [(64, 64, 0), (64, 64, 1), (128, 128, 0), (128, 128, 1), (256, 128, 0), (256, 256, 0)])
@pytest.mark.parametrize("pad", [1, 2, 3, 4, 8, 12, 20])
def test_every_tile_at_every_alignment(context, tile, pad):
    """Rows at multiples of 4 bytes and at any; the matrices of groups apart by multiples of what rows are and not."""
    context.force_tile(*tile)
    try:
        for k in (32, 352, 640, 1024, 1025, 1027):
            run_mul(context, S.F32, 140, 70, k, None, (pad, 0, 0, 4))
            run_mul(context, S.BF16, 70, 140, k, np.array([0, 33, 33, 100, 140]), (pad, 4, 12, 0), 4, 4 * (pad % 3), COL, 1, True, seed=1)
            run_mul(context, S.F16, 65, 66, k, np.array([0, 66]), (0, 0, pad, 1), pad % 4, 0, ROW, 0, True, seed=2)
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("k", [32, 33, 95, 480, 511, 512, 513, 1000, 2048, 3333, 4096, 4111, 16384, 40000])
def test_streams(context, k):
    """Fewer chunks than waves and more, cut short anywhere; one lot of tokens and several, as many as LDS has room for."""
    context.force_tile(16, 16)
    try:
        for m, n in ((200, 1), (33, 20), (130, 70)):
            run_mul(context, S.BF16, m, n, k, scales=(126, 128) if k <= 7281 else (120, 133), seed=n)
            assert context.last_kernel_name() == "mxfp4_stream"
        run_mul(context, S.F32, 97, 90, k, np.array([0, 33, 33, 40, 90]), (3, 1, 1, 2), 1, 5, COL, 1, True, 0.0, seed=1, scales=(120, 133))
        run_mul(context, S.F16, 70, 40, k, None, (16, 4, 0, 1), 0, 0, ROW, 0, True, seed=2, scales=(124, 129))
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("k", [32, 64, 256, 480, 512, 544, 768, 1024, 1280, 1504, 2048, 2080, 4096, 7168, 22528])
def test_tiles_of_four_stages(context, k):
    """Fewer steps than stages, as many, more, pairs cut short anywhere; the deepest that LDS has scales for, and (on
    another tile) deeper."""
    context.force_tile(64, 64, 1)
    try:
        run_mul(context, S.BF16, 200, 130, k)
        assert context.last_kernel_name() == "mxfp4_mfma"
        run_mul(context, S.F32, 97, 300, k, np.array([0, 33, 33, 250, 300]), (16 - (k // 2) % 16, 3, 0, 2), 0, 16, COL, 1, True, 0.0, seed=1)
        run_mul(context, S.F16, 70, 65, k, None, (16 - (k // 2) % 16, 4, 16 - (k // 2) % 16, 1), 0, 0, ROW, 0, True, seed=2)
        run_mul(context, S.F32, 70, 65, k + 1600, scales=(120, 133), seed=3)
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("k", [512, 640, 768, 896, 1024, 1152, 1664, 2048, 4096])
def test_tiles_of_steps_of_128(context, k):
    """Every number of steps to a last lot of scales; one tile and several, cut short on either side."""
    context.force_tile(256, 128)
    try:
        run_mul(context, S.BF16, 256, 128, k)
        assert context.last_kernel_name() == "mxfp4_mfma"
        run_mul(context, S.F32, 300, 290, k, np.array([0, 33, 33, 200, 290]), (4, 4, 12, 8), 4, 16, COL, 1, True, 0.0, seed=1)
        run_mul(context, S.F16, 257, 513, k, None, (16, 4, 0, 0), 0, 0, ROW, 0, True, seed=2)
        run_mul(context, S.BF16, 1000, 700, k, seed=3, scales=(120, 133))
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("tile", [(128, 128, 1), (256, 128, 0), (256, 256, 0)])
@pytest.mark.parametrize("k", [512, 544, 576, 608, 640, 992, 1056, 1120, 1184, 2080, 4064])
def test_scales_at_any_address(context, tile, k):
    """Rows of scales of any number and any distance, beginning anywhere, where they go to LDS as they lie; the last ones end with their
    memory."""
    context.force_tile(*tile)
    try:
        for pad, shift in ((0, 0), (1, 4), (2, 12), (3, 4)):
            run_mul(context, S.BF16, 300, 140, k, None, (0, pad, 16, 0), shift, seed=pad)
            run_mul(context, S.F32, 70, 300, k, np.array([0, 33, 33, 200, 300]), (4, 0, 0, pad), shift, 4 * pad + 4, COL, 1, True, 0.0, seed=pad)
        rng = np.random.default_rng(k)
        m, n = 129, 131
        held = []
        for rows in (m, n):
            numbers, scales = rng.integers(0, 16, (rows, k), dtype=np.uint8), rng.integers(126, 129, (rows, k // 32)).astype(np.uint8)
            odd = torch.zeros(rows * (k // 32) + 1, dtype=torch.uint8, device="cuda")
            odd[1:] = torch.from_numpy(scales).flatten()
            held.append((api.MxFp4Matrix(rows, k, torch.from_numpy(Q.pack(numbers)).cuda(), odd.data_ptr() + 1), odd, Q.values(numbers, scales)))
        y = torch.full((n, m), -77.0, device="cuda")
        api.mul_mxfp4(held[0][0], held[1][0], params_of(S.F32), context, api.Matrix(S.F32, y, api.Layout(m, n, m, COL)))
        assert torch.equal(y.double(), torch.from_numpy(held[1][2] @ held[0][2].T).cuda())
        assert context.last_kernel_name() == "mxfp4_mfma"
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("k", [512, 640, 768, 896, 1024, 1152, 1280, 1408, 1536, 2048, 2176, 2688, 4096, 4224, 7168])
def test_the_largest_tile(context, k):
    """Odd and even numbers of steps and of pairs of steps, whole and cut short by one to three quarters of 512."""
    context.force_tile(256, 256)
    try:
        run_mul(context, S.BF16, 512, 256, k)
        run_mul(context, S.F32, 700, 300, k, None, (16, 4 - k // 32 % 4, 32, 4), 0, 0, COL, 1, True, seed=1)
        run_mul(context, S.F16, 260, 700, k, np.array([0, 5, 5, 300, 650]), (0, 0, 16, 16 - k // 32 % 16), 0, 32, ROW, 0, True, 0.0, seed=2)
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("m,n,k,offsets", [
    (4200, 4352, 512, None), (4352, 4096, 640, None), (5120, 3700, 1152, None), (4352, 4090, 1120, None), (4352, 4096, 544, None), (16384, 1100, 512, None),
    (2048, 9000, 512, [0, 1874, 3199, 4281, 5218, 6056, 6821, 7530, 9000]), (4096, 4480, 768, [0, 0, 4400, 4401, 4480]),
    (512, 33300, 512, list(range(0, 33301, 333)))])
def test_tiles_left_after_full_rounds(context, m, n, k, offsets):
    """More tiles of 256 x 256 than there are CUs: few ones more, half a round of them, and more than that."""
    context.force_tile(256, 256)
    try:
        run_mul(context, S.BF16, m, n, k, offsets and np.array(offsets), bias=True, low=0.0)
        run_mul(context, S.F32, m, n, k, offsets and np.array(offsets), (12, 4, 4, 8), 0, 16, COL, 3, seed=1)
    finally:
        context.force_tile(0, 0)


@pytest.mark.parametrize("m,n,k", [(100, 3, 4096), (64, 20, 1000), (130, 140, 2048), (300, 300, 8000), (16, 1, 40000)])
def test_products_of_scales_of_any_size(context, kernel, m, n, k):
    run_mul(context, S.F32, m, n, k, scales=(110, 140))
    run_mul(context, S.BF16, m, n, k, None, (3, 1, 1, 2), 1, scales=(120, 133), seed=1)


@pytest.mark.parametrize("m,n,k", [(70, 2, 96), (70, 100, 1030), (200, 130, 512)])
def test_scales_at_the_ends_of_their_range(context, kernel, m, n, k):
    """One side's scales 2^-127 .. and the other's 2^100 ..: sums of ordinary size; and products that are
    too small for fp32, which are 0 or as small as these."""
    for a, b in [((0, 3), (250, 254)), ((251, 254), (0, 5)), ((0, 0), (1, 1)), ((254, 254), (127, 127))]:
        rng = np.random.default_rng(7)
        lhs, rhs = random_held(rng, m, k, low=a[0], high=a[1]), random_held(rng, n, k, low=b[0], high=b[1])
        dst = Buffer(S.F32, m, n, COL)
        announce("ends", m, n, k, a, b)
        api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params_of(S.F32), context, dst.matrix())
        w, x = lhs.values(), rhs.values()
        want, magnitude = w @ x.t().contiguous(), w.abs() @ x.abs().t().contiguous()
        # (Each block's sum may be lost where it is below 2^-126.)
        bound = R.error_bound(magnitude, k, want, S.F32) + -(-k // 32) * 2.0 ** -126
        got = dst.view().double()
        fits = magnitude < 2.0 ** 127
        assert ((got - want).abs()[fits] <= bound[fits]).all()


@pytest.mark.parametrize("m,n,k", [(40, 1, 64), (100, 3, 1000), (70, 100, 1030), (300, 140, 512)])
def test_scales_that_are_not_numbers(context, kernel, m, n, k):
    """NaN where a row or a column has one, and nowhere else; pads are 0xff throughout."""
    rng = np.random.default_rng(2)
    lhs, rhs = random_held(rng, m, k, 1, 5), random_held(rng, n, k, 16, 16)
    lhs.parts()[1][m // 2, -1] = 255
    lhs.parts()[1][0, 0] = 255
    rhs.parts()[1][n // 2, k // 64] = 255
    lhs.parts()[0][0] = 0  # (also where all values are 0)
    dst = Buffer(S.BF16, m, n, COL)
    api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params_of(S.BF16), context, dst.matrix())
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[m // 2], want[0], want[:, n // 2] = True, True, True
    assert torch.equal(torch.isnan(dst.view()), want)


def test_empty_calls(context, kernel):
    # No depth: the bias, clamped.
    dst = Buffer(S.F32, 5, 3, COL)
    bias = torch.arange(5.0, device="cuda")
    api.mul_mxfp4(api.MxFp4Matrix(5, 0, None, None), api.MxFp4Matrix(3, 0, None, None), params_of(S.F32, bias, 1.5), context,
                  dst.matrix())
    assert torch.equal(dst.view(), bias.clamp(min=1.5)[:, None].expand(5, 3))
    some = random_held(np.random.default_rng(0), 5, 64)
    for m, n in [(0, 3), (3, 0), (0, 0)]:
        api.mul_mxfp4(api.MxFp4Matrix(m, 64, some.data if m else None, some.scales if m else None),
                      api.MxFp4Matrix(n, 64, some.data if n else None, some.scales if n else None), params_of(S.F32), context,
                      api.Matrix(S.F32, None, api.Layout(m, n, m, COL)))
    api.quantize_mxfp4(api.Matrix(S.F32, None, api.Layout(0, 64, 64, ROW)), context, api.MxFp4Matrix(0, 64, None, None))
    api.quantize_mxfp4(api.Matrix(S.F32, None, api.Layout(5, 0, 0, ROW)), context, api.MxFp4Matrix(5, 0, None, None))
    api.dequantize_mxfp4(api.MxFp4Matrix(5, 0, None, None), context, api.Matrix(S.F32, None, api.Layout(5, 0, 0, ROW)))


@pytest.mark.parametrize("stride", [1 << 23, (1 << 23) + 4, 1 << 25])
def test_rows_far_from_each_other(context, stride):
    """Rows of values, scales and results that lie up to 2^32 bytes and more behind the first one's, and just inside what the offsets of a
    tile of 256 rows reach."""
    m, n, k = 300, 270, 640
    rng = np.random.default_rng(0)
    flat = [torch.empty((rows - 1) * stride + k // 2, dtype=torch.uint8, device="cuda") for rows in (m, m, n, n)]
    values = []
    for rows, data, scales in ((m, *flat[:2]), (n, *flat[2:])):
        numbers, s = rng.integers(0, 16, (rows, k), dtype=np.uint8), rng.integers(126, 129, (rows, k // 32)).astype(np.uint8)
        torch.as_strided(data, (rows, k // 2), (stride, 1)).copy_(torch.from_numpy(Q.pack(numbers)))
        torch.as_strided(scales, (rows, k // 32), (stride, 1)).copy_(torch.from_numpy(s))
        values.append(torch.from_numpy(Q.values(numbers, s)).cuda())
    want = values[1] @ values[0].t().contiguous()
    apart = 1 << 22  # (of columns of dst, in values)
    y = torch.empty((n - 1) * apart + k, dtype=torch.float32, device="cuda")
    results = torch.as_strided(y, (n, m), (apart, 1))
    matrices = [api.MxFp4Matrix(m, k, *flat[:2], stride, stride), api.MxFp4Matrix(n, k, *flat[2:], stride, stride)]
    try:
        for tile in ((16, 16), (64, 64), (64, 64, 1), (128, 128), (128, 128, 1), (256, 128), (256, 256), None):
            announce("far rows", stride, tile)
            context.force_tile(*(tile or (0, 0)))
            context.force_generic_kernel(tile is None)
            results.fill_(-77)
            api.mul_mxfp4(*matrices, params_of(S.F32), context, api.Matrix(S.F32, y, api.Layout(m, n, apart, COL)))
            assert torch.equal(results.double(), want)
    finally:
        context.force_tile(0, 0)
        context.force_generic_kernel(False)
    # Quantised there from columns far from each other, and back.
    x = torch.as_strided(y, (n, k), (apart, 1))
    x.copy_(values[1])
    for t, width in zip(flat[2:], (k // 2, k // 32)):
        torch.as_strided(t, (n, width), (stride, 1)).zero_()
    api.quantize_mxfp4(api.Matrix(S.F32, y, api.Layout(n, k, apart, ROW)), context, matrices[1])
    x.zero_()
    api.dequantize_mxfp4(matrices[1], context, api.Matrix(S.F32, y, api.Layout(n, k, apart, ROW)))
    numbers, scales = Q.quantize(values[1].cpu().numpy())
    assert torch.equal(x.double().cpu(), torch.from_numpy(Q.values(numbers, scales)))


def test_gradients_of_a_product_on_its_values(context):
    """What straight-through training does: forward in 4 bits, the gradient of tokens on dequantised
    weights. With whole numbers, <dy, difference of y> is <dx, step> exactly."""
    m, n, k = 64, 40, 256
    rng = np.random.default_rng(4)
    w, x, step = random_held(rng, m, k, low=127, high=127), random_held(rng, n, k, low=127, high=127), random_held(rng, n, k, low=127, high=127)
    offsets = torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda")
    groups = api.Groups(offsets, 2)
    both = random_held(rng, m, k, count=2, low=127, high=127)
    dy = torch.randint(-4, 5, (n, m), device="cuda").bfloat16()
    values = torch.zeros(2 * m, k, dtype=torch.bfloat16, device="cuda")
    flat = api.MxFp4Matrix(2 * m, k, both.data, both.scales)
    api.dequantize_mxfp4(flat, context, api.Matrix(S.BF16, values, api.Layout(2 * m, k, k, ROW)))
    dx = torch.zeros(n, k, device="cuda")
    api.mul_grouped(api.Matrix(S.BF16, values, api.Layout(k, m, k, COL)), api.Matrix(S.BF16, dy, api.Layout(m, n, m, COL)), groups,
                    params_of(S.F32), context, api.Matrix(S.F32, dx, api.Layout(k, n, k, COL)))
    ys = []
    for held in (x, step):
        y = Buffer(S.F32, m, n, COL)
        api.mul_mxfp4(both.matrix(), held.matrix(), params_of(S.F32), context, y.matrix(), groups)
        ys.append(y.view().double())
    difference = (ys[1] - ys[0]).t()
    assert (difference * dy.double()).sum() == ((step.values() - x.values()) * dx.double()).sum()
    assert w.values().shape == (m, k)


def test_refusals(context):
    held = Held(8, 64)
    host = torch.zeros(4096, dtype=torch.uint8)
    out = torch.zeros(64, device="cuda")

    def refused(code, f, *arguments):
        with pytest.raises(api.RuyAmdError) as e:
            f(*arguments)
        assert e.value.code == code and str(e.value)

    def mx(rows=8, cols=64, data=held.data, scales=held.scales, *strides):
        return api.MxFp4Matrix(rows, cols, data, scales, *strides)

    def mat(rows=8, cols=8, dtype=S.F32, data=out, stride=None, order=COL, zero_point=0):
        return api.Matrix(dtype, data, api.Layout(rows, cols, (rows if order == COL else cols) if stride is None else stride, order),
                          zero_point)

    p = params_of(S.F32)
    mul = api.mul_mxfp4
    bad_mx = [mx(-1), mx(8, -2), mx(8, 64, None), mx(8, 64, held.data, None), mx(8, 64, held.data, held.scales, 31),
              mx(8, 64, held.data, held.scales, 0, 1), mx(8, 64, held.data, held.scales, -1), mx(8, 64, held.data, held.scales, 0, 0, -1)]
    for bad in bad_mx + [mx(7), mx(8, 63)]:
        refused(S.E_INVALID, mul, bad, mx(), p, context, mat())
        refused(S.E_INVALID, mul, mx(), bad, p, context, mat())
    for bad in (mx(8, 64, host), mx(8, 64, held.data, host)):
        refused(S.E_UNSUPPORTED, mul, bad, mx(), p, context, mat())
        refused(S.E_UNSUPPORTED, mul, mx(), bad, p, context, mat())
    for bad in (mat(7), mat(8, 7), mat(stride=7), mat(data=None), mat(zero_point=1), mat(order=2)):
        refused(S.E_INVALID, mul, mx(), mx(), p, context, bad)
    refused(S.E_UNSUPPORTED, mul, mx(), mx(), p, context, mat(data=host))
    refused(S.E_UNSUPPORTED, mul, mx(), mx(), api.MulParams(S.F64, S.F64), context, mat(dtype=S.F64))
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (api.Groups(offsets, 0), api.Groups(offsets, 65537), api.Groups(None, 1), api.Groups(offsets, 1, -1),
                api.Groups(offsets.data_ptr() + 1, 1)):
        refused(S.E_INVALID, mul, mx(), mx(), p, context, mat(), bad)
    bad_p = params_of(S.F32, host)
    refused(S.E_UNSUPPORTED, mul, mx(), mx(), bad_p, context, mat())
    by_column = params_of(S.F32, out)
    by_column.set_channel_dimension(api.ChannelDimension.kCol)
    refused(S.E_UNSUPPORTED, mul, mx(), mx(), by_column, context, mat())
    refused(S.E_INVALID, mul, mx(), mx(), params_of(S.F32, None, float("nan")), context, mat())

    src = torch.zeros(8, 64, device="cuda")
    for bad in bad_mx + [mx(7), mx(8, 63)]:
        refused(S.E_INVALID, api.quantize_mxfp4, mat(8, 64, data=src, order=ROW), context, bad)
        refused(S.E_INVALID, api.dequantize_mxfp4, bad, context, mat(8, 64, data=src, order=ROW))
    refused(S.E_UNSUPPORTED, api.quantize_mxfp4, mat(8, 64, S.I8, src, order=ROW), context, mx())
    refused(S.E_UNSUPPORTED, api.quantize_mxfp4, mat(8, 64, data=torch.zeros(8, 64), order=ROW), context, mx())
    places = torch.zeros(16, dtype=torch.int32, device="cuda")
    for bad in (api.Routing(7, 1, 1, None, places), api.Routing(8, 1, 0, None, places), api.Routing(8, 1, 1, None, None)):
        refused(S.E_INVALID, api.quantize_mxfp4, mat(8, 64, data=src, order=ROW), context, mx(), bad)


@pytest.mark.parametrize("m,n,k", [(2048, 1, 2048), (300, 260, 1024)])
def test_replayed_from_a_graph(context, m, n, k):
    """Quantising and a product recorded once, replayed on other values with eager work in between."""
    x = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    w = random_held(np.random.default_rng(0), m, k)

    def buffers():
        return Held(n, k), torch.zeros(n, m, dtype=torch.bfloat16, device="cuda")

    def step(held, y):
        api.quantize_mxfp4(api.Matrix(S.BF16, x, api.Layout(n, k, k, ROW)), context, held.matrix())
        api.mul_mxfp4(w.matrix(), held.matrix(), params_of(S.BF16), context, api.Matrix(S.BF16, y, api.Layout(m, n, m, COL)))

    own, recorded = buffers(), buffers()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    context.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            step(*recorded)
    finally:
        context.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(*own)
        torch.cuda.synchronize()
        assert own[1].abs().sum() > 0 and torch.equal(own[1], recorded[1]), i


def test_two_contexts_on_their_own_streams():
    """Products of two contexts side by side, of every kind of kernel, again and again: always what each is alone."""
    cases = [((16, 16, 0), 500, 20, 2048), ((64, 64, 0), 500, 300, 1024), ((64, 64, 1), 300, 200, 2080), ((128, 128, 0), 700, 500, 1024),
             ((128, 128, 1), 700, 500, 1120), ((256, 128, 0), 900, 700, 1024), ((256, 256, 0), 900, 700, 1056), ((256, 256, 0), 4352, 4096, 512)]
    contexts, streams = [api.Context() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for ctx, stream in zip(contexts, streams):
        ctx.set_stream(stream.cuda_stream)
        ctx.set_synchronous(False)
    rng = np.random.default_rng(0)
    sets = []
    for tile, m, n, k in cases:
        lhs, rhs = random_held(rng, m, k), random_held(rng, n, k)
        sets.append((tile, lhs, rhs, [[torch.full((n, m), -77.0, device="cuda") for _ in range(3)] for _ in contexts], (m, n)))
    torch.cuda.synchronize()
    announce("two contexts")
    for r in range(3):
        for i in range(len(cases)):
            for c, ctx in enumerate(contexts):
                tile, lhs, rhs, out, (m, n) = sets[(i + 3 * c) % len(cases)]  # (other cases side by side)
                ctx.force_tile(*tile)
                api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params_of(S.F32), ctx, api.Matrix(S.F32, out[c][r], api.Layout(m, n, m, COL)))
    torch.cuda.synchronize()
    for tile, lhs, rhs, out, _ in sets:
        want = (rhs.values() @ lhs.values().t().contiguous()).float()
        for c in range(2):
            for r in range(3):
                assert torch.equal(out[c][r], want), (tile, c, r)
    for ctx in contexts:
        ctx.close()
