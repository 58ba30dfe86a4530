"""4-bit products (ruyamd_mul_int4) where a sum of anything but (q - zero) * x, or a token taken apart, would lose what the
definition keeps. Problems of whole numbers have to be exact; see test_gpu_grouped.py for all others."""
import sys

import pytest
import torch

import grouped_reference as R
from grouped_reference import COL, ROW, Buffer
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

TYPES = [S.BF16, S.F16, S.F32]
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


@pytest.fixture(params=["generic", "chosen"])
def kernel(request, context):
    context.force_generic_kernel(request.param == "generic")
    yield request.param
    context.force_generic_kernel(False)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Weights:
    """rows x cols random 4-bit weights; `scales`: what becomes of random numbers between 0 and 1."""

    def __init__(self, g, rows, cols, group_size, zeros, scale_type, scales):
        groups = -(-cols // group_size)
        self.q = torch.randint(16, (rows, cols + cols % 2), generator=g, device="cuda", dtype=torch.uint8)
        self.scales = scales(torch.rand(rows, groups, generator=g, device="cuda")).to(R.TORCH[scale_type])
        self.zeros = torch.randint(16, (rows, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
        self.shape, self.group_size, self.scale_type = (rows, cols), group_size, scale_type

    def set_to_zero_point(self, cols):
        at = torch.tensor(cols, device="cuda")
        self.q[:, at] = 8 if self.zeros is None else self.zeros[:, at // self.group_size]

    def matrix(self):
        self.data = self.q[:, 0::2] | self.q[:, 1::2] << 4
        return api.Int4Matrix(*self.shape, self.group_size, self.data.contiguous(), self.scales, self.scale_type, self.zeros)

    def values(self):
        self.matrix()
        return R.int4_values(self.data, self.scales, self.zeros, *self.shape, self.group_size)


def product(context, weights, x, type_, dst_type, order=COL):
    (m, k), n = weights.shape, x.shape[1]
    rhs, dst = Buffer(type_, k, n, order).set(x), Buffer(dst_type, m, n, COL)
    matrix = weights.matrix()
    api.mul_int4(matrix, rhs.matrix(), api.MulParams(S.F32, dst_type), context, dst.matrix())
    return dst.view(), rhs.view().double()


def powers_of_two(random):
    return torch.exp2(torch.floor(random * 5) - 2)


# What weights equal to their zero point meet leaves no trace.
@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group_size", [32, 64, 96, 128, 5000])
def test_large_tokens_against_weights_of_zero(context, kernel, type_, zeros, group_size):
    large = {S.BF16: 2.0 ** 100, S.F16: 2.0 ** 15, S.F32: 2.0 ** 100}[type_]
    for m, k, n in [(48, 512, 1), (40, 1000, 5), (33, 2051, 20), (64, 700, 40)]:
        announce("zeros", name_of(type_), m, k, n, group_size, zeros)
        g = generator(k)
        w = Weights(g, m, k, group_size, zeros, S.F32, powers_of_two)
        places = [0, 77, k // 2, k - 1]
        w.set_to_zero_point(places)
        x = R.whole_numbers(g, (k, n), 3)
        x[torch.tensor(places, device="cuda")] = large
        for order in (COL, ROW):
            got, x = product(context, w, x, type_, S.F32, order)
            assert torch.equal(got.double(), w.values() @ x)


# Tokens below the normal numbers, multiples of the smallest one. Scales bring the results back; sums of up to 2^24 smallest
# parts are exact.
@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group_size", [32, 64, 96, 128, 5000])
def test_tokens_below_the_normal_numbers(context, kernel, type_, zeros, group_size):
    smallest = {S.BF16: -133, S.F16: -24, S.F32: -149}[type_]
    for m, k, n in [(48, 512, 1), (40, 300, 5), (33, 2051, 20), (64, 700, 40)]:
        announce("small tokens", name_of(type_), m, k, n, group_size, zeros)
        g = generator(k)
        w = Weights(g, m, k, group_size, zeros, S.F32, lambda r: torch.exp2(torch.floor(r * 5) - smallest - 30))
        x = R.whole_numbers(g, (k, n), min(2 ** 24 // (15 * 16 * k), 127)) * 2.0 ** smallest
        # (Ordinary tokens beside them.)
        x[:, 1::3] = R.whole_numbers(g, (k, len(range(1, n, 3))), 3) * 2.0 ** (smallest + 30)
        for order in (COL, ROW):
            got, x = product(context, w, x, type_, S.F32, order)
            assert torch.equal(got.double(), w.values() @ x)


# One value to a token, of 20 bits, from the smallest numbers up to where its parts hold all of them.
@pytest.mark.parametrize("group_size", [32, 128])
def test_tokens_around_the_smallest_that_parts_hold(context, kernel, group_size):
    for m, k, n in [(40, 300, 12), (33, 2051, 12), (64, 520, 60)]:
        announce("20 bits", m, k, n, group_size)
        g = generator(n)
        w = Weights(g, m, k, group_size, True, S.F32, lambda r: torch.exp2(torch.floor(r * 5) + 60))
        x = torch.zeros(k, n, device="cuda", dtype=torch.double)
        for j in range(n):
            x[(37 * j + 5) % k, j] = (2 ** 19 + 2 * j + 1) * 2.0 ** (-149 + j * 36 // n)
        got, x = product(context, w, x, S.F32, S.F32)
        assert torch.equal(got.double(), w.values() @ x)


# Ordinary values by the norm of their error: tests/test_int4_tolerance.py shows which mistakes this finds.
@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group_size", [32, 64, 96, 128, 10000])
def test_norms_of_ordinary_values(context, kernel, type_, zeros, group_size):
    for m, k, n in [(200, 2048, 1), (96, 2051, 3), (64, 8192, 40), (130, 300, 20), (256, 64, 7)]:
        for dst_type in {S.F32, type_}:
            for scale_type in {type_, S.F32}:
                g = generator(k)
                w = Weights(g, m, k, group_size, zeros, scale_type, lambda r: r + 0.5)
                for order in (COL, ROW):
                    got, x = product(context, w, torch.randn(k, n, generator=g, device="cuda").double(), type_, dst_type, order)
                    far = R.relative_error(got, w.values() @ x)
                    bound = R.relative_bound(k + len(w.scales[0]), dst_type)
                    announce("norms", name_of(type_), name_of(dst_type), name_of(scale_type), m, k, n, group_size, zeros,
                             "%.3g of %.3g" % (far, bound))
                    assert far <= bound


# The same beside tokens some thousand times larger that meet weights equal to their zero point.
@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("group_size", [32, 128])
def test_norms_beside_large_tokens(context, kernel, type_, group_size):
    for m, k, n in [(200, 2048, 1), (64, 4100, 40)]:
        g = generator(m)
        w = Weights(g, m, k, group_size, True, S.F32, lambda r: r + 0.5)
        places = [5, k // 3]
        w.set_to_zero_point(places)
        x = torch.randn(k, n, generator=g, device="cuda").double()
        x[torch.tensor(places, device="cuda")] *= 4096
        got, x = product(context, w, x, type_, S.F32)
        far, bound = R.relative_error(got, w.values() @ x), R.relative_bound(k + len(w.scales[0]), S.F32)
        announce("norms beside large tokens", name_of(type_), m, k, n, group_size, "%.3g of %.3g" % (far, bound))
        assert far <= bound
