"""Grouped and 4-bit products from their definitions, in 64 bits, and random
problems for them."""
import numpy as np
import torch

from ruy_amd import _structs as S
from ruy_amd import api

TORCH = {S.BF16: torch.bfloat16, S.F16: torch.float16, S.F32: torch.float32}
# Half the distance from 1 to the next number, and the smallest normal number.
UNIT = {S.BF16: 2.0 ** -8, S.F16: 2.0 ** -11, S.F32: 2.0 ** -24}
SMALLEST = {S.BF16: 2.0 ** -126, S.F16: 2.0 ** -14, S.F32: 2.0 ** -126}
ROW, COL = api.Order.kRowMajor, api.Order.kColMajor


def held_ranges(offsets, total):
    """What the kernels take the caller's offsets for: [(begin, end)] a group."""
    held = [max(0, min(int(o), total)) for o in offsets]
    return [(b, max(b, e)) for b, e in zip(held, held[1:])]


class Buffer:
    """A rows x cols matrix (or `count` of them) in device memory: any order, `pad`
    values between its runs, `shift` values in front, `gap` between matrices."""

    def __init__(self, dtype, rows, cols, order=ROW, pad=0, shift=0, count=1, gap=0, fill=float("nan")):
        self.dtype, self.rows, self.cols, self.order = dtype, rows, cols, order
        inner, outer = (cols, rows) if order == ROW else (rows, cols)
        self.stride, self.shift, self.count = inner + pad, shift, count
        self.matrix_stride = outer * self.stride + gap
        self.flat = torch.full((shift + count * self.matrix_stride + 1,), fill, dtype=TORCH[dtype], device="cuda")

    def _view(self, flat, i):
        strides = (self.stride, 1) if self.order == ROW else (1, self.stride)
        return torch.as_strided(flat, (self.rows, self.cols), strides, self.shift + i * self.matrix_stride)

    def view(self, i=0):
        return self._view(self.flat, i)

    def set(self, values, i=0):
        self.view(i).copy_(values)
        return self

    def matrix(self):
        address = self.flat.data_ptr() + self.shift * self.flat.element_size()
        return api.Matrix(self.dtype, address, api.Layout(self.rows, self.cols, self.stride, self.order))

    def untouched(self, before, outside):
        """Whether everything but the `outside(i)` part (an index or None: all of
        it) of the matrices is as it was."""
        now, then = self.flat.clone(), before.clone()
        for i in range(self.count):
            for flat in (now, then):
                part = outside(i)
                if part is not None:
                    self._view(flat, i)[part] = 0
        kind = torch.int16 if now.element_size() == 2 else torch.int32
        return torch.equal(now.view(kind), then.view(kind))


def whole_numbers(g, shape, largest):
    return torch.randint(-largest, largest + 1, shape, generator=g, device="cuda").double()


def rounded(values, dtype):
    """64-bit values as a destination holds them (they are exact in fp32 here)."""
    return values.float().to(TORCH[dtype])


def clamp(values, low, high):
    return values.clamp(max=high).clamp(min=low)


def error_bound(magnitudes, depth, values, dst_dtype):
    """The largest error of an fp32 sum of depth + 2 terms in any order and by
    any grouping, each addition off by one unit of its result at most (2^-23 of
    it: instructions may cut off), and of the rounding to the destination."""
    return ((depth + 2) * 2.0 ** -23 * magnitudes + UNIT[dst_dtype] * 1.01 * values.abs()
            + SMALLEST[dst_dtype] * UNIT[dst_dtype])


def int4_values(data, scales, zeros, rows, cols, group_size):
    """(q - zero) * scale in 64 bits; data rows x bytes, scales and zeros rows x groups."""
    k = torch.arange(cols, device=data.device)
    q = (data[:rows][:, k // 2].int() >> (4 * (k % 2)).int()) & 15
    z = 8 if zeros is None else zeros[:rows][:, k // group_size].int()
    return (q - z).double() * scales[:rows][:, k // group_size].double()


def random_offsets(rng, count, total, empty=0.3):
    """count + 1 offsets from 0 to total; about `empty` of the groups have nothing."""
    shares = rng.random(count) ** 3 * (rng.random(count) >= empty)
    if shares.sum() == 0:
        shares[rng.integers(count)] = 1.0
    return np.concatenate(([0], np.floor(np.cumsum(shares) / shares.sum() * total + 1e-9).astype(np.int64)))


def relative_error(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def relative_bound(terms, dst_dtype):
    """The norm of an fp32 sum's error by that of many sums of `terms` terms without a common sign: a partial sum is
    in the mean no larger than the whole, each addition is off by 2^-23 of it at most (instructions may cut off), and
    what additions are off by has no common sign either. Then the rounding to the destination."""
    return terms ** 0.5 * 2.0 ** -23 + (UNIT[dst_dtype] if dst_dtype != S.F32 else 0.0)
