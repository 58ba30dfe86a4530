"""Microscaled 4-bit floating point from its definition, in 64 bits on the host."""
import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BLOCK = 32


def quantize(x):
    """(numbers 0 .. 15, scales) of the rows of a float64 array that fp32 holds exactly."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    numbers, scales = np.zeros((rows, cols), np.uint8), np.zeros((rows, blocks), np.uint8)
    for b in range(blocks):
        v = x[:, b * BLOCK:(b + 1) * BLOCK]
        fine = np.isfinite(v).all(axis=1)
        v = np.where(fine[:, None], v, 0.0)
        largest = np.abs(v).max(axis=1)
        # frexp: largest = f * 2 ** e with f in [0.5, 1), so its power of two is e - 1.
        exponent = np.where(largest > 0, np.maximum(np.frexp(largest)[1] - 1 - 2, -127), -127)
        scaled = np.ldexp(np.abs(v), -exponent[:, None])
        low = np.clip(np.searchsorted(MAGNITUDES, scaled, side="right") - 1, 0, 6)
        middle = (MAGNITUDES[low] + MAGNITUDES[low + 1]) / 2
        # (A tie goes to the number whose last bit is 0.)
        n = low + ((scaled > middle) | ((scaled == middle) & (low % 2 == 1)))
        n = n + 8 * np.signbit(v)
        numbers[:, b * BLOCK:(b + 1) * BLOCK] = np.where(fine[:, None], n, 0)
        scales[:, b] = np.where(fine, exponent + 127, 255)
    return numbers, scales


def pack(numbers):
    """Two numbers to a byte, the first one low; the unused half of a last byte is 0."""
    if numbers.shape[1] % 2:
        numbers = np.concatenate([numbers, np.zeros((len(numbers), 1), np.uint8)], axis=1)
    return numbers[:, 0::2] | numbers[:, 1::2] << 4


def unpack(data, cols):
    return np.stack([data & 15, data >> 4], axis=2).reshape(len(data), -1)[:, :cols]


def values(numbers, scales):
    """float64 values; NaN where the scale is 255."""
    v = MAGNITUDES[numbers & 7] * np.where(numbers & 8, -1.0, 1.0)
    s = scales.astype(np.int64).repeat(BLOCK, axis=1)[:, :v.shape[1]]
    return np.where(s == 255, np.nan, np.ldexp(v, (s - 127).astype(np.int32)))
