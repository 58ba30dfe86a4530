"""What the tolerance of the 4-bit products' ordinary values finds: the definition with one mistake in it, in the formula
itself and on the CPU, has to lie beyond it at every size that it is used at. (With an fp32 destination, which every
kernel is tested with; a rounding to 16 bits is larger than what one position in thousands brings.)"""
import pytest
import torch

import grouped_reference as R
from ruy_amd import _structs as S


def problem(m, k, n, group_size):
    g = torch.Generator().manual_seed(k)
    groups = -(-k // group_size)
    q = torch.randint(16, (m, k + k % 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(m, groups, generator=g) + 0.5
    zeros = torch.randint(16, (m, groups), generator=g, dtype=torch.uint8)
    return q, scales, zeros, torch.randn(k, n, generator=g).double()


def values(q, scales, zeros, k, group_size):
    return R.int4_values(q[:, 0::2] | q[:, 1::2] << 4, scales, zeros, q.shape[0], k, group_size)


@pytest.mark.parametrize("group_size", [32, 64, 96, 128, 10000])
@pytest.mark.parametrize("m,k,n", [(200, 2048, 1), (96, 2051, 3), (64, 8192, 40), (130, 300, 20), (256, 64, 7)])
def test_one_mistake_is_beyond_the_tolerance(m, k, n, group_size):
    q, scales, zeros, x = problem(m, k, n, group_size)
    want = values(q, scales, zeros, k, group_size) @ x
    groups = scales.shape[1]
    bound = R.relative_bound(k + groups, S.F32)

    def beyond(what, w, x=x):
        far = R.relative_error(w @ x, want)
        assert far > 2 * bound, "%s: %.3g, bound %.3g" % (what, far, bound)

    assert R.relative_error(want.float(), want) <= bound
    for at in (0, k // 2, k - 1):
        left_out = x.clone()
        left_out[at] = 0
        beyond("a depth position left out", values(q, scales, zeros, k, group_size), left_out)
    last = groups - 1
    other = zeros.clone()
    other[:, last] ^= 1
    beyond("a group's zero point off by one", values(q, scales, other, k, group_size))
    if groups > 1:
        other = scales.clone()
        other[:, last] = scales[:, last - 1]
        beyond("a group with the scale of its neighbour", values(q, other, zeros, k, group_size))
    swapped = q.clone()
    swapped[:, :32] = q[:, :32].view(m, 16, 2).flip(2).reshape(m, 32)
    beyond("halves of a row's first bytes exchanged", values(swapped, scales, zeros, k, group_size))
