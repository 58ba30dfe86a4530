"""A product of 4-bit floats whose destination lies by rows is the one with lhs
and rhs exchanged whose destination lies by columns (ruyamd_mul_mxfp4)."""
import numpy as np
import pytest
import torch

import grouped_reference as R
from test_gpu_mxfp4 import COL, ROW, TYPES, announce, context, name_of, params_of, random_held  # noqa: F401  (context: a fixture)
from ruy_amd import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dst_type", TYPES, ids=name_of)
@pytest.mark.parametrize("m,n,k", [(1, 300, 96), (300, 1, 2048), (130, 257, 1030), (600, 300, 512)])
def test_exchanged(context, dst_type, m, n, k):  # noqa: F811
    announce("exchanged", name_of(dst_type), m, n, k)
    rng = np.random.default_rng(k)
    lhs, rhs = random_held(rng, m, k, 1, 1), random_held(rng, n, k)
    by_rows = torch.full((m, n), float("nan"), dtype=R.TORCH[dst_type], device="cuda")
    exchanged = torch.full_like(by_rows, float("nan"))
    params = params_of(dst_type, None, -50.0, 70.0)
    api.mul_mxfp4(lhs.matrix(), rhs.matrix(), params, context, api.Matrix(dst_type, by_rows, api.Layout(m, n, n, ROW)))
    api.mul_mxfp4(rhs.matrix(), lhs.matrix(), params, context, api.Matrix(dst_type, exchanged, api.Layout(n, m, n, COL)))
    # (Sums of these are exact in fp32, in any order.)
    want = R.rounded(R.clamp(lhs.values() @ rhs.values().t().contiguous(), -50.0, 70.0), dst_type)
    assert torch.equal(by_rows, want) and torch.equal(exchanged, want)
