"""The bare loops of matrix instructions (ruyamd_diag_mfma_ceiling)."""
import pytest
import torch

from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

# Published dense rates of the card, TOP/s: no loop is faster.
PEAKS = {0: 5.04e3, 1: 5.04e3, 2: 5.04e3, 3: 10.07e3}


@pytest.fixture(scope="module")
def context():
    ctx = api.Context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


@pytest.mark.parametrize("from_lds", [False, True], ids=["registers", "lds"])
@pytest.mark.parametrize("instruction", list(PEAKS))
def test_rates_are_below_the_published_ones(context, instruction, from_lds):
    for random_operands in (False, True):
        rate, ms = context.mfma_ceiling(instruction, from_lds, random_operands, 5.0)
        print("[ceiling]", instruction, from_lds, random_operands, rate, ms, flush=True)
        assert ms > 0 and 0 < rate < PEAKS[instruction]


def test_the_rate_is_that_of_the_operations(context):
    """1024 iterations of 2 * 128^3 operations a wave, twice that on 4-bit values, four waves to a CU."""
    units = torch.cuda.get_device_properties(0).multi_processor_count
    for instruction, times in ((1, 1), (3, 2)):
        rate, ms = context.mfma_ceiling(instruction, False, False, 5.0)
        assert rate * 1e12 * ms * 1e-3 == pytest.approx(times * 2 * 128 ** 3 * 1024 * 4 * units, rel=1e-9)


def test_refusals(context):
    for instruction in (-1, 4):
        with pytest.raises(api.RuyAmdError) as e:
            context.mfma_ceiling(instruction, False, False, 1.0)
        assert e.value.code == S.E_INVALID
    with pytest.raises(api.RuyAmdError):
        context.mfma_ceiling(3, False, False, -1.0)
