"""CPU tests of the filtered sampler's argument checks. No call has a row, so that none would launch."""
import pytest

import efm_capi as C

P = 4096   # an address that is never read


def _rc(t):
    return C.load().efm_sampler_filtered(0, 100, P, C.EFM_DTYPE_F32, 0, t, 0, 1.0, 0.0, P, P, None, 0, None)


@pytest.mark.parametrize("t", [1.1e36, 1e37, 1e38, 3.4e38])
def test_temperatures_at_which_distances_overflow(t):
    """Past 1e36 logits whose distance is no finite fp32 number would have mass."""
    assert _rc(t) == C.EFM_ERR_INVALID_ARGUMENT
    assert b"temperature" in C.load().efm_last_error()


@pytest.mark.parametrize("t", [1e-6, 1.0, 1e20, 1e36])
def test_temperatures(t):
    assert _rc(t) == C.EFM_OK
