"""CPU test that the sizes of the FP4 linear layers' GPU tests reach every form of their kernels."""
from ctypes import byref, c_int32

import pytest

import efm_capi as C
from _fp4_sizes import LINEAR_LONG, SWIGLU_LONG


def _form(m, k, out, swiglu):
    forms, steps = c_int32(), c_int32()
    at = C.load().efm_testing_fp4_linear_form(m, k, out, swiglu, byref(forms), byref(steps))
    return at, forms.value, steps.value


@pytest.mark.parametrize("sizes,swiglu", [(LINEAR_LONG, 0), (SWIGLU_LONG, 1)])
def test_every_form_refills_its_rings(sizes, swiglu):
    """A ring has three places, and a step reads two ahead."""
    seen = set()
    for m, k, out in sizes:
        at, forms, steps = _form(m, k, out, swiglu)
        assert at >= 0 and k % 64 == 32
        if steps >= 8:
            seen.add(at)
    assert len(seen) == forms


def test_sizes_without_a_form():
    assert _form(4, 128, 64, 0)[0] == -1 and _form(5, 120, 64, 0)[0] == -1 and _form(5, 128, 0, 1)[0] == -1
    assert C.load().efm_testing_fp4_linear_form(5, 128, 64, 0, None, None) == -1
