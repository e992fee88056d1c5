"""Factors of sh_rope_steps whose reciprocal is no number: refused without a GPU, as its other arguments are."""
from __future__ import annotations

import pytest

from softhier_mlir_amd import shops

ONE = 1 << 20                                   # never dereferenced: the checks fail first


@pytest.mark.parametrize("scaling", [shops.SH_ROPE_LINEAR, shops.SH_ROPE_BANDS, shops.SH_ROPE_RAMP])
@pytest.mark.parametrize("factor", [5e-324, 1e-310, 5.5e-309])
def test_factors_without_a_reciprocal(lib, factor, scaling):
    assert 1.0 / factor == float("inf")         # frequencies would be infinite, steps no numbers
    assert lib.sh_rope_steps(ONE, 64, 1e4, scaling, factor, 1.0, 4.0, 8192) == -1
    code, text = shops.last_error()
    assert code == -1 and "[sh_rope_steps]" in text
