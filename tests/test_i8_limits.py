"""The largest sizes of the 8-bit integer calls that include/minicompiler_hip.h states are refused past them, before
anything reaches a device."""

import pytest

P = 1 << 20  # an aligned address that is never read


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_columns(mc, dtype):
    n = 536870784 + 1
    with pytest.raises(mc.HipError, match="536870784") as e:
        mc.quantize_i8_columns(dtype, P, n, P, P, 1, n)
    assert e.value.code == 1
