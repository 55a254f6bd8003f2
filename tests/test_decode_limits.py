"""The sizes that a decoder's operators take, at their ends, without a GPU."""
import numpy as np
import pytest

import juliavision_b200 as jv
from juliavision_b200 import _lib
from tests.test_decode_host import F16, I32, FakeCtx, arr, refused


def test_rotary_takes_up_to_1024_elements():
    """The plan refuses what no call would take; so does the library, whoever made the plan."""
    plan = jv.rotaryplan(FakeCtx(), 1024)
    with pytest.raises(jv.B200Error) as e:
        jv.rotaryplan(FakeCtx(), 1026)
    assert e.value.code == 17
    x = arr(F16, (2048, 3, 1, 1))
    refused(17, jv.rotary_, jv.RotaryPlan(1026, False, 1.0, plan.freq), x, x, lens=arr(I32, (1,)))
    x = arr(F16, (4098, 3, 1, 1))
    refused(17, jv.rotary_, plan, x, x, lens=arr(I32, (1,)))
    s = _lib.Strided4()
    s.ptr, s.stride[0] = 1 << 20, 1
    assert _lib.lib().b200_rotary_f16(FakeCtx.handle, 2048, 3, 1, 1, s, s, 1 << 20, 1026, 0, 1.0, None, 0, 0, 1 << 20, None) == 17
