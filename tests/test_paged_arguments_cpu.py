"""Arguments of the operators over pages: ranges."""
import math

import pytest

import _paged_oracle as oracle
from ghost_flow_b200 import ops


@pytest.mark.parametrize("scale", [2.0 ** 127, -1e300, math.inf, math.nan])
def test_a_scale_beyond_32_bits_is_refused(scale):
    s = oracle.batch([40, 9], [3, 1], 4, 2, 64, 16)
    with pytest.raises(ValueError, match="scale"):
        ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], scale=scale)
