"""What the decoding operators refuse beside shapes and pointers (no GPU needed)."""
import math

import pytest

from tests.test_decoding_args import P16, S, refused
from oasr_b200 import _lib


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_fmha_q4_refuses_a_scale_that_is_no_number(scale):
    refused("fmha_q4", [P16, S, P16, S, P16, P16, P16, P16, P16, P16, None, None, 4, 16, 8, 2, 4, 2, 1, 64, scale, 0, _lib.DT_BF16, None], _lib.ERR_INVALID)
