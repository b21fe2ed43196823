"""What the decoding operators refuse beside shapes and pointers (no GPU needed)."""
import math

import pytest

from tests.test_decoding_args import P16, S, refused
from oasr_b200 import _lib


def attend(per=4, block=16, scale=0.1):
    return [P16, S, P16, S, P16, P16, P16, P16, P16, P16, None, None, per, block, 8, 2, 4, 2, 1, 64, scale, 0, _lib.DT_BF16, None]


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_fmha_q4_refuses_a_scale_that_is_no_number(scale):
    refused("fmha_q4", attend(scale=scale), _lib.ERR_INVALID)


@pytest.mark.parametrize("per,block", [((1 << 27) - 1, 16), ((1 << 26) - 1, 32)])
def test_fmha_q4_refuses_tables_whose_last_tile_passes_32_bits(per, block):
    """The last position has 31 bits, the end of its tile of 128 has not."""
    refused("fmha_q4", attend(per=per, block=block), _lib.ERR_INVALID)
