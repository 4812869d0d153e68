"""Refusals of the batched attention operators beside those of test_kv8_cpu.py, before any device work."""
import math

import pytest

from roofline_decoding_b200 import _lib
from test_kv8_cpu import FAKE, batch, cache, heads


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_a_scale_that_is_no_number_is_refused(scale):
    """(1e39 leaves fp32.) One kernel made it NaN, the other a uniform softmax."""
    def call(scale, rows):
        return _lib.load().w4_kv8_attention(cache(), batch(rows=rows), heads(), heads(), 1, scale,
                                            FAKE, 1 << 30, None)

    assert call(scale, 5) == _lib.W4_ERR_INVALID_ARG and call(scale, 0) == _lib.W4_ERR_INVALID_ARG
    assert call(-3e38, 0) == _lib.W4_OK
