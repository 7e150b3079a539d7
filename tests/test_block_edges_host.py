"""Edges of the transformer-block operators' arguments that need no GPU."""
import ctypes as C
import math

import pytest

from blast3r_b200 import _lib as L
from tests.test_block_host import _desc


@pytest.mark.parametrize('scale', [math.inf, 1e-39, 2.0 ** -101])
def test_c_abi_refuses_scales_out_of_range(scale):
    d = _desc(scale=scale)
    for f in ('b3r_attention_fwd', 'b3r_attention_bwd'):
        with pytest.raises(L.B3RError, match='scale'):
            L.call(f, C.byref(d), None)
