"""Empty calls of the 4-bit operators and the norms that are allowed, without a GPU."""
import ctypes

import pytest

from tracea_b200 import ffi
from test_mx_cpu import norm, opt, refused, view


@pytest.mark.parametrize("groups", [0, 1, 4])
def test_a_batch_of_no_samples_has_no_conditioning_either(lib, groups):
    """Every number of groups divides no rows, 0 among them."""
    x, g = view((0, 40), ptr=None), view((groups, 40), ptr=None if groups == 0 else 0x10000)
    n = norm(scale=g, shift=g)
    assert lib.tracea_block_norm(x.c, ctypes.byref(n), opt(x), None, None) == ffi.SUCCESS, ffi.last_error()
    assert lib.tracea_block_norm_add(x.c, x.c, ctypes.byref(norm()), opt(g), 1.0, opt(x), ctypes.byref(n), opt(x), None, None) == ffi.SUCCESS
    refused(ffi.INVALID_PARAMS, "gate has 39", lib.tracea_block_norm_add(x.c, x.c, ctypes.byref(norm()), opt(view((groups, 39))), 1.0, opt(x),
                                                                         None, None, None, None))
    some = view((6, 40))                                       # rows without any group are refused as before
    if groups != 1:
        refused(ffi.INVALID_PARAMS, "gate ", lib.tracea_block_norm_add(some.c, some.c, ctypes.byref(norm()), opt(g), 1.0, opt(some), None, None,
                                                                       None, None))
