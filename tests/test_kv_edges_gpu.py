"""Heads, the cache and attention on a B200 where single values, rows or warps go their own way: waits that run out for some warps of a
block and not for others."""
import pytest
import torch

from test_kv_gpu import check_attention, ints, random_cache, rows
from tracea_b200 import ffi, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stop", [0, 1, 2, 3, 5])
def test_waits_that_run_out_behind_one_silent_warp(stop):
    """One of the four warps that widen the cache's elements leaves: the products wait in vain for its part, the other three for the
    products. All give up as whole warps, the kernel returns, and the next call is right."""
    lib = ffi.load()
    cache = random_cache(40, 2, 64, 128, 5)
    pages, lengths, starts = [list(range(20))], [1200], [0, 1200]
    q = rows(1200, 4, 128, "bf16", 6)
    assert lib.tracea_b200_device_status(0) == 0
    try:
        lib.tracea_b200_test_hooks(400000, 65536 + stop)
        ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts))
        torch.cuda.synchronize()
    finally:
        lib.tracea_b200_test_hooks(0, -1)
    assert lib.tracea_b200_device_status(0) != 0
    assert lib.tracea_b200_device_status(0) == 0
    check_attention(q, cache, pages, lengths, starts)
