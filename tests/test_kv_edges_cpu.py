"""Heads and the cache without a GPU: what is refused beside test_kv_cpu.py's refusals. The pointers are not memory."""
import pytest
import torch

from test_kv_cpu import cache, heads, refused, sequences, view
from tracea_b200 import ffi, ops


def test_more_heads_of_queries_than_are_counted_in_32_bits_are_refused(lib):
    k = view((3, 2, 64))
    q = view((3, 2 ** 23 + 2, 64))
    refused(ffi.UNSUPPORTED_CONFIG, "heads of q: up to", lib.tracea_kv_append(cache(), sequences(), k.c, k.c, None, heads(q, y=q), 0, 0.0, None, None))
    if not torch.cuda.is_available():            # 2^23 are taken: the call goes on to the device, which is not there
        q = view((3, 2 ** 23, 64))
        assert lib.tracea_kv_append(cache(), sequences(), k.c, k.c, None, heads(q, y=q), 0, 0.0, None, None) == ffi.CUDA_ERROR


class Unsettled:
    def __bool__(self):
        raise RuntimeError("neither true nor false")


def test_a_truth_value_that_has_none_is_an_error(lib):
    x, pos, f = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), ops.rotary_frequencies(64)
    c, table = ops.KvCache.empty(4, 2, 64, device="cpu"), torch.zeros(3, 4, dtype=torch.int32)
    for call in (lambda: ops.head_norm_rotate(x, None, pos, f, Unsettled()), lambda: ops.kv_append(c, x, x, table, pos, None, f, Unsettled()),
                 lambda: ops.kv_attention(x.bfloat16(), c, table, pos, causal=Unsettled())):
        with pytest.raises(RuntimeError, match="neither true nor false"):
            call()
    native = ops._native()
    with pytest.raises(RuntimeError, match="neither true nor false"):
        native.conv2d(x, x, None, None, x, Unsettled(), 0, 1, 1, 0, 0, 1, 1, 1)
    with pytest.raises(RuntimeError, match="neither true nor false"):
        native.block_norm(x[:, 0], None, None, None, None, 0, 1e-6, Unsettled())
