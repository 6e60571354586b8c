"""Heads and the cache without a GPU: what is refused beside test_kv_cpu.py's refusals. The pointers are not memory."""
import torch

from test_kv_cpu import cache, heads, refused, sequences, view
from tracea_b200 import ffi


def test_more_heads_of_queries_than_are_counted_in_32_bits_are_refused(lib):
    k = view((3, 2, 64))
    q = view((3, 2 ** 23 + 2, 64))
    refused(ffi.UNSUPPORTED_CONFIG, "heads of q: up to", lib.tracea_kv_append(cache(), sequences(), k.c, k.c, None, heads(q, y=q), 0, 0.0, None, None))
    if not torch.cuda.is_available():            # 2^23 are taken: the call goes on to the device, which is not there
        q = view((3, 2 ** 23, 64))
        assert lib.tracea_kv_append(cache(), sequences(), k.c, k.c, None, heads(q, y=q), 0, 0.0, None, None) == ffi.CUDA_ERROR
