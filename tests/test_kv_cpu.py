"""Rows of heads, the paged cache and attention over it without a GPU: the 64-bit reference against known values, and everything the
entry points refuse. The pointers are not memory: what is refused is refused before anything is read."""
import ctypes

import pytest
import torch

import kvref
from tracea_b200 import ffi, nn, ops

P = 1 << 20                                      # an aligned address
BF16, F16, F32, I32, I8 = ffi.DTYPE_BFLOAT16, ffi.DTYPE_FLOAT16, ffi.DTYPE_FLOAT32, ffi.DTYPE_INT32, ffi.DTYPE_INT8
_alive = []                                      # views own the arrays that the C structures point to


def view(shape, dtype=BF16, stride=None, ptr=P, device=0):
    if stride is None:
        stride, n = [], 1
        for d in reversed(shape):
            stride.insert(0, n)
            n *= d
    v = ffi.View(ptr, shape, stride, dtype, device)
    _alive.append(v)
    return v


def ref(v):
    return None if v is None else ctypes.byref(v.c)


def heads(x, weight=None, y=None):
    h = ffi.Heads(x.c, ctypes.pointer(weight.c) if weight is not None else None, ctypes.pointer(y.c) if y is not None else None)
    return ctypes.byref(h)


def rotation(pairs=32, interleaved=0, ptr=P):
    return ctypes.byref(ffi.Rotation(ptr, pairs, interleaved))


def cache(pages=10, n=2, size=64, d=64, ptr=P, device=0, k=None):
    return ffi.KvCache(ptr if k is None else k, ptr, ptr, ptr, pages, n, size, d, device)


def sequences(b=3, width=4, starts=None, pages=None, lengths=None):
    pages = pages or view((b, width), I32)
    lengths = lengths or view((b,), I32)
    return ffi.Sequences(pages.c, lengths.c, ctypes.pointer(starts.c) if starts is not None else None)


def refused(status, text, got):
    assert got == status and text in ffi.last_error(), (got, ffi.last_error())


# --------------------------------------------------------------------------------------------------- the reference itself
def test_reference_elements():
    v = torch.tensor([0.0, 448.0, 449.0, 1e9, 17.0, 19.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -0.3, float("nan")])
    got = kvref.e4m3(v)
    assert got[:-1].tolist() == [0, 448, 448, 448, 16, 20, 2.0 ** -9, 0, 2.0 ** -8, -0.3125] and torch.isnan(got[-1])
    x = torch.randn(50000, generator=torch.Generator().manual_seed(0)) * 3
    assert torch.equal(kvref.e4m3(x).float(), x.to(torch.float8_e4m3fn).float())


def test_reference_scales():
    assert kvref.exponent(torch.tensor([0.0, 1e-30, 448.0, 449.0, 896.0, 897.0, 1e30])).tolist() == [-40, -40, 0, 1, 1, 2, 40]


def test_reference_rotation_keeps_lengths():
    x = torch.randn(4, 3, 32, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    f = ops.rotary_frequencies(32)
    for interleaved in (False, True):
        y, _ = kvref.rotate(x, torch.tensor([0, 1, 5, 100000]), f, interleaved)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[0], x[0]) and not torch.allclose(y[1], x[1])


def test_reference_attention_of_one_token_is_its_value():
    k = torch.zeros(1, 1, 16, 16, dtype=torch.float64)
    v = torch.arange(16.0).repeat(16, 1).view(1, 1, 16, 16)
    s = torch.full((1, 1), 128, dtype=torch.uint8)
    y, _ = kvref.attention(torch.ones(1, 1, 16), k, v, s, s, [[0]], [1], None, 1.0, True, 0, 0)
    assert y[0, 0].tolist() == [2.0 * i for i in range(16)]


# --------------------------------------------------------------------------------------------------- refusals: norm and rotation
X, Y, POS = view((5, 2, 64)), view((5, 2, 64)), view((5,), I32)


@pytest.mark.parametrize("q, k, kind, eps, rot, pos, status, text", [
    (None, None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "neither queries nor keys"),
    (heads(X), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "no output"),
    (heads(view((5, 128)), y=Y), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "[tokens, heads, columns]"),
    (heads(view((5, 2, 64), device=-1), y=Y), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "device tensors"),
    (heads(X, y=view((5, 2, 64), device=1)), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "device 1"),
    (heads(X, y=view((5, 3, 64))), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "heads"),
    (heads(X, y=view((5, 2, 64), F32)), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "dtype"),
    (heads(X, y=view((5, 2, 64), stride=(64, 64, 1))), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "overlap"),
    (heads(view((5, 2, 64), I8), y=view((5, 2, 64), I8)), None, 1, 1e-6, None, None, ffi.UNSUPPORTED_CONFIG, "int8"),
    (heads(view((5, 2, 63)), y=view((5, 2, 63))), None, 1, 1e-6, None, None, ffi.UNSUPPORTED_CONFIG, "even number"),
    (heads(view((5, 2, 258)), y=view((5, 2, 258))), None, 1, 1e-6, None, None, ffi.UNSUPPORTED_CONFIG, "even number"),
    (heads(view((5, 2, 64), stride=(256, 128, 2)), y=Y), None, 1, 1e-6, None, None, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (heads(view((5, 2, 64), ptr=P + 1), y=Y), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "aligned"),
    (heads(X, view((32,), F32), Y), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "weight must have shape [64]"),
    (heads(X, view((64,), F16), Y), None, 1, 1e-6, None, None, ffi.INVALID_PARAMS, "float32 or have the rows' dtype"),
    (heads(X, y=Y), heads(view((6, 2, 64)), y=view((6, 2, 64))), 1, 1e-6, None, None, ffi.INVALID_PARAMS, "tokens"),
    (heads(X, y=Y), None, 2, 1e-6, None, None, ffi.UNSUPPORTED_CONFIG, "none or rms"),
    (heads(X, y=Y), None, 1, -1.0, None, None, ffi.INVALID_PARAMS, "eps"),
    (heads(X, y=Y), None, 1, float("nan"), None, None, ffi.INVALID_PARAMS, "eps"),
    (heads(X, y=Y), None, 0, 0.0, rotation(33), POS, ffi.INVALID_PARAMS, "33 pairs"),
    (heads(X, y=Y), None, 0, 0.0, rotation(32, ptr=None), POS, ffi.INVALID_PARAMS, "no frequencies"),
    (heads(X, y=Y), None, 0, 0.0, rotation(32, ptr=P + 4), POS, ffi.INVALID_PARAMS, "aligned"),
    (heads(X, y=Y), None, 0, 0.0, rotation(), None, ffi.INVALID_PARAMS, "takes positions"),
    (heads(X, y=Y), None, 0, 0.0, rotation(), view((4,), I32), ffi.INVALID_PARAMS, "positions must have shape [5]"),
    (heads(X, y=Y), None, 0, 0.0, rotation(), view((5,), F32), ffi.INVALID_PARAMS, "int32"),
    (heads(X, y=Y), None, 0, 0.0, rotation(), view((5,), I32, stride=(2,)), ffi.UNSUPPORTED_CONFIG, "contiguous"),
])
def test_head_norm_rotate_refuses(lib, q, k, kind, eps, rot, pos, status, text):
    refused(status, text, lib.tracea_head_norm_rotate(q, k, kind, eps, rot, ref(pos), None))


# --------------------------------------------------------------------------------------------------- refusals: the cache
K3 = view((3, 2, 64))


@pytest.mark.parametrize("c, s, k, v, q, status, text", [
    (cache(device=-1), sequences(), K3, K3, None, ffi.INVALID_PARAMS, "device memory"),
    (cache(size=48), sequences(), K3, K3, None, ffi.UNSUPPORTED_CONFIG, "pages of 48 tokens"),
    (cache(size=256), sequences(), K3, K3, None, ffi.UNSUPPORTED_CONFIG, "pages of 256 tokens"),
    (cache(d=72), sequences(), view((3, 2, 72)), view((3, 2, 72)), None, ffi.UNSUPPORTED_CONFIG, "multiple of 16"),
    (cache(d=144), sequences(), view((3, 2, 144)), view((3, 2, 144)), None, ffi.UNSUPPORTED_CONFIG, "up to 128"),
    (cache(n=0), sequences(), K3, K3, None, ffi.INVALID_PARAMS, "out of range"),
    (cache(ptr=None), sequences(), K3, K3, None, ffi.INVALID_PARAMS, "NULL pointer"),
    (cache(k=P + 8), sequences(), K3, K3, None, ffi.INVALID_PARAMS, "16-byte aligned"),
    (cache(), sequences(), view((3, 4, 64)), view((3, 4, 64)), None, ffi.INVALID_PARAMS, "the cache 2 of 64"),
    (cache(), sequences(), K3, view((3, 2, 64), F16), None, ffi.INVALID_PARAMS, "dtype of k"),
    (cache(), sequences(), K3, view((4, 2, 64)), None, ffi.INVALID_PARAMS, "v has 4 tokens"),
    (cache(), sequences(b=4), K3, K3, None, ffi.INVALID_PARAMS, "3 rows of 4 sequences"),
    (cache(), sequences(starts=view((3,), I32)), K3, K3, None, ffi.INVALID_PARAMS, "starts must have shape [4]"),
    (cache(), sequences(starts=view((4,), F32)), K3, K3, None, ffi.INVALID_PARAMS, "starts must be int32"),
    (cache(), sequences(lengths=view((2,), I32)), K3, K3, None, ffi.INVALID_PARAMS, "lengths must have shape [3]"),
    (cache(), sequences(lengths=view((3,), I32, device=-1)), K3, K3, None, ffi.INVALID_PARAMS, "lengths must be on device 0"),
    (cache(), sequences(pages=view((3, 4), F32)), K3, K3, None, ffi.INVALID_PARAMS, "pages must be int32"),
    (cache(), sequences(pages=view((3,), I32)), K3, K3, None, ffi.INVALID_PARAMS, "[sequences, pages]"),
    (cache(), sequences(pages=view((3, 4), I32, stride=(1, 3))), K3, K3, None, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (cache(), sequences(pages=view((3, 4), I32, ptr=P + 2)), K3, K3, None, ffi.INVALID_PARAMS, "aligned"),
    (cache(), sequences(), K3, K3, heads(view((3, 3, 64)), y=view((3, 3, 64))), ffi.INVALID_PARAMS, "no multiple"),
    (cache(), sequences(), K3, K3, heads(view((3, 4, 64))), ffi.INVALID_PARAMS, "q has no output"),
    (cache(), sequences(), K3, K3, heads(view((3, 4, 64), F16), y=view((3, 4, 64), F16)), ffi.INVALID_PARAMS, "dtype of k"),
])
def test_kv_append_refuses(lib, c, s, k, v, q, status, text):
    refused(status, text, lib.tracea_kv_append(c, s, k.c, v.c, None, q, 0, 0.0, None, None))


Q3, PARAMS = view((3, 4, 64)), ffi.KvAttentionParams(0.125, 1, 0, None)


@pytest.mark.parametrize("q, c, s, out, params, status, text", [
    (Q3, cache(), sequences(), None, PARAMS, ffi.INVALID_PARAMS, "Null pointer"),
    (view((3, 4, 64), F32), cache(), sequences(), view((3, 4, 64), F32), PARAMS, ffi.UNSUPPORTED_CONFIG, "float16 or bfloat16"),
    (Q3, cache(), sequences(), view((3, 4, 64), F16), PARAMS, ffi.INVALID_PARAMS, "dtype of q"),
    (Q3, cache(), sequences(), view((3, 2, 64)), PARAMS, ffi.INVALID_PARAMS, "out has 2 heads"),
    (Q3, cache(), sequences(), view((3, 4, 64), stride=(0, 64, 1)), PARAMS, ffi.INVALID_PARAMS, "overlap"),
    (view((3, 3, 64)), cache(), sequences(), view((3, 3, 64)), PARAMS, ffi.INVALID_PARAMS, "the cache 2 of 64"),
    (view((3, 4, 48)), cache(), sequences(), view((3, 4, 48)), PARAMS, ffi.INVALID_PARAMS, "the cache 2 of 64"),
    (Q3, cache(d=80), sequences(), Q3, PARAMS, ffi.INVALID_PARAMS, "the cache 2 of 80"),
    (Q3, cache(), sequences(), Q3, ffi.KvAttentionParams(float("inf"), 1, 0, None), ffi.INVALID_PARAMS, "finite"),
    (Q3, cache(), sequences(), Q3, ffi.KvAttentionParams(float("nan"), 1, 0, None), ffi.INVALID_PARAMS, "finite"),
    (Q3, cache(), sequences(), Q3, ffi.KvAttentionParams(1.0, 1, 1 << 31, None), ffi.INVALID_PARAMS, "window"),
    (view((4, 4, 64)), cache(), sequences(), view((4, 4, 64)), PARAMS, ffi.INVALID_PARAMS, "4 rows of 3 sequences"),
])
def test_kv_attention_refuses(lib, q, c, s, out, params, status, text):
    refused(status, text, lib.tracea_kv_attention(q.c, c, s, ref(out), params))


def test_empty_calls_are_no_ops(lib):
    e, none = view((0, 2, 64), ptr=None), view((0,), I32, ptr=None)
    s = sequences(b=0, pages=view((0, 4), I32, ptr=None), lengths=none)
    assert lib.tracea_head_norm_rotate(heads(e, y=e), None, 1, 0.0, rotation(), ref(none), None) == ffi.SUCCESS
    assert lib.tracea_kv_append(cache(), s, e.c, e.c, None, None, 0, 0.0, None, None) == ffi.SUCCESS
    assert lib.tracea_kv_attention(e.c, cache(), s, ref(e), PARAMS) == ffi.SUCCESS


def test_valid_calls_without_a_gpu_fail_loudly(lib):
    if torch.cuda.is_available():
        pytest.skip("there is a GPU: these pointers are not memory")
    for st in (lib.tracea_head_norm_rotate(heads(X, y=Y), None, 1, 0.0, rotation(), ref(POS), None),
               lib.tracea_kv_append(cache(), sequences(), K3.c, K3.c, None, heads(Q3, y=Q3), 0, 0.0, rotation(), None),
               lib.tracea_kv_attention(Q3.c, cache(), sequences(), ref(Q3), PARAMS)):
        assert st == ffi.CUDA_ERROR and ffi.last_error()


# --------------------------------------------------------------------------------------------------- the Python surface
def test_python_surface_refuses(lib):
    c = ops.KvCache.empty(4, 2, 64, device="cpu")
    k, table, lengths = torch.zeros(3, 2, 64), torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ffi.TraceaError, match="device tensors"):
        ops.head_norm_rotate(k, None)
    with pytest.raises(ValueError, match="neither q nor k"):
        ops.head_norm_rotate(None, None)
    with pytest.raises(ValueError, match="three dimensions"):
        ops.head_norm_rotate(torch.zeros(3, 64), None)
    with pytest.raises(ValueError, match="Unknown norm"):
        ops.head_norm_rotate(k, None, kind="batch")
    with pytest.raises(ValueError, match="float64 vector"):
        ops.head_norm_rotate(k, None, lengths, torch.ones(32))
    with pytest.raises(ValueError, match="float64 vector"):
        ops.head_norm_rotate(k, None, lengths, torch.ones(2, 16, dtype=torch.float64))
    with pytest.raises(ValueError, match="even number"):
        ops.rotary_frequencies(63)
    with pytest.raises(ffi.TraceaError, match="device memory"):
        ops.kv_append(c, k, k, table, lengths)
    with pytest.raises(ffi.TraceaError, match="device memory"):
        ops.kv_attention(k.bfloat16(), c, table, lengths)
    with pytest.raises(ValueError, match="window"):
        ops.kv_attention(k.bfloat16(), c, table, lengths, window=-1)
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        ops.kv_append(c, k, k, [[0]], lengths)


@pytest.mark.parametrize("change", [dict(k=lambda t: t.view(torch.uint8)), dict(v=lambda t: t[:2]), dict(k_scales=lambda t: t.int()),
                                    dict(v_scales=lambda t: t[:, :1]), dict(k=lambda t: t.transpose(1, 2)), dict(v_scales=lambda t: t.t())])
def test_a_cache_whose_tensors_do_not_fit_is_refused(lib, change):
    c = ops.KvCache.empty(4, 2, 64, device="cpu")
    for name, f in change.items():
        setattr(c, name, f(getattr(c, name)))
    with pytest.raises(ValueError, match="a cache is contiguous tensors"):
        ops.kv_append(c, torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32))


def test_cache_and_module_refuse():
    with pytest.raises(ValueError, match="page_size"):
        ops.KvCache.empty(4, 2, 64, 48, "cpu")
    with pytest.raises(ValueError, match="head_dim"):
        ops.KvCache.empty(4, 2, 72, 64, "cpu")
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        nn.MxAttention(256, 4, 3)
    with pytest.raises(ValueError, match="give head_dim"):
        nn.MxAttention(100, 3)
    with pytest.raises(ValueError, match="multiple of 16"):
        nn.MxAttention(160, 4)
    with pytest.raises(ValueError, match="multiple of 16"):
        nn.MxAttention(1024, 4)


def test_module_keeps_its_frequencies_in_64_bits():
    block = nn.MxAttention(128, 2).to(torch.bfloat16)
    assert block._frequencies.dtype == torch.float64 and torch.equal(block._frequencies, ops.rotary_frequencies(64))
    assert "_frequencies" not in block.state_dict() and block.q_weight.dtype == torch.bfloat16
    c = block.cache(5, 32)
    assert c.k.shape == (5, 2, 32, 64) and c.page_size == 32 and c.device == torch.device("cpu") and "5 pages of 32" in repr(c)
