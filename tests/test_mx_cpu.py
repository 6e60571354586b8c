"""The 4-bit microscaled operators and the norms without a GPU: the format's reference against known values, sizes, and everything
the entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

import mxref
from tracea_b200 import ffi, nn, ops


# --------------------------------------------------------------------------------------------------- the reference itself
def test_reference_rounds_ties_to_even_and_saturates():
    x = np.zeros((1, 32))
    x[0, :16] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 7.9, -.25, -2.5, -5, .2, .3, -6]
    codes, scales = mxref.encode(x)
    assert scales[0, 0] == 127
    assert mxref.decode(codes, scales)[0, :16].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -2, -4, 0, .5, -6]


@pytest.mark.parametrize("peak, byte", [(0.0, 0), (4.0, 127), (7.99, 127), (8.0, 128), (3.99, 126), (2.0 ** -125, 0), (2.0 ** -140, 0),
                                        (2.0 ** 127, 252), (np.inf, 255), (np.nan, 255)])
def test_reference_scale_byte(peak, byte):
    assert mxref.encode(np.full((1, 1), peak))[1][0, 0] == byte


def test_reference_layout_round_trip():
    x = np.random.default_rng(0).standard_normal((300, 333))
    codes, scales = mxref.encode(x)
    c, s, rest = mxref.unpack(*mxref.pack(codes, scales), 300, 333)
    assert (c == codes).all() and (s == scales).all() and (rest == 0).all()


# --------------------------------------------------------------------------------------------------- sizes
@pytest.mark.parametrize("m, k", [(1, 1), (1, 32), (128, 128), (129, 129), (7, 4096), (300, 33), (0, 64)])
def test_sizes(lib, m, k):
    assert lib.tracea_mx_data_bytes(m, k) == m * 16 * -(-k // 32)
    assert lib.tracea_mx_scale_bytes(m, k) == -(-m // 128) * -(-k // 128) * 512
    assert lib.tracea_mx_data_bytes(1 << 40, 32) == 0 and lib.tracea_mx_scale_bytes(1, 1 << 40) == 0


# --------------------------------------------------------------------------------------------------- refusals of the C ABI
# Device pointers that nothing ever follows: every call here is refused before a device is touched.
P = 0x10000


def view(shape, stride=None, dtype=ffi.DTYPE_BFLOAT16, ptr=P, device=0):
    if stride is None:
        stride, s = [], 1
        for d in reversed(shape):
            stride.insert(0, s)
            s *= d
    return ffi.View(ptr, shape, stride, dtype, device)


def mx(rows, cols, data=P, scales=P, device=0):
    return ffi.MxMatrix(data, scales, rows, cols, device)


def norm(kind=ffi.NORM_RMS, eps=1e-6, **views):
    n = ffi.Norm(kind, eps)
    n.keep = views
    for k, v in views.items():
        setattr(n, k, ctypes.pointer(v.c))
    return n


def refused(status, text, st):
    assert st == status, (st, ffi.last_error())
    assert text in ffi.last_error(), ffi.last_error()


def opt(v):
    return ctypes.byref(v.c) if v is not None else None


@pytest.mark.parametrize("x, q, status, text", [
    (view((4, 64)), mx(4, 63), ffi.INVALID_PARAMS, "expected [4,64]"),
    (view((4, 64)), mx(5, 64), ffi.INVALID_PARAMS, "expected [4,64]"),
    (view((4, 0)), mx(4, 0), ffi.INVALID_PARAMS, "out of range"),
    (view((4, 64), device=-1), mx(4, 64), ffi.INVALID_PARAMS, "device tensors"),
    (view((4, 64)), mx(4, 64, device=1), ffi.INVALID_PARAMS, "on device 1"),
    (view((4, 64)), mx(4, 64, data=None), ffi.INVALID_PARAMS, "NULL"),
    (view((4, 64)), mx(4, 64, scales=P + 8), ffi.INVALID_PARAMS, "16-byte aligned"),
    (view((4, 64), ptr=None), mx(4, 64), ffi.INVALID_PARAMS, "NULL"),
    (view((4, 64), ptr=P + 1), mx(4, 64), ffi.INVALID_PARAMS, "aligned to its elements"),
    (view((4, 64), dtype=ffi.DTYPE_INT8), mx(4, 64), ffi.UNSUPPORTED_CONFIG, "int8"),
    (view((4, 64, 1)), mx(4, 64), ffi.INVALID_PARAMS, "rank 3"),
    (view((4, 64), (-64, 1)), mx(4, 64), ffi.INVALID_PARAMS, "negative stride"),
])
def test_quantize_refuses(lib, x, q, status, text):
    refused(status, text, lib.tracea_mx_quantize(x.c, ctypes.byref(q), None))
    if status == ffi.INVALID_PARAMS and x.c.device_id == 0:
        refused(status, text, lib.tracea_mx_dequantize(q, opt(x), None)) if "on device" not in text else None


def test_quantize_refuses_null_and_overlapping_outputs(lib):
    refused(ffi.INVALID_PARAMS, "Null pointer", lib.tracea_mx_quantize(view((4, 64)).c, None, None))
    refused(ffi.INVALID_PARAMS, "Null pointer", lib.tracea_mx_dequantize(mx(4, 64), None, None))
    for stride in ((0, 1), (63, 1), (64, 0)):
        refused(ffi.INVALID_PARAMS, "rows overlap", lib.tracea_mx_dequantize(mx(4, 64), opt(view((4, 64), stride)), None))


A, W, C = mx(8, 64), mx(16, 64), view((8, 16))


@pytest.mark.parametrize("a, w, bias, res, c, cq, kind, status, text", [
    (A, mx(16, 65), None, None, C, None, 0, ffi.INVALID_PARAMS, "Inner dimension mismatch"),
    (A, W, None, None, None, None, 0, ffi.INVALID_PARAMS, "exactly one"),
    (A, W, None, None, C, mx(8, 16), 0, ffi.INVALID_PARAMS, "exactly one"),
    (A, W, None, None, view((8, 17)), None, 0, ffi.INVALID_PARAMS, "does not match"),
    (A, W, None, None, None, mx(8, 17), 0, ffi.INVALID_PARAMS, "expected [8,16]"),
    (A, mx(0, 64), None, None, view((8, 0)), None, 0, ffi.INVALID_PARAMS, "no rows"),
    (A, W, None, None, view((8, 16), (1, 8)), None, 0, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (A, W, None, None, view((8, 16), (15, 1)), None, 0, ffi.INVALID_PARAMS, "rows overlap"),
    (A, W, None, None, view((8, 16), dtype=ffi.DTYPE_INT32), None, 0, ffi.UNSUPPORTED_CONFIG, "int32"),
    (A, W, None, None, view((8, 16), device=1), None, 0, ffi.INVALID_PARAMS, "on device 1"),
    (A, W, view((15,), dtype=ffi.DTYPE_FLOAT32), None, C, None, ffi.EPILOGUE_BIAS_ADD, ffi.INVALID_PARAMS, "bias must have shape"),
    (A, W, view((16,), dtype=ffi.DTYPE_FLOAT16), None, C, None, ffi.EPILOGUE_BIAS_ADD, ffi.INVALID_PARAMS, "float32 or"),
    (A, W, view((16,), (2,), dtype=ffi.DTYPE_FLOAT32), None, C, None, ffi.EPILOGUE_BIAS_ADD, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (A, W, view((16,)), None, None, mx(8, 16), ffi.EPILOGUE_BIAS_ADD, ffi.INVALID_PARAMS, "float32 or"),
    (A, W, None, view((8, 15)), C, None, ffi.EPILOGUE_RESIDUAL, ffi.INVALID_PARAMS, "residual shape"),
    (A, W, None, view((8, 16), dtype=ffi.DTYPE_FLOAT32), C, None, ffi.EPILOGUE_RESIDUAL, ffi.INVALID_PARAMS, "dtype of c"),
    (A, W, None, C, None, mx(8, 16), ffi.EPILOGUE_RESIDUAL, ffi.UNSUPPORTED_CONFIG, "residual needs"),
    (A, W, None, None, C, None, 77, ffi.INVALID_PARAMS, "unknown epilogue"),
    (mx(8, 64, device=-1), W, None, None, C, None, 0, ffi.INVALID_PARAMS, "device tensors"),
])
def test_gemm_refuses(lib, a, w, bias, res, c, cq, kind, status, text):
    p = ffi.GemmParams(kind, None)
    q = ctypes.byref(cq) if cq is not None else None
    refused(status, text, lib.tracea_mx_gemm(a, w, opt(bias), opt(res), opt(c), q, p))
    x = view((8, 64), device=a.device_id)
    refused(status, text, lib.tracea_mx_linear(x.c, w, opt(bias), opt(res), opt(c), q, p))


@pytest.mark.parametrize("dtype", [ffi.DTYPE_FLOAT32, ffi.DTYPE_BFLOAT16])
def test_a_bias_between_elements_is_refused(lib, dtype):
    bias = ffi.View(P + 1, (16,), (1,), dtype, 0)
    p = ffi.GemmParams(ffi.EPILOGUE_BIAS_ADD, None)
    refused(ffi.INVALID_PARAMS, "bias is not aligned", lib.tracea_mx_gemm(A, W, opt(bias), None, opt(C), None, p))
    refused(ffi.INVALID_PARAMS, "bias is not aligned", lib.tracea_mx_linear(view((8, 64)).c, W, opt(bias), None, opt(C), None, p))


def test_more_rows_than_can_be_numbered_are_refused(lib):
    x = view(((1 << 31) - 1, 64), device=0)
    y = view(((1 << 31) - 1, 16), device=0)
    p = ffi.GemmParams(0, None)
    refused(ffi.UNSUPPORTED_CONFIG, "rows, at most", lib.tracea_mx_linear(x.c, W, None, None, opt(y), None, p))
    n = norm()
    refused(ffi.UNSUPPORTED_CONFIG, "rows, at most", lib.tracea_block_norm(x.c, ctypes.byref(n), opt(x), None, None))
    refused(ffi.UNSUPPORTED_CONFIG, "rows, at most",
            lib.tracea_block_norm_add(x.c, x.c, ctypes.byref(n), None, 1.0, opt(x), None, None, None, None))


X = view((6, 40))
V = view((40,), dtype=ffi.DTYPE_FLOAT32)


@pytest.mark.parametrize("x, n, y, yq, status, text", [
    (X, norm(), None, None, ffi.INVALID_PARAMS, "exactly one"),
    (X, norm(), X, mx(6, 40), ffi.INVALID_PARAMS, "exactly one"),
    (X, norm(), view((6, 41)), None, ffi.INVALID_PARAMS, "y is [6,41]"),
    (X, norm(), None, mx(6, 41), ffi.INVALID_PARAMS, "expected [6,40]"),
    (X, norm(), view((6, 40), dtype=ffi.DTYPE_FLOAT32), None, ffi.INVALID_PARAMS, "dtype of x"),
    (X, norm(), view((6, 40), (39, 1)), None, ffi.INVALID_PARAMS, "rows overlap"),
    (view((6, 40), (1, 6)), norm(), X, None, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (view((6, 0)), norm(), view((6, 0)), None, ffi.INVALID_PARAMS, "no columns"),
    (view((1, 16385)), norm(), view((1, 16385)), None, ffi.UNSUPPORTED_CONFIG, "at most 16384"),
    (X, norm(kind=7), X, None, ffi.INVALID_PARAMS, "unknown norm"),
    (X, norm(eps=-1.0), X, None, ffi.INVALID_PARAMS, "eps"),
    (X, norm(eps=float("nan")), X, None, ffi.INVALID_PARAMS, "eps"),
    (X, norm(weight=view((39,))), X, None, ffi.INVALID_PARAMS, "weight has 39"),
    (X, norm(weight=view((1, 40))), X, None, ffi.INVALID_PARAMS, "weight must have shape"),
    (X, norm(bias=view((40,), dtype=ffi.DTYPE_FLOAT16)), X, None, ffi.INVALID_PARAMS, "float32 or"),
    (X, norm(bias=view((40,), (2,))), X, None, ffi.UNSUPPORTED_CONFIG, "contiguous"),
    (X, norm(scale=view((40,))), X, None, ffi.INVALID_PARAMS, "scale must have shape"),
    (X, norm(scale=view((4, 40))), X, None, ffi.INVALID_PARAMS, "do not divide"),
    (X, norm(scale=view((2, 40)), shift=view((3, 40))), X, None, ffi.INVALID_PARAMS, "another argument has 2"),
    (X, norm(weight=view((40,), device=1)), X, None, ffi.INVALID_PARAMS, "weight must be on device 0"),
    (view((6, 40), device=-1), norm(), X, None, ffi.INVALID_PARAMS, "device tensors"),
])
def test_block_norm_refuses(lib, x, n, y, yq, status, text):
    q = ctypes.byref(yq) if yq is not None else None
    refused(status, text, lib.tracea_block_norm(x.c, ctypes.byref(n), opt(y), q, None))


@pytest.mark.parametrize("h, n, gate, r, following, y, status, text", [
    (view((5, 40)), norm(), None, X, None, None, ffi.INVALID_PARAMS, "h is [5,40]"),
    (view((6, 40), dtype=ffi.DTYPE_FLOAT32), norm(), None, X, None, None, ffi.INVALID_PARAMS, "dtype of x"),
    (X, norm(), None, view((6, 41)), None, None, ffi.INVALID_PARAMS, "r is [6,41]"),
    (X, norm(), None, None, None, None, ffi.INVALID_PARAMS, "Null pointer"),
    (X, norm(), view((4, 40)), X, None, None, ffi.INVALID_PARAMS, "gate has 4 groups"),
    (X, norm(), view((2, 39)), X, None, None, ffi.INVALID_PARAMS, "gate has 39"),
    (X, norm(), None, X, None, X, ffi.INVALID_PARAMS, "without the norm"),
    (X, norm(), None, X, norm(), None, ffi.INVALID_PARAMS, "exactly one"),
    (X, norm(scale=view((2, 40))), view((3, 40)), X, None, None, ffi.INVALID_PARAMS, "another argument has 2"),
])
def test_block_norm_add_refuses(lib, h, n, gate, r, following, y, status, text):
    f = ctypes.byref(following) if following is not None else None
    refused(status, text, lib.tracea_block_norm_add(h.c, X.c, ctypes.byref(n), opt(gate), 1.0, opt(r), f, opt(y), None, None))


def test_valid_calls_without_a_gpu_fail_loudly(lib):
    if torch.cuda.is_available():
        pytest.skip("there is a GPU: these pointers are not memory")
    p = ffi.GemmParams(0, None)
    for st in (lib.tracea_mx_quantize(view((4, 64)).c, ctypes.byref(mx(4, 64)), None),
               lib.tracea_mx_dequantize(mx(4, 64), opt(view((4, 64))), None),
               lib.tracea_mx_gemm(A, W, None, None, opt(C), None, p),
               lib.tracea_mx_linear(view((8, 64)).c, W, None, None, opt(C), None, p),
               lib.tracea_block_norm(X.c, ctypes.byref(norm()), opt(X), None, None),
               lib.tracea_block_norm_add(X.c, X.c, ctypes.byref(norm()), None, 1.0, opt(X), None, None, None, None)):
        assert st == ffi.CUDA_ERROR and ffi.last_error()


def test_empty_calls_are_no_ops(lib):
    p = ffi.GemmParams(0, None)
    assert lib.tracea_mx_quantize(view((0, 64), ptr=None).c, ctypes.byref(mx(0, 64, None, None)), None) == ffi.SUCCESS
    assert lib.tracea_mx_gemm(mx(0, 64, None, None), W, None, None, opt(view((0, 16), ptr=None)), None, p) == ffi.SUCCESS
    assert lib.tracea_block_norm(view((0, 40), ptr=None).c, ctypes.byref(norm()), opt(view((0, 40), ptr=None)), None, None) == ffi.SUCCESS


# --------------------------------------------------------------------------------------------------- refusals of the Python surface
def tensors(m, k):
    return torch.zeros(m, 16 * -(-k // 32), dtype=torch.uint8), torch.zeros(-(-m // 128), -(-k // 128), 512, dtype=torch.uint8)


def test_python_surface_refuses(lib):
    q = ops.MxTensor(*tensors(8, 64), (8, 64))
    w = ops.MxTensor(*tensors(16, 64), (16, 64))
    with pytest.raises(ffi.TraceaError, match="device tensors"):
        ops.mx_quantize(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="two dimensions"):
        ops.mx_quantize(torch.zeros(4))
    with pytest.raises(ffi.TraceaError, match="device tensors"):
        ops.mx_gemm(q, w)
    with pytest.raises(TypeError, match="MxTensor"):
        ops.mx_gemm(q, torch.zeros(16, 64))
    with pytest.raises(ValueError, match="Inner dimension mismatch"):
        ops.mx_gemm(q, ops.MxTensor(*tensors(16, 96), (16, 96)))
    with pytest.raises(ValueError, match="2D"):
        ops.mx_gemm(torch.zeros(2, 3, 64), w)
    with pytest.raises(ValueError, match="no bias argument"):
        ops.mx_gemm(q, w, None, "bias")
    with pytest.raises(ValueError, match="either dtype or quantize"):
        ops.mx_gemm(q, w, dtype=torch.float32, quantize=True)
    with pytest.raises(TypeError, match="output type"):
        ops.mx_gemm(q, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="Unknown norm"):
        ops.block_norm(torch.zeros(4, 64), kind="batch")
    with pytest.raises(ffi.TraceaError, match="device tensors"):
        ops.block_norm(torch.zeros(4, 64))
    with pytest.raises(ffi.TraceaError, match="device tensors"):
        ops.block_norm_add(torch.zeros(4, 64), torch.zeros(4, 64), following={"quantize": True})
    with pytest.raises(TypeError):
        ops.block_norm_add(torch.zeros(4, 64), torch.zeros(4, 64), following={"gate": None})
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        ops.block_norm([1.0])


@pytest.mark.parametrize("data, scales", [((7, 32), (1, 1, 512)), ((8, 31), (1, 1, 512)), ((8, 32), (1, 1, 511)), ((8, 32), (2, 1, 512))])
def test_a_matrix_whose_tensors_do_not_fit_is_refused(lib, data, scales):
    q = ops.MxTensor(torch.zeros(data, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), (8, 64))
    with pytest.raises(ValueError, match="8 x 64 matrix takes"):
        q.dequantize()
    with pytest.raises(ValueError, match="matrix takes"):
        ops.MxTensor(*(t.int() for t in tensors(8, 64)), (8, 64)).dequantize()


def test_linear_module_refuses_other_epilogues():
    with pytest.raises(NotImplementedError, match="gelu"):
        nn.MxLinear(8, 8, epilogue="gelu")
