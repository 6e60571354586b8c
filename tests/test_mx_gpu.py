"""4-bit microscaled matrices on a B200: conversions to the bit, products against 64-bit ones.

Tolerance of a product, per element: values of the format and their products are exact in fp32, and so only sums round. K terms
summed in fp32 in any order, even with each addition truncated, are off by at most K 2^-23 sum|a w|; bias, residual and activation
add 4 2^-23 of their terms' sizes. fp32 activations (expf, tanhf, a division) are good to 2^-20 of the value; 16-bit outputs use
exp to 2^-16 (its argument is rounded, which costs |x| 2^-23, |x| < 90) and tanh to 2^-10.9, half of which times |x| reaches a GELU.
The output's own rounding is half a step, finfo.eps / 2.
"""
import ctypes
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import mxref
from tracea_b200 import ffi, nn, ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEFAULT_CONFIG = not any(k.startswith("TRACEA_B200_") for k in os.environ)


def status_ok():
    torch.cuda.synchronize()
    assert ffi.load().tracea_b200_device_status(0) == 0


def matrix(m, k, seed, size=1.0):
    """Random codes and scales as an MxTensor whose scale bytes of rows past the last one are NaN, and its values."""
    rng = np.random.default_rng([seed, m, k])
    codes, scales = mxref.encode(rng.standard_normal((m, k)) * size * np.exp(rng.standard_normal((1, k))))
    data, s = mxref.pack(codes, scales)
    t = ops.MxTensor(torch.from_numpy(data).cuda(), torch.from_numpy(s).cuda(), (m, k))
    return t, torch.from_numpy(mxref.decode(codes, scales)[:, :k]).cuda()


def bytes_of(q):
    return q.data.cpu().numpy(), q.scales.cpu().numpy()


def assert_is_encoding(q, x):
    """The MxTensor is x's encoding, padding included."""
    m, k = x.shape
    codes, scales, rest = mxref.unpack(*bytes_of(q), m, k)
    want_codes, want_scales = mxref.encode(x)
    assert (scales == want_scales).all()
    assert (codes == want_codes).all()
    assert (rest == 0).all()


# --------------------------------------------------------------------------------------------------- conversions
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, k", [(1, 1), (1, 32), (3, 33), (127, 128), (128, 129), (129, 31), (5, 256), (200, 1000), (33, 4104), (257, 8)])
def test_quantize_is_its_definition(m, k, dtype):
    rng = np.random.default_rng([m, k])
    x = torch.from_numpy(rng.standard_normal((m, k)) * np.exp(2 * rng.standard_normal((m, 1)))).to(DT[dtype])
    q = ops.mx_quantize(x.cuda())
    status_ok()
    assert q.shape == (m, k)
    assert_is_encoding(q, x.double().numpy())
    assert torch.equal(q.dequantize(torch.float32).double().cpu(), torch.from_numpy(mxref.values(x.double().numpy())))


def test_quantize_every_bf16_and_f16_value():
    for dtype in (torch.bfloat16, torch.float16):
        bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
        alone = torch.zeros(65536, 32, dtype=dtype)
        alone[:, 7] = bits
        for x in (bits.view(2048, 32), alone):
            assert_is_encoding(ops.mx_quantize(x.cuda()), x.double().numpy())


def test_quantize_ties_and_fp32_extremes():
    rng = np.random.default_rng(5)
    e = rng.integers(-149, 126, (4000, 1)).astype(np.float64)
    grid = rng.integers(-28, 29, (4000, 32)) / 4.0        # multiples of a quarter: every border between codes among them
    x = (np.exp2(e) * grid).astype(np.float32)
    x[::7, 3] = np.inf
    x[::11, 5] = np.nan
    x[5] = 0
    x[6] = -0.0
    x[8] = np.finfo(np.float32).max
    assert_is_encoding(ops.mx_quantize(torch.from_numpy(x).cuda()), x)


@pytest.mark.parametrize("layout", ["wide rows", "offset", "transposed", "every second", "one row broadcast"])
def test_quantize_strided_inputs(layout):
    base = torch.randn(300, 400, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    x = {"wide rows": base[:, :96], "offset": base[1:, 3:99], "transposed": base.t()[:97, :130], "every second": base[::2, ::2],
         "one row broadcast": base[:1, :100].expand(140, 100)}[layout]
    assert_is_encoding(ops.mx_quantize(x), x.double().cpu().numpy())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dequantize_every_code_under_every_scale(dtype):
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    q = ops.MxTensor(*(torch.from_numpy(t).cuda() for t in mxref.pack(codes, scales)), (256, 32))
    want = torch.from_numpy(mxref.decode(codes, scales)).to(DT[dtype])     # exact in fp32 and bf16, one rounding in fp16
    assert torch.equal(torch.nan_to_num(q.dequantize(DT[dtype]).cpu(), nan=123.0), torch.nan_to_num(want, nan=123.0))


@pytest.mark.parametrize("m, k", [(1, 1), (130, 200), (40, 33)])
def test_dequantize_into_a_view_leaves_the_rest(m, k):
    q, want = matrix(m, k, 3)
    for make in (lambda: torch.full((m, k + 7), 9.0, device="cuda")[:, 5:5 + k], lambda: torch.full((k, m + 1), 9.0, device="cuda")[:, :m].t()):
        out = make()
        whole = out._base
        v = ffi.View(out.data_ptr(), out.shape, out.stride(), ffi.DTYPE_FLOAT32, 0)
        mx = ffi.MxMatrix(q.data.data_ptr(), q.scales.data_ptr(), m, k, 0)
        assert ffi.load().tracea_mx_dequantize(mx, ctypes.byref(v.c), None) == ffi.SUCCESS
        torch.cuda.synchronize()
        assert torch.equal(out.double(), want)
        assert (whole == 9.0).sum().item() == whole.numel() - m * k + (want == 9.0).sum().item()


# --------------------------------------------------------------------------------------------------- products
def split(epilogue):
    parts = (epilogue or "").split("+")
    return "bias" in parts, "residual" in parts, next((p for p in parts if p in ("relu", "silu", "gelu")), "")


def reference(a, w, epilogue, bias, residual, out):
    """(result, bound on |error|) in 64 bits, on the GPU."""
    use_b, use_r, act = split(epilogue)
    k = a.shape[1]
    y, size = a @ w.t(), a.abs() @ w.abs().t()
    err = (k * 2.0 ** -23) * size
    if use_b:
        y, err = y + bias.double(), err + 2.0 ** -23 * bias.double().abs()
    if use_r:
        y, err = y + residual.double(), err + 2.0 ** -23 * residual.double().abs()
    err = err + 4 * 2.0 ** -23 * y.abs()
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "silu":
        z, y = y, y * torch.sigmoid(y)
        err = 1.1 * err + (2.0 ** -20 if out == torch.float32 else 2.0 ** -16) * y.abs() + 1e-37
    elif act == "gelu":
        z, y = y, y * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3))
        err = 1.13 * err + (2.0 ** -20 if out == torch.float32 else 2.0 ** -11.9) * z.abs()
    return y, err


def assert_close(got, y, err):
    f = torch.finfo(got.dtype)
    err = err + (f.eps / 2) * y.abs() + f.smallest_normal * f.eps     # ... below the normal range, a fixed half step
    bad = (got.double() - y).abs() > err
    assert not bad.any(), "%d of %d, worst %g of the bound" % (bad.sum(), bad.numel(), ((got.double() - y).abs() / err).max())


EPILOGUES = [None, "bias", "relu", "bias+silu", "gelu", "bias+residual", "bias+residual+relu"]
# one token to several tiles of every form, K of one block to many k-steps, nothing a multiple of anything
SHAPES = [(1, 1, 1), (1, 128, 64), (1, 1000, 2048), (3, 50, 33), (17, 200, 777), (32, 129, 4096), (64, 1000, 2048), (65, 64, 256),
          (128, 300, 5000), (129, 130, 100), (200, 1030, 64), (300, 77, 1111), (1000, 1000, 300), (2100, 520, 260), (1300, 2600, 513)]


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", SHAPES)
def test_product(m, n, k, out):
    a, av = matrix(m, k, 1)
    w, wv = matrix(n, k, 2, k ** -0.5)
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    bias = torch.randn(n, generator=gen, device="cuda")
    res = torch.randn(m, n, generator=gen, device="cuda").to(DT[out])
    for e in EPILOGUES:
        use_b, use_r, _ = split(e)
        b = None if not use_b else (bias if m % 2 else bias.to(DT[out]))
        got = ops.mx_gemm(a, w, b, e, res if use_r else None, dtype=DT[out])
        assert got.shape == (m, n) and got.dtype == DT[out]
        assert_close(got, *reference(av, wv, e, b, res, DT[out]))
    status_ok()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", [(1, 300, 64), (1, 4096, 4096), (2, 77, 1001), (8, 1000, 2048), (16, 130, 260), (20, 500, 600), (150, 260, 500)])
def test_product_of_an_input_that_the_call_quantizes(m, n, k, dtype):
    w, wv = matrix(n, k, 2, k ** -0.5)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)).to(DT[dtype])
    xv = torch.from_numpy(mxref.values(x.double().numpy())).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    res = torch.randn(m, n).to(DT[dtype]).cuda()
    wide = torch.full((m, k + 3), float("nan"), dtype=DT[dtype], device="cuda")
    wide[:, 1:k + 1] = x.cuda()
    for data in (x.cuda(), wide[:, 1:k + 1], x.t().contiguous().cuda().t()):
        for e in ("bias+silu", "bias+residual", None):
            assert_close(ops.mx_gemm(data, w, bias if e else None, e, res if e == "bias+residual" else None),
                         *reference(xv, wv, e, bias, res, DT[dtype]))
    got = ops.mx_gemm(x.cuda(), w, dtype=torch.float32)
    assert_close(got, *reference(xv, wv, None, None, None, torch.float32))
    q = ops.mx_gemm(x.cuda(), w, bias, "bias", quantize=True)
    assert_quantized(q, *reference(xv, wv, "bias", bias, None, torch.float32))
    status_ok()


def assert_quantized(q, y, err):
    """Each value lies between the encodings of y - err and y + err, under the block's scale; blocks whose largest value may be on
    either side of a power of two may have either scale."""
    y, err = y.cpu().numpy(), err.cpu().numpy()
    m, n = y.shape
    codes, scales, rest = mxref.unpack(*bytes_of(q), m, n)
    assert (rest == 0).all()
    assert (codes[:, n:] & 7 == 0).all()
    pad = lambda t: np.pad(t, ((0, 0), (0, codes.shape[1] - n))).reshape(m, -1, 32)
    peak, slack = np.abs(pad(y)).max(-1), pad(err).max(-1)
    of = lambda p: np.clip(np.where(p > 0, np.frexp(p)[1] - 3, -127), -127, 125) + 127
    assert ((scales >= of(np.maximum(peak - slack, 0))) & (scales <= of(peak + slack))).all()
    s = np.exp2(scales.astype(np.float64) - 127)[..., None]

    def under(t):
        v = np.minimum(np.abs(t) / s, 6.0)
        step = np.where(v < 2, .5, np.where(v < 4, 1.0, 2.0))
        return np.sign(t) * np.minimum(np.round(v / step) * step, 6.0) * s

    got = pad(mxref.decode(codes, scales)[:, :n])
    assert ((got >= under(pad(y - err))) & (got <= under(pad(y + err)))).all()


@pytest.mark.parametrize("epilogue", [None, "bias", "relu", "bias+silu", "gelu"])
@pytest.mark.parametrize("m, n, k", [(1, 1, 32), (1, 130, 64), (5, 4096, 300), (64, 33, 2048), (130, 40, 100), (300, 161, 64), (600, 1000, 513), (1300, 2600, 256)])
def test_quantized_output(m, n, k, epilogue):
    a, av = matrix(m, k, 4)
    w, wv = matrix(n, k, 5, k ** -0.5)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    use_b, _, act = split(epilogue)
    q = ops.mx_gemm(a, w, bias if use_b else None, epilogue, quantize=True)
    status_ok()
    # the activations of a quantised output are those of 16-bit ones
    assert_quantized(q, *reference(av, wv, epilogue, bias, None, torch.bfloat16))


FORMS = """
import sys
sys.path[:0] = [%r, %r]
import torch
import test_mx_gpu as t
for m, n, k in ((1, 1, 1), (129, 193, 100), (300, 400, 1111), (700, 513, 2304), (2000, 1000, 256)):
    for out in ("f32", "bf16"):
        t.test_product(m, n, k, out)
    for e in (None, "bias+silu"):
        t.test_quantized_output(m, n, k, e)
print("forms ok")
"""


@pytest.mark.parametrize("columns", [64, 128, 192, 256])
def test_every_tile_width_is_right_for_every_size(columns):
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, TRACEA_B200_MX_BN=str(columns), TRACEA_B200_MX_TOKENS="0")
    r = subprocess.run([sys.executable, "-c", FORMS % (here, os.path.dirname(here))], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "forms ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("m, n, k", [(1, 70, 100), (5, 1000, 2048), (40, 33, 64), (300, 161, 300), (700, 1001, 513), (2500, 2500, 256)])
def test_scales_of_rows_past_the_end_reach_no_bit(m, n, k):
    """0, NaN and random bytes there: the same results, where neighbouring columns share a reciprocal above all."""
    a, _ = matrix(m, k, 20)
    w, _ = matrix(n, k, 21, 0.3)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    gen = torch.Generator(device="cuda").manual_seed(2)

    def refilled(q, fill):
        rows = torch.arange(q.scales.shape[0] * 128, device="cuda").view(-1, 4, 32).permute(0, 2, 1)     # row of (tile, lane, word)
        past = (rows >= q.shape[0])[:, None, :, :, None].expand(-1, q.scales.shape[1], -1, -1, 4).reshape(q.scales.shape)
        s = q.scales.clone()
        other = torch.randint(0, 256, s.shape, generator=gen, device="cuda", dtype=torch.uint8) if fill is None else torch.full_like(s, fill)
        s[past] = other[past]
        return ops.MxTensor(q.data, s, q.shape)

    for e in ("bias+silu", "bias", "gelu"):
        b = bias if "bias" in e else None
        for out in (torch.bfloat16, torch.float32):
            first = ops.mx_gemm(a, w, b, e, dtype=out)
            assert not first.isnan().any()
            for fill in (0, None, 130):
                assert torch.equal(ops.mx_gemm(refilled(a, fill), refilled(w, fill), b, e, dtype=out), first)
        q = ops.mx_gemm(a, w, b, e, quantize=True)
        for fill in (0, None):
            q2 = ops.mx_gemm(refilled(a, fill), refilled(w, fill), b, e, quantize=True)
            assert torch.equal(q2.data, q.data) and torch.equal(q2.dequantize(torch.float32), q.dequantize(torch.float32))
    status_ok()


def test_a_nan_block_reaches_its_row_and_nothing_else():
    for m, n, k in ((3, 200, 300), (300, 200, 300)):
        a, av = matrix(m, k, 6)
        w, wv = matrix(n, k, 7)
        clean = ops.mx_gemm(a, w, dtype=torch.float32)
        x = av.float()
        x[1, 40], x[2, 299] = float("nan"), float("-inf")
        got = ops.mx_gemm(ops.mx_quantize(x), w, dtype=torch.float32)
        assert got[1].isnan().all() and got[2].isnan().all()
        rest = torch.tensor([i for i in range(m) if i not in (1, 2)], device="cuda")
        assert torch.equal(got[rest], clean[rest])
        y = wv.float()
        y[5, 0] = float("inf")
        got = ops.mx_gemm(a, ops.mx_quantize(y), dtype=torch.float32)
        assert got[:, 5].isnan().all()
        cols = torch.tensor([i for i in range(n) if i != 5], device="cuda")
        assert torch.equal(got[:, cols], clean[:, cols])
        q = ops.mx_gemm(a, ops.mx_quantize(y), quantize=True).dequantize(torch.float32)
        assert q[:, :32].isnan().all() and not q[:, 32:].isnan().any()


def test_results_past_the_output_type_are_infinite():
    x = torch.full((4, 64), 3e4, device="cuda")
    got = ops.mx_gemm(ops.mx_quantize(x), ops.mx_quantize(x), dtype=torch.float16)
    assert got.isinf().all()


@pytest.mark.parametrize("m, n, k", [(1, 100, 64), (40, 130, 2048), (300, 130, 64), (300, 33, 64), (700, 192, 300)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_strided_outputs_and_residuals(m, n, k, out):
    a, av = matrix(m, k, 8)
    w, wv = matrix(n, k, 9)
    for pitch, first in ((n + 8, 0), (n + 3, 1), (n + 16, 8)):
        whole = torch.full((m, pitch + first), 7.0, dtype=DT[out], device="cuda")
        c = whole[:, first:first + n]
        res_whole = torch.randn(m, pitch + 5, device="cuda").to(DT[out])
        res = res_whole[:, 2:2 + n]
        views = [ffi.View(t.data_ptr(), t.shape, t.stride(), ops._DTYPES[t.dtype], 0) for t in (res, c)]
        mats = [ffi.MxMatrix(q.data.data_ptr(), q.scales.data_ptr(), *q.shape, 0) for q in (a, w)]
        p = ffi.GemmParams(ffi.EPILOGUE_RESIDUAL, torch.cuda.current_stream().cuda_stream)
        assert ffi.load().tracea_mx_gemm(*mats, None, ctypes.byref(views[0].c), ctypes.byref(views[1].c), None, p) == ffi.SUCCESS
        torch.cuda.synchronize()
        assert_close(c, *reference(av, wv, "residual", None, res, DT[out]))
        outside = torch.ones(pitch + first, dtype=torch.bool)
        outside[first:first + n] = False
        assert (whole[:, outside.cuda()] == 7.0).all()
        # the output may be the residual itself
        kept = c.clone()
        c.copy_(res)
        assert ffi.load().tracea_mx_gemm(*mats, None, ctypes.byref(views[1].c), ctypes.byref(views[1].c), None, p) == ffi.SUCCESS
        torch.cuda.synchronize()
        assert torch.equal(c, kept)


# more CTAs than SMs; several groups of rows, the last one of a single row; and both with the input quantised inside
@pytest.mark.parametrize("m, n, k", [(1, 20011, 300), (7, 19300, 64), (33, 25000, 100), (64, 19999, 2050), (129, 300, 4100), (200, 130, 8192),
                                     (450, 300, 4097), (385, 40, 10000)])
def test_few_rows_beyond_one_wave_and_beyond_one_group(m, n, k):
    w, wv = matrix(n, k, 2, k ** -0.5)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    av = torch.from_numpy(mxref.values(x.double().numpy())).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    res = torch.randn(m, n, generator=torch.Generator().manual_seed(k)).bfloat16().cuda()
    lib = ffi.load()
    for a in (x.cuda(), ops.mx_quantize(x.cuda())):
        before = lib.tracea_b200_launch_count_of(ffi.KERNEL_MX_TOKENS)
        assert_close(ops.mx_gemm(a, w, bias, "bias+residual", res), *reference(av, wv, "bias+residual", bias, res, torch.bfloat16))
        assert_quantized(ops.mx_gemm(a, w, bias, "bias+silu", quantize=True), *reference(av, wv, "bias+silu", bias, None, torch.bfloat16))
        few = m <= 32 or k > 7 * 256                  # more rows than 32 take that form over a longer K only
        assert lib.tracea_b200_launch_count_of(ffi.KERNEL_MX_TOKENS) == before + (2 if few else 0)
    status_ok()


@pytest.mark.parametrize("m, k", [(1, 64), (5, 4096), (300, 64), (1000, 513)])
def test_one_column_and_a_matrix_times_itself(m, k):
    a, av = matrix(m, k, 8)
    assert_close(ops.mx_gemm(a, a, dtype=torch.float32), *reference(av, av, None, None, None, torch.float32))
    w, wv = matrix(1, k, 9)
    for pitch, dtype in ((1, torch.bfloat16), (8, torch.bfloat16), (3, torch.float32), (4, torch.float32)):
        whole = torch.full((m, pitch), 7.0, dtype=dtype, device="cuda")
        c = whole[:, :1]
        mats = [ffi.MxMatrix(q.data.data_ptr(), q.scales.data_ptr(), *q.shape, 0) for q in (a, w)]
        v = ffi.View(c.data_ptr(), c.shape, (pitch, 1), ops._DTYPES[dtype], 0)
        p = ffi.GemmParams(0, torch.cuda.current_stream().cuda_stream)
        assert ffi.load().tracea_mx_gemm(*mats, None, None, ctypes.byref(v.c), None, p) == ffi.SUCCESS
        torch.cuda.synchronize()
        assert_close(c, *reference(av, wv, None, None, None, dtype))
        assert (whole[:, 1:] == 7).all()
    status_ok()


def test_no_rows():
    w, _ = matrix(40, 64, 1)
    x = torch.empty(0, 64, device="cuda")
    q = ops.mx_quantize(x)
    assert q.data.shape == (0, 32) and q.scales.shape == (0, 1, 512) and q.dequantize().shape == (0, 64)
    for a in (x, q):
        assert ops.mx_gemm(a, w).shape == (0, 40) and ops.mx_gemm(a, w, quantize=True).shape == (0, 40)
    assert ops.block_norm(x).shape == (0, 64) and ops.block_norm(x, quantize=True).shape == (0, 64)
    r, y = ops.block_norm_add(x, x, following={"quantize": True})
    assert r.shape == (0, 64) and y.shape == (0, 64)
    assert nn.MxLinear(64, 40, device="cuda")(x.view(2, 0, 64)).shape == (2, 0, 40)
    assert nn.MxFeedForward(64, 40, device="cuda")(x.view(2, 0, 64)).shape == (2, 0, 64)
    with pytest.raises(ffi.TraceaError, match="no rows"):
        ops.mx_gemm(ops.mx_quantize(torch.ones(3, 64, device="cuda")), q)


def test_two_threads_at_once():
    a, _ = matrix(500, 1024, 1)
    w, _ = matrix(600, 1024, 2, 0.03)
    x = torch.randn(5, 1024, device="cuda").bfloat16()
    wanted = [ops.mx_gemm(a, w), ops.mx_gemm(x, w), ops.block_norm(x, kind="layer")]
    torch.cuda.synchronize()
    wrong = []

    def worker():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                got = [ops.mx_gemm(a, w), ops.mx_gemm(x, w), ops.block_norm(x, kind="layer")]
                torch.cuda.current_stream().synchronize()
                wrong.extend(1 for g, t in zip(got, wanted) if not torch.equal(g, t))

    threads = [threading.Thread(target=worker) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    status_ok()


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    with torch.cuda.device(1):
        x, wt = torch.randn(5, 256).cuda(), torch.randn(200, 256).cuda()
    with torch.cuda.device(0):
        w = ops.mx_quantize(wt)
        got = [ops.mx_gemm(x, w), ops.mx_gemm(x, w, quantize=True).dequantize(), ops.block_norm_add(x, x)]
        torch.cuda.synchronize(1)
    with torch.cuda.device(1):
        want = [ops.mx_gemm(x, w), ops.mx_gemm(x, w, quantize=True).dequantize(), ops.block_norm_add(x, x)]
    assert all(torch.equal(g, t) for g, t in zip(got, want))
    with pytest.raises(ffi.TraceaError, match="is on device"):
        ops.mx_gemm(x.to("cuda:0"), w)


def test_the_same_call_gives_the_same_bits():
    for m, n, k in ((1, 4096, 4096), (48, 256, 16384), (700, 900, 1000), (2100, 2100, 2100)):
        a, _ = matrix(m, k, 10)
        w, _ = matrix(n, k, 11)
        first = ops.mx_gemm(a, w, dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(ops.mx_gemm(a, w, dtype=torch.float32), first)


def test_launches():
    if not DEFAULT_CONFIG:
        pytest.skip("a knob is set")
    w, _ = matrix(512, 1024, 1)
    x = torch.randn(1, 1024, device="cuda").bfloat16()
    big, _ = matrix(512, 1024, 2)
    count = lambda: [ffi.launch_count_of(k) for k in (ffi.KERNEL_MX_COPY, ffi.KERNEL_MX_GEMM, ffi.KERNEL_MX_TOKENS, ffi.KERNEL_NORM)]
    for call, want in ((lambda: ops.mx_gemm(x, w), [0, 0, 1, 0]),                              # quantised inside
                       (lambda: ops.mx_gemm(ops.mx_quantize(x), w), [1, 0, 1, 0]),
                       (lambda: ops.mx_gemm(big, w), [0, 1, 0, 0]),
                       (lambda: ops.mx_gemm(x.expand(300, 1024), w), [1, 1, 0, 0]),
                       (lambda: ops.block_norm(x, quantize=True), [0, 0, 0, 1])):
        before = count()
        call()
        assert [b - a for a, b in zip(before, count())] == want


# --------------------------------------------------------------------------------------------------- streams, graphs, devices
def test_streams_graphs_and_changed_inputs():
    w, wv = matrix(300, 512, 1, 0.05)
    x = torch.randn(4, 512, device="cuda").bfloat16()
    wide = torch.randn(300, 512, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.mx_gemm(x, w), ops.mx_gemm(wide, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        small, large = ops.mx_gemm(x, w), ops.mx_gemm(wide, w, quantize=True).dequantize()
    for seed in range(3):
        x.copy_(torch.randn(4, 512, generator=torch.Generator().manual_seed(seed)))
        wide.copy_(torch.randn(300, 512, generator=torch.Generator().manual_seed(seed + 9)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(small, ops.mx_gemm(x, w))
        assert torch.equal(large, ops.mx_gemm(wide, w, quantize=True).dequantize())
    status_ok()


def test_many_streams_at_once():
    """Clusters of several launches side by side on the SMs, next to launches that need a whole SM."""
    w, _ = matrix(4096, 2048, 1, 0.02)
    a, _ = matrix(600, 2048, 2)
    xs = [torch.randn(3, 2048, device="cuda").bfloat16() for _ in range(6)]
    want = [ops.mx_gemm(x, w) for x in xs]
    large = ops.mx_gemm(a, w)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got, big = [None] * len(xs), []
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.mx_gemm(xs[i], w)
                if i % 3 == 2:
                    big.append(ops.mx_gemm(a, w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, t) for g, t in zip(got, want)) and all(torch.equal(b, large) for b in big)
    status_ok()


def test_offsets_past_32_bits():
    m, k = 70000, 32768                               # 2.3 G elements
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-200:] = torch.randn(200, k, device="cuda").bfloat16()
    q = ops.mx_quantize(x)
    tail = ops.mx_quantize(x[-200:])
    assert torch.equal(q.data[-200:], tail.data) and (q.data[:-200] == 0).all()
    v = q.dequantize()
    assert torch.equal(v[-200:], tail.dequantize())
    del v, x, q
    a, av = matrix(66000, 64, 1)
    w, wv = matrix(33000, 64, 2)
    c = ops.mx_gemm(a, w)                             # 2.2 G results
    rows = torch.tensor([0, 1, 32767, 65071, 65999], device="cuda")
    assert_close(c[rows], *reference(av[rows], wv, None, None, None, torch.bfloat16))
    status_ok()


def test_wait_limit():
    """The producer goes silent: every wait runs out, the call after it reports that, and the next one is right again."""
    lib = ffi.load()
    for m, n, k in ((1, 600, 4096), (300, 600, 4096), (6000, 4096, 1024)):
        a, av = matrix(m, k, 1)
        w, wv = matrix(n, k, 2)
        good = ops.mx_gemm(a, w)
        torch.cuda.synchronize()
        lib.tracea_b200_test_hooks(2000000, 1)
        try:
            ops.mx_gemm(a, w)
            torch.cuda.synchronize()
        finally:
            lib.tracea_b200_test_hooks(0, -1)
        with pytest.raises(ffi.TraceaError, match="gave up a bounded wait"):
            ops.mx_gemm(a, w)
        assert torch.equal(ops.mx_gemm(a, w), good)
        status_ok()


# --------------------------------------------------------------------------------------------------- modules
def test_linear_module():
    lin = nn.MxLinear(300, 130, epilogue="silu", device="cuda")
    wv = lambda: torch.from_numpy(mxref.values(lin.weight.detach().double().cpu().numpy())).cuda()
    x = torch.randn(2, 5, 300, device="cuda")
    xv = torch.from_numpy(mxref.values(x.view(10, 300).double().cpu().numpy())).cuda()
    for _ in range(2):
        y = lin(x)
        assert y.shape == (2, 5, 130) and not y.requires_grad
        assert_close(y.view(10, 130), *reference(xv, wv(), "bias+silu", lin.bias.detach(), None, torch.float32))
        with torch.no_grad():
            lin.weight.add_(0.5)                      # a new version
    lin.weight.data = torch.randn(130, 300, device="cuda")
    assert_close(lin(x).view(10, 130), *reference(xv, wv(), "bias+silu", lin.bias.detach(), None, torch.float32))
    for _ in range(20):                               # parameters that come and go may reuse an address, never a result
        lin.weight = torch.nn.Parameter(torch.randn(130, 300, device="cuda"))
        assert_close(lin(x).view(10, 130), *reference(xv, wv(), "bias+silu", lin.bias.detach(), None, torch.float32))
    half = nn.MxLinear(64, 32, bias=False, device="cuda", dtype=torch.float16)
    assert half(torch.randn(3, 64, device="cuda").half()).dtype == torch.float16


def test_linear_module_on_other_streams_and_in_graphs():
    lin = nn.MxLinear(512, 256, device="cuda", epilogue="silu")
    x = torch.randn(3, 512, device="cuda")

    def change():
        lin.weight.data.copy_(torch.randn(256, 512, device="cuda"))
        lin.requantize()

    result = lambda: ops.mx_gemm(x, ops.mx_quantize(lin.weight.detach()), lin.bias.detach(), "bias+silu")
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):                                # the first stream is late with the quantised weight
        change()
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    torch.cuda._sleep(20000000)
                got.append(lin(x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], result()) and torch.equal(got[1], result())
    # quantised in the graph: nothing to read before a replay, and each replay reads the weight as it is
    change()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(x)
    assert torch.equal(lin(x), result())
    for _ in range(2):
        change()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, result())
    # quantised before: the graph keeps to that weight after the layer has dropped it
    lin(x)
    h = torch.cuda.CUDAGraph()
    with torch.cuda.graph(h):
        y = lin(x)
    old = result()
    change()
    for _ in range(50):
        lin.weight.data.add_(0.0)
        lin.requantize()
        assert torch.equal(lin(x), result())
    junk = [torch.full((256, 256), 119, dtype=torch.uint8, device="cuda") for _ in range(50)]
    h.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, old) and len(junk) == 50
    with torch.inference_mode():
        assert torch.equal(lin(x), result())
    lin.half()                                        # a 16-bit bias is added as it is, or, into a quantised output, as fp32
    x = x.half()
    assert torch.equal(lin(x), result())
    q = lin.product(x, quantize=True)
    want = ops.mx_gemm(x, ops.mx_quantize(lin.weight.detach()), lin.bias.detach().float(), "bias+silu", quantize=True)
    assert torch.equal(q.data, want.data)
    status_ok()


@pytest.mark.parametrize("samples, positions, c, hidden, dtype", [(1, 1, 64, 96, "bf16"), (3, 49, 200, 333, "f16"), (4, 196, 512, 1024, "bf16")])
def test_feed_forward_module_is_its_operators(samples, positions, c, hidden, dtype):
    """The block's parts, each against its definition on the input it got, which are themselves tested above; and the whole, whose
    4-bit steps may fall to either side of a border, by the size of a step: both products' inputs are off by at most a quarter of
    themselves in few places -- a tenth of the result bounds them by far -- so this tells a wrong wiring, not a rounding."""
    ff = nn.MxFeedForward(c, hidden, norm="layer", residual_scale=0.5, device="cuda", dtype=DT[dtype])
    x = torch.randn(samples, positions, c, device="cuda").to(DT[dtype])
    gate, scale, shift = (0.3 * torch.randn(samples, c, device="cuda") for _ in range(3))
    rows = x.view(-1, c)
    q = ops.block_norm(rows, ff.pre_weight.detach(), None, scale, shift, "layer", quantize=True)
    u = ops.mx_gemm(q, ops.mx_quantize(ff.up.weight.detach()), ff.up.bias.detach().float(), "bias+silu", quantize=True)
    h = ops.mx_gemm(u, ops.mx_quantize(ff.down.weight.detach()), ff.down.bias.detach().float(), "bias", dtype=DT[dtype])
    r = ops.block_norm_add(h, rows, ff.post_weight.detach(), gate=gate, residual_scale=0.5, kind="layer")
    assert torch.equal(ff(x, gate, scale, shift).view(-1, c), r)
    d = lambda t: t.detach().double().cpu().numpy()
    xs = d(rows)
    y = mxref.values(mxref.norm(xs, "layer", 1e-6, d(ff.pre_weight), None, d(scale), d(shift))[0])
    z = mxref.values(mxref.activation(y @ mxref.values(d(ff.up.weight)).T + d(ff.up.bias), "silu"))
    z = z @ mxref.values(d(ff.down.weight)).T + d(ff.down.bias)
    n = mxref.norm(z, "layer", 1e-6, d(ff.post_weight))[0] * np.repeat(d(gate), positions, axis=0)
    want = 0.5 * xs + n
    assert np.linalg.norm(d(r) - want) <= 0.1 * np.linalg.norm(n) + 0.01 * np.linalg.norm(want)
    status_ok()
