"""Values at which an epilogue of the 4-bit products can go wrong on a B200: NaN behind a ReLU, results far apart that share
arithmetic, and activations where their formula cancels.

Most of these put exact values in front of an activation: codes of zero as input, and the values as an fp32 bias."""
import pytest
import torch

import mxref
from test_mx_gpu import DT, assert_close, assert_quantized, matrix, status_ok
from tracea_b200 import ops

pytestmark = pytest.mark.gpu


def zeros(m, k):
    return ops.mx_quantize(torch.zeros(m, k, device="cuda"))


# rows of both forms of the product, and a K at which 40 rows take the one for few
@pytest.mark.parametrize("m, k", [(1, 300), (40, 300), (40, 2048), (300, 300), (700, 513)])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "mx"])
def test_relu_keeps_nan(m, k, out):
    n = 200
    _, av = matrix(m, k, 1)
    w, wv = matrix(n, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3)).cuda()

    def product(a, b, epilogue, residual=None):
        args = (a, b, bias if "bias" in epilogue else None, epilogue, residual)
        return ops.mx_gemm(*args, quantize=True).dequantize(torch.float32) if out == "mx" else ops.mx_gemm(*args, dtype=DT[out])

    x = av.float()
    clean = ops.mx_quantize(x)
    x[m // 2, 40] = float("nan")
    y = wv.float()
    y[5, 0] = float("inf")
    rest = torch.arange(m, device="cuda") != m // 2
    for e in ("relu", "bias+relu"):
        want = product(clean, w, e)
        assert (want >= 0).all() and (want == 0).any()
        inputs = [ops.mx_quantize(x)] + ([x.to(DT[out])] if out != "mx" else [x])
        got = product(inputs[0], w, e)
        assert got[m // 2].isnan().all() and torch.equal(got[rest], want[rest])
        assert product(inputs[1], w, e)[m // 2].isnan().all()
        got = product(clean, ops.mx_quantize(y), e)
        assert got[:, 5].isnan().all()
        others = torch.arange(n, device="cuda") != 5 if out != "mx" else torch.arange(n, device="cuda") >= 32   # a block is NaN as a whole
        assert torch.equal(got[:, others], want[:, others])
    if out != "mx":
        r = torch.randn(m, n, generator=torch.Generator().manual_seed(4)).to(DT[out]).cuda()
        want = product(clean, w, "bias+residual+relu", r)
        r[0, 7] = float("nan")
        got = product(clean, w, "bias+residual+relu", r)
        assert got[0, 7].isnan() and got.isnan().sum() == 1
        assert torch.equal(got.nan_to_num(nan=0.0), torch.where(got.isnan(), 0.0, want))
    status_ok()


@pytest.mark.parametrize("m", [1, 300])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "mx"])
def test_silu_of_values_far_apart(m, out):
    """Neighbours of 32 columns share reciprocals: none of them may carry another's size into a result. -19.9 and the like are the
    lowest that do; next to them values up to the type's largest, in every place of four."""
    large = {"f16": [6e4, 3e3, 65504.0, 1.0], "mx": [1e30, 1e20, 3e38, 2e38]}.get(out, [1e30, 1e20, 3e38, 1.0])
    low = [-19.9, -19.0, -12.0, -1.0]
    v = torch.tensor([low[(i // 32 + i) % 4] for i in range(512)])
    for i in range(64):
        v[8 * i + i % 8] = large[i // 8 % 4]
    v[256::16] = large[0]
    bias = v.cuda()
    a, w = zeros(m, 64), zeros(512, 64)
    y = (bias.double() * torch.sigmoid(bias.double())).expand(m, 512)
    err = (2.0 ** -20 if out == "f32" else 2.0 ** -16) * y.abs() + 1e-37          # as in test_mx_gpu.py
    if out == "mx":
        assert_quantized(ops.mx_gemm(a, w, bias, "bias+silu", quantize=True), y, err)
    else:
        got = ops.mx_gemm(a, w, bias, "bias+silu", dtype=DT[out])
        assert got.isfinite().all()
        assert_close(got, y, err)
    status_ok()


def columns(values):
    """(a row of ones, w, x): a w^T is x, close to `values`, exactly: each as four elements of the format in blocks of their own."""
    left, w = values.double().numpy().copy(), torch.zeros(len(values), 128, dtype=torch.float64)
    for b in range(4):
        w[:, 32 * b] = torch.from_numpy(mxref.values(left[:, None])[:, 0])
        left -= w[:, 32 * b].numpy()
    a = torch.zeros(1, 128)
    a[:, ::32] = 1.0
    return a.cuda(), ops.mx_quantize(w.float().cuda()), w.sum(1).cuda()


@pytest.mark.parametrize("m", [1, 300])
@pytest.mark.parametrize("out", ["f16", "bf16", "mx"])
def test_gelu_is_good_to_the_outputs_rounding_where_it_cancels(m, out):
    """x / (1 + e^z), z = -2 sqrt(2 / pi) (x + 0.044715 x^3). In fp32 z is off by at most five half steps, 5 2^-24 |z|, by which e^z is
    off relative to itself; the exponential (2^-22), the sum, the quotient (2^-22) and the product add less than 2^-20. The output's
    rounding, half a step, is assert_close's."""
    a, w, x = columns(torch.linspace(-14, 14, 4096))
    a = ops.mx_quantize(a.expand(m, 128))
    z = -2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)
    y = (x / (1 + torch.exp(z))).expand(m, -1)
    err = (z.abs() * 2.0 ** -21 + 2.0 ** -20) * y.abs() + 1e-37
    if out == "mx":
        assert_quantized(ops.mx_gemm(a, w, None, "gelu", quantize=True), y, err)
    else:
        assert_close(ops.mx_gemm(a, w, None, "gelu", dtype=DT[out]), y, err)
    a, w, x = columns(torch.tensor([2.0 ** 70, -2.0 ** 70, 1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127, 0.0, 32.0, -32.0, 1.5 * 2.0 ** 126] * 8))
    if out == "bf16":
        got = ops.mx_gemm(ops.mx_quantize(a.expand(m, 128)), w, None, "gelu", dtype=torch.bfloat16)
        assert torch.equal(got, x.clamp(min=0).bfloat16().expand(m, -1))
    status_ok()
