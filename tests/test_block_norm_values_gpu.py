"""Rows and layouts at which the norms around a block can go wrong on a B200."""
import pytest
import torch

import mxref
from test_block_norm_gpu import EPS, assert_rows, d, rows, vectors
from test_mx_gpu import DT, bytes_of, status_ok
from tracea_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m, c", [(12, 8), (12, 40), (12, 200), (12, 333), (700, 520), (12, 1032), (12, 2056), (5, 8200)])
def test_scale_bytes_past_the_last_block_are_zero_whatever_the_row_holds(m, c, dtype):
    x = rows(m, c, dtype, 1)
    x[0, 0], x[1, c - 1], x[2, c // 2] = float("nan"), float("inf"), float("-inf")
    x[3] = 0
    h = rows(m, c, dtype, 2)
    h[4, c // 3] = float("nan")
    for kind in ("rms", "layer", "none"):
        for eps in (1e-6, 0.0):                               # a row of zeros without an epsilon is 0 / 0
            for q in (ops.block_norm(x, kind=kind, eps=eps, quantize=True),
                      ops.block_norm_add(h, x, kind=kind, eps=eps, following={"kind": kind, "eps": eps, "quantize": True})[1]):
                codes, scales, rest = mxref.unpack(*bytes_of(q), m, c)
                assert (rest == 0).all() and (codes[:, c:] & 7 == 0).all()
                assert (scales[0] == 255).any() and (kind == "none" or (scales[0] == 255).all())
    status_ok()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m, c", [(7, 8), (30, 200), (700, 1000), (640, 1001), (40, 2048), (9, 2051)])
def test_bits_of_a_join_with_a_norm_behind_it(m, c, dtype):
    """Those of two calls where the rows are aligned as the second call's are, in whole tensors or in slices of wider ones; where only
    the second call's are, its norm to the bound."""
    v = vectors(c, 1, torch.float32, 4)
    for pad, first in ((0, 0), (8, 8), (8, 0), (5, 3)):
        h, x = (rows(m, c + pad, dtype, 5 + i)[:, first:first + c] for i in range(2))
        for following in ({"kind": "layer", "weight": v["weight"]}, {"kind": "rms", "quantize": True}):
            r, y = ops.block_norm_add(h, x, v["weight"], following=following)
            want = ops.block_norm(r, **following)
            alike = c % 8 != 0 or (pad % 8 == 0 and first % 8 == 0)
            if "quantize" in following:
                assert not alike or torch.equal(y.data, want.data)
            elif alike:
                assert torch.equal(y, want)
            else:
                assert_rows(y, *mxref.norm(d(r), "layer", EPS, d(v["weight"])))
    status_ok()
