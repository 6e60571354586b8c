"""Rows and layouts at which the norms around a block can go wrong on a B200."""
import pytest
import torch

import mxref
from test_block_norm_gpu import rows, stage, vectors
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
