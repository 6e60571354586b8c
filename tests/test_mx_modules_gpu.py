"""nn.MxLinear's quantised weight on a B200 as a program changes the weight, from optimizers, streams and threads."""
import threading

import pytest
import torch

from test_mx_gpu import status_ok
from tracea_b200 import nn, ops

pytestmark = pytest.mark.gpu


def result(lin, x):
    return ops.mx_gemm(x, ops.mx_quantize(lin.weight.detach()), lin.bias.detach(), "bias")


@pytest.mark.parametrize("options", [{}, {"foreach": True}, {"fused": True}, {"fused": True, "capturable": True}])
def test_optimizer_steps(options):
    lin = nn.MxLinear(256, 192, device="cuda")
    x = torch.randn(5, 256, device="cuda")
    optimizer = torch.optim.AdamW(lin.parameters(), lr=0.1, **options)
    for _ in range(3):
        for p in lin.parameters():
            p.grad = torch.randn_like(p)
        before = lin(x)
        optimizer.step()
        assert torch.equal(lin(x), result(lin, x)) and not torch.equal(lin(x), before)
    status_ok()
