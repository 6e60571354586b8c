"""nn.TraceaConv2d's packed weight on a B200 as a program changes the weight, from optimizers, streams and graphs."""
import pytest
import torch

from tracea_b200 import nn, ops

pytestmark = pytest.mark.gpu


def layer():
    return nn.TraceaConv2d(64, 64, 3, padding=1, device="cuda", dtype=torch.bfloat16), torch.randn(2, 64, 12, 12, device="cuda").bfloat16()


def result(conv, x):
    return ops.conv2d_nchw(x, conv.weight.detach().clone(), conv.bias.detach(), None, 1, 1, 1, 1, "bias")


@pytest.mark.parametrize("options", [{}, {"foreach": True}, {"fused": True}])
def test_optimizer_steps(options):
    conv, x = layer()
    optimizer = torch.optim.AdamW(conv.parameters(), lr=0.1, **options)
    for _ in range(3):
        for p in conv.parameters():
            p.grad = torch.randn_like(p)
        before = conv(x)
        optimizer.step()
        assert torch.equal(conv(x), result(conv, x)) and not torch.equal(conv(x), before)


def test_a_first_call_in_a_capture_keeps_nothing_that_only_a_replay_computes():
    conv, x = layer()
    want = result(conv, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = conv(x)
    assert torch.equal(conv(x), want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    with torch.no_grad():
        conv.weight.mul_(-2.0)
    graph.replay()                                 # packed in the graph: each replay reads the weight as it is
    torch.cuda.synchronize()
    assert torch.equal(y, result(conv, x)) and torch.equal(conv(x), y)


def test_other_streams():
    conv, x = layer()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):                             # the first stream is late with the packed weight
        with torch.no_grad():
            conv.weight.normal_()
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    torch.cuda._sleep(20000000)
                got.append(conv(x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], result(conv, x)) and torch.equal(got[1], got[0])


def test_parameters_that_come_and_go():
    conv, x = layer()
    for _ in range(20):
        conv(x)
        for _ in range(3):
            conv.weight = torch.nn.Parameter(torch.randn(64, 64, 3, 3, device="cuda").bfloat16())
        assert torch.equal(conv(x), result(conv, x))
    with torch.inference_mode():
        conv.weight = torch.nn.Parameter(torch.randn(64, 64, 3, 3, device="cuda").bfloat16(), requires_grad=False)
        assert torch.equal(conv(x), result(conv, x))
