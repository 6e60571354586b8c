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


def test_a_new_weight_while_another_thread_captures():
    """A capture that is open to other threads' work (thread-local mode) survives a first call with a new weight, and the call too."""
    lin = nn.MxLinear(512, 256, device="cuda")
    x, c = torch.randn(3, 512, device="cuda"), torch.randn(64, 64, device="cuda")
    lin(x)
    torch.cuda.synchronize()
    begun, done, got = threading.Event(), threading.Event(), []

    def capture():
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.capture_begin(capture_error_mode="thread_local")
                try:
                    y = c + 1
                    begun.set()
                    done.wait(60)
                    y = y + 1
                finally:
                    begun.set()
                    graph.capture_end()
            graph.replay()
            torch.cuda.synchronize()
            got.append(torch.equal(y, c + 1 + 1))
        except RuntimeError as e:
            got.append(e)

    thread = threading.Thread(target=capture)
    thread.start()
    begun.wait(60)
    try:
        with torch.no_grad():
            lin.weight.mul_(2.0)
        y = lin(x)
        lin.requantize()
        z = lin(x)
    finally:
        done.set()
        thread.join()
    assert got == [True]
    assert torch.equal(y, result(lin, x)) and torch.equal(z, y)
    status_ok()


def test_a_replaced_weight_is_not_overwritten_while_another_stream_reads_it():
    """The other stream is late: by the time it reads the old quantised weight, the layer has a new one and its memory has been free for
    a while, to a stream that allocates and writes as much again and again."""
    lin = nn.MxLinear(1024, 1024, device="cuda")
    x = torch.randn(3, 1024, device="cuda")
    side = torch.cuda.Stream()
    lin(x), torch.cuda.synchronize()
    for _ in range(2):
        want = result(lin, x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100000000)
            got = lin(x)
        with torch.no_grad():
            lin.weight.mul_(2.0)
        new = lin(x)
        size = ops.mx_quantize(lin.weight.detach()).data.untyped_storage().nbytes()
        lin.requantize()
        junk = [torch.full((size,), 119, dtype=torch.uint8, device="cuda") for _ in range(20)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(new, result(lin, x)) and len(junk) == 20
        lin(x), torch.cuda.synchronize()
    status_ok()


def test_feed_forward_of_no_samples():
    ff = nn.MxFeedForward(64, 96, device="cuda")
    none = torch.empty(0, 64, device="cuda")
    assert ff(torch.empty(0, 7, 64, device="cuda"), gate=none, scale=none, shift=none).shape == (0, 7, 64)
