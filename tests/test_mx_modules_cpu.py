"""What nn.MxLinear keeps between calls, without a GPU: the conversion is replaced by one that counts and copies."""
import copy
import io
import types

import pytest
import torch

from tracea_b200 import nn


@pytest.fixture
def quantized(monkeypatch):
    """The weights that have been quantised; a quantised weight is a copy of it."""
    made = []

    def quantize(w):
        made.append(w)
        return w.detach().clone()

    monkeypatch.setattr(nn.ops, "mx_quantize", quantize)
    stream = types.SimpleNamespace(synchronize=lambda: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(nn, "_stream_handle", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def bump(layer, version):
    with torch.no_grad():
        while layer.weight._version < version:
            layer.weight.add_(1.0)


@pytest.mark.parametrize("how", ["deepcopy", "copy", "pickle"])
def test_a_copy_of_the_layer_takes_nothing_of_what_the_layer_keeps(quantized, how):
    """A copied parameter counts its versions from zero again: one of them will be the number that the original's stands under."""
    lin = nn.MxLinear(8, 4)
    bump(lin, 5)
    assert torch.equal(lin._kernel_weight(), lin.weight)
    if how == "pickle":
        f = io.BytesIO()
        torch.save(lin, f)
        f.seek(0)
        other = torch.load(f, weights_only=False)
    else:
        other = copy.deepcopy(lin) if how == "deepcopy" else copy.copy(lin)
    if how != "copy":
        bump(other, lin.weight._version)
    assert torch.equal(other._kernel_weight(), other.weight)
    assert torch.equal(lin._kernel_weight(), lin.weight)
    before = len(quantized)
    for layer in (lin, other):                            # and both keep theirs
        layer._kernel_weight()
    assert len(quantized) == before


@pytest.mark.parametrize("make", [lambda p: torch.optim.Adam(p, fused=True), lambda p: torch.optim.AdamW(p, lr=0.1, fused=True),
                                  lambda p: torch.optim.SGD(p, lr=0.1, fused=True), lambda p: torch.optim.SGD(p, lr=0.1)])
def test_a_step_of_any_optimizer_is_seen(quantized, make):
    """Fused ones write the weight without counting a version of it."""
    lin = nn.MxLinear(8, 4)
    optimizer = make(lin.parameters())
    for _ in range(3):
        lin.weight.grad = torch.ones_like(lin.weight)
        lin._kernel_weight()
        optimizer.step()
        assert torch.equal(lin._kernel_weight(), lin.weight)
    before = len(quantized)
    lin._kernel_weight()
    assert len(quantized) == before
