"""torch.nn front end of the conv path: the reference's `TraceaConv2d` / `patch_conv2d`
(tracea-python/python/tracea/__init__.py:19-56), forward only; and of the 4-bit products, `MxLinear` and `MxFeedForward`, which
the reference does not have.

Differences from the reference's module, all deliberate:
  * dilation > 1 is computed here (the reference falls back to PyTorch for it);
  * configurations the library does not compute (groups != 1, a padding_mode other than "zeros", string paddings)
    raise NotImplementedError instead of silently running PyTorch's own convolution: this package has no fallback
    path, and a caller should know which backend produced its numbers;
  * OIHW-contiguous weights are packed into the kernel's [K][R][S][C] layout once per weight version
    (`ops.prepack_conv2d_weight`) and then read in place on every call.
"""
import weakref

import torch
from torch.optim.optimizer import register_optimizer_step_post_hook

from . import ops


class TraceaConv2d(torch.nn.Conv2d):
    """Drop-in for torch.nn.Conv2d on CUDA tensors (fp32 as TF32, fp16, bf16). The output takes the memory format of
    the input; channels-last inputs are consumed in place."""

    def _check(self):
        if self.groups != 1:
            raise NotImplementedError("TraceaConv2d: groups=%d is not supported (groups must be 1)" % self.groups)
        if self.padding_mode != "zeros":
            raise NotImplementedError("TraceaConv2d: padding_mode=%r is not supported" % self.padding_mode)
        if isinstance(self.padding, str):
            raise NotImplementedError("TraceaConv2d: padding=%r is not supported, pass integers" % (self.padding,))

    def _kernel_weight(self):
        w = self.weight.detach()
        vec = 16 // w.element_size()
        if w.stride(1) == 1 or w.shape[1] % vec != 0:
            return w            # already channels-last, or channel-padded per call inside the library
        key = (w._version, w.data_ptr(), w.dtype, w.device)
        cached = getattr(self, "_tracea_packed", None)
        if cached is None or cached[0] != key:
            cached = (key, ops.prepack_conv2d_weight(w))
            self._tracea_packed = cached
        return cached[1]

    def forward(self, x):
        self._check()
        bias = self.bias.detach() if self.bias is not None else None
        return ops.conv2d_nchw(x, self._kernel_weight(), bias, None, self.stride, self.padding, self.dilation, 1,
                               "bias" if bias is not None else None)


def _stream_handle(device_index):
    """The current stream's handle. torch.cuda.current_stream takes 2 us, a fifth of a layer's call."""
    return torch._C._cuda_getCurrentRawStream(device_index)


# Layers that keep a quantised weight. Some optimizers, torch's fused ones among them, write a weight without counting a version of it,
# so the layers that a step has changed are told.
_quantized_layers = weakref.WeakSet()
_step_hook = None


def _after_step(optimizer, args, kwargs):
    written = {id(p) for group in optimizer.param_groups for p in group["params"] if p.grad is not None}
    for layer in list(_quantized_layers):
        if id(layer.weight) in written:
            layer.requantize()


def _watch(layer):
    global _step_hook
    if _step_hook is None:
        _step_hook = register_optimizer_step_post_hook(_after_step)
    _quantized_layers.add(layer)


class MxLinear(torch.nn.Linear):
    """Drop-in for torch.nn.Linear on CUDA tensors whose weight and input are multiplied in the 4-bit microscaled format
    (``ops.mx_gemm``): the weight is quantised once per version, the input, of any leading shape and fp32, fp16 or bf16, in every
    call. The output has the input's type; ``epilogue`` is an activation of ``ops.gemm``. Forward only, as TraceaConv2d.

    A new version waits once for the current stream: other streams may read the quantised weight from then on. (Like any call
    that may allocate, it ends a capture that another thread has open in torch's "global" mode; "thread_local" ones go on.) A CUDA
    graph that is captured with a quantised weight at hand keeps to that one, whatever becomes of the layer's, and the layer holds it
    as long as it lives; captured right after ``requantize()``, or after a step of an optimizer, it quantises the weight in every
    replay. A weight made in inference mode has no versions and is quantised in every call."""

    def __init__(self, in_features, out_features, bias=True, epilogue=None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device, dtype)
        if epilogue not in (None, "relu", "silu"):
            raise NotImplementedError("MxLinear: epilogue=%r is not supported" % (epilogue,))
        self.epilogue = epilogue

    def _kernel_weight(self):
        w = self.weight.detach()
        if w.is_inference():                      # no version to go by
            return ops.mx_quantize(w)
        # The cached entry holds the weight it was made from, so that another one cannot lie at its address.
        cached, version = getattr(self, "_tracea_quantized", None), w._version
        if (cached is None or cached[1] != version or cached[0].data_ptr() != w.data_ptr() or cached[0].dtype != w.dtype
                or cached[0].device != w.device or cached[0].shape != w.shape or cached[0].stride() != w.stride()):
            q = ops.mx_quantize(w)
            if torch.cuda.is_current_stream_capturing():
                return q                          # the graph's: nothing is in it before a replay
            torch.cuda.current_stream(w.device).synchronize()    # complete for every stream (no capture lets the device be waited for)
            self._tracea_quantized = (w, version, q, w.device.index, _stream_handle(w.device.index))
            _watch(self)
            return q
        if torch.cuda.is_current_stream_capturing():
            self.__dict__.setdefault("_tracea_captured", {})[id(cached)] = cached     # graphs read it as long as the layer lives
        elif _stream_handle(cached[3]) != cached[4]:
            # once it is dropped, its memory, one allocation, waits for what this stream reads
            cached[2].data.record_stream(torch.cuda.current_stream(w.device))
        return cached[2]

    def __getstate__(self):
        """Copies and pickles go without the quantised weight: their parameter counts its versions anew."""
        return {k: v for k, v in super().__getstate__().items() if k not in ("_tracea_quantized", "_tracea_captured")}

    def requantize(self):
        """Forget the quantised weight. Needed after a change that torch does not count: one through ``weight.data``, or by the replay
        of a graph. (Steps of a torch.optim.Optimizer are noticed, those that torch does not count too.)"""
        self._tracea_quantized = None

    def product(self, rows, dtype=None, quantize=False):
        """The layer on (M, in_features) rows, a tensor or an MxTensor; see ``ops.mx_gemm`` for dtype and quantize."""
        bias = None if self.bias is None else self.bias.detach()
        out = dtype or (torch.bfloat16 if isinstance(rows, ops.MxTensor) else rows.dtype)
        if bias is not None and bias.dtype != torch.float32 and (quantize or bias.dtype != out):
            bias = bias.float()
        parts = [p for p in ("bias" if bias is not None else None, self.epilogue) if p]
        return ops.mx_gemm(rows, self._kernel_weight(), bias, "+".join(parts) or None, None, dtype, quantize)

    def forward(self, x):
        y = self.product(x.detach().reshape(-1, self.in_features))
        return y.view(*x.shape[:-1], self.out_features)


class MxFeedForward(torch.nn.Module):
    """A feed-forward block with a norm in front and one behind it, in four launches (five where ``up`` has a 16-bit bias):

        r = residual_scale * x + gate * (norm(down(silu(up(norm(x) * (1 + scale) + shift)))))

    Both products read 4-bit operands; the norm in front and the first product write theirs in that format. x: (..., C), its
    leading dimension the samples when gate, scale or shift, (samples, C), are given. Forward only."""

    def __init__(self, dim, hidden, norm="rms", eps=1e-6, residual_scale=1.0, bias=True, device=None, dtype=None):
        super().__init__()
        self.norm, self.eps, self.residual_scale = norm, eps, residual_scale
        self.pre_weight = torch.nn.Parameter(torch.ones(dim, device=device))
        self.post_weight = torch.nn.Parameter(torch.ones(dim, device=device))
        self.up = MxLinear(dim, hidden, bias, "silu", device, dtype)
        self.down = MxLinear(hidden, dim, bias, None, device, dtype)

    def forward(self, x, gate=None, scale=None, shift=None):
        rows = x.detach().reshape(-1, x.shape[-1])
        q = ops.block_norm(rows, self.pre_weight.detach(), None, scale, shift, self.norm, self.eps, quantize=True)
        h = self.down.product(self.up.product(q, quantize=True), dtype=x.dtype)
        r = ops.block_norm_add(h, rows, self.post_weight.detach(), gate=gate, residual_scale=self.residual_scale, kind=self.norm,
                               eps=self.eps)
        return r.view(x.shape)


def patch_conv2d():
    """Replace torch.nn.Conv2d with TraceaConv2d for modules constructed afterwards
    (tracea-python/python/tracea/__init__.py:19-26)."""
    torch.nn.Conv2d = TraceaConv2d
