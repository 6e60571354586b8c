"""torch.nn front end of the conv path: the reference's `TraceaConv2d` / `patch_conv2d`
(tracea-python/python/tracea/__init__.py:19-56), forward only; and of the 4-bit products, `MxLinear`, `MxFeedForward` and
`MxAttention`, which the reference does not have.

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


def _stream_handle(device_index):
    """The current stream's handle. torch.cuda.current_stream takes 2 us, a fifth of a layer's call."""
    return torch._C._cuda_getCurrentRawStream(device_index)


# Layers that keep a form of their weight. Some optimizers, torch's fused ones among them, write a weight without counting a version of
# it, so the layers that a step has changed are told.
_keeping_layers = weakref.WeakSet()
_step_hook = None


def _after_step(optimizer, args, kwargs):
    written = {id(p) for group in optimizer.param_groups for p in group["params"] if p.grad is not None}
    for layer in list(_keeping_layers):
        if id(layer.weight) in written:
            layer._forget_weight()


class _KeepsWeight:
    """A layer that keeps its weight in the form that the kernels read, made once per version of the weight.

    A new version waits once for the current stream: other streams may read the form from then on. (Like any call that may allocate, it
    ends a capture that another thread has open in torch's "global" mode; "thread_local" ones go on.) A CUDA graph that is captured
    with the form at hand keeps to that one, whatever becomes of the layer's, and the layer holds it as long as it lives; captured
    without, as after a step of an optimizer, the graph makes it in every replay. A weight made in inference mode has no versions: its
    form is made in every call."""

    def _make_form(self, w):
        """The weight's form, and the tensor whose memory it is."""
        raise NotImplementedError

    def _weight_form(self):
        w = self.weight
        if w.is_inference():                      # no version to go by
            return self._make_form(w.detach())[0]
        # The kept entry holds the weight it was made from, so that another one cannot lie at its address.
        kept, version = getattr(self, "_tracea_kept", None), w._version
        if (kept is None or kept[1] != version or kept[0].data_ptr() != w.data_ptr() or kept[0].dtype != w.dtype
                or kept[0].device != w.device or kept[0].shape != w.shape or kept[0].stride() != w.stride()):
            w = w.detach()
            form, memory = self._make_form(w)
            if torch.cuda.is_current_stream_capturing():
                return form                       # the graph's: nothing is in it before a replay
            torch.cuda.current_stream(w.device).synchronize()    # complete for every stream (no capture lets the device be waited for)
            self._tracea_kept = (w, version, form, memory, w.device.index, _stream_handle(w.device.index))
            global _step_hook
            if _step_hook is None:
                _step_hook = register_optimizer_step_post_hook(_after_step)
            _keeping_layers.add(self)
            return form
        if torch.cuda.is_current_stream_capturing():
            self.__dict__.setdefault("_tracea_captured", {})[id(kept)] = kept     # graphs read it as long as the layer lives
        elif _stream_handle(kept[4]) != kept[5]:
            # once it is dropped, its memory waits for what this stream reads
            kept[3].record_stream(torch.cuda.current_stream(w.device))
        return kept[2]

    def _forget_weight(self):
        self._tracea_kept = None

    def __getstate__(self):
        """Copies and pickles go without what is kept: their parameter counts its versions anew."""
        return {k: v for k, v in super().__getstate__().items() if k not in ("_tracea_kept", "_tracea_captured")}


class TraceaConv2d(_KeepsWeight, torch.nn.Conv2d):
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
        w = self.weight
        vec = 16 // w.element_size()
        if w.stride(1) == 1 or w.shape[1] % vec != 0:
            return w.detach()   # already channels-last, or channel-padded per call inside the library
        return self._weight_form()

    def _make_form(self, w):
        packed = ops.prepack_conv2d_weight(w)
        return packed, packed

    def forward(self, x):
        self._check()
        bias = self.bias.detach() if self.bias is not None else None
        return ops.conv2d_nchw(x, self._kernel_weight(), bias, None, self.stride, self.padding, self.dilation, 1,
                               "bias" if bias is not None else None)


class MxLinear(_KeepsWeight, torch.nn.Linear):
    """Drop-in for torch.nn.Linear on CUDA tensors whose weight and input are multiplied in the 4-bit microscaled format
    (``ops.mx_gemm``): the weight is quantised once per version, the input, of any leading shape and fp32, fp16 or bf16, in every
    call. The output has the input's type; ``epilogue`` is an activation of ``ops.gemm``. Forward only, as TraceaConv2d.

    A CUDA graph that is captured with a quantised weight at hand keeps to that one, whatever becomes of the layer's; captured right
    after ``requantize()``, or after a step of an optimizer, it quantises the weight in every replay. A weight made in inference mode is
    quantised in every call. More on what is kept: _KeepsWeight."""

    def __init__(self, in_features, out_features, bias=True, epilogue=None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device, dtype)
        if epilogue not in (None, "relu", "silu"):
            raise NotImplementedError("MxLinear: epilogue=%r is not supported" % (epilogue,))
        self.epilogue = epilogue

    def _make_form(self, w):
        q = ops.mx_quantize(w)
        return q, q.data                          # its scales lie in the same allocation

    _kernel_weight = _KeepsWeight._weight_form

    def requantize(self):
        """Forget the quantised weight. Needed after a change that torch does not count: one through ``weight.data``, or by the replay
        of a graph. (Steps of a torch.optim.Optimizer are noticed, those that torch does not count too.)"""
        self._forget_weight()

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


class MxAttention(torch.nn.Module):
    """An attention block on a paged cache in 8 bits, with a norm in front and one behind it, as MxFeedForward is for the other half of
    a layer; for prompts, pieces of them and single tokens alike:

        q, k, v = qkv(norm(x) * (1 + scale) + shift);  q, k normalised per head (``head_norm``) and rotated by position
        r = residual_scale * x + gate * norm(out(attention(q, cache with k and v)))

    Both projections are MxLinear; keys and values go into the cache, which the caller keeps (``cache`` makes one that fits), in the same
    launch that rotates the queries. x: (T, dim), float16 or bfloat16, the last tokens of the sequences that ``pages``, ``lengths`` and
    ``starts`` describe (``ops.kv_append``); gate, scale, shift: (G, dim) with G dividing T. Forward only."""

    def __init__(self, dim, heads, kv_heads=None, head_dim=None, norm="rms", head_norm=True, eps=1e-6, base=10000.0, window=0,
                 residual_scale=1.0, bias=False, device=None, dtype=None):
        super().__init__()
        self.heads, self.kv_heads = heads, kv_heads or heads
        if self.heads % self.kv_heads != 0:
            raise ValueError("heads must be a multiple of kv_heads")
        if head_dim is None and dim % heads != 0:
            raise ValueError("dim is no multiple of heads: give head_dim")
        self.head_dim = head_dim or dim // heads
        if self.head_dim % 16 != 0 or self.head_dim > 128:
            raise ValueError("head_dim must be a multiple of 16 up to 128")
        self.norm, self.eps, self.base, self.window, self.residual_scale = norm, eps, base, window, residual_scale
        self.pre_weight = torch.nn.Parameter(torch.ones(dim, device=device))
        self.post_weight = torch.nn.Parameter(torch.ones(dim, device=device))
        self.q_weight = torch.nn.Parameter(torch.ones(self.head_dim, device=device)) if head_norm else None
        self.k_weight = torch.nn.Parameter(torch.ones(self.head_dim, device=device)) if head_norm else None
        self.qkv = MxLinear(dim, (self.heads + 2 * self.kv_heads) * self.head_dim, bias, None, device, dtype)
        self.out = MxLinear(self.heads * self.head_dim, dim, bias, None, device, dtype)
        self._frequencies = ops.rotary_frequencies(self.head_dim, base, self.pre_weight.device)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        # neither a parameter nor a buffer: a change of type would round them
        self._frequencies = ops.rotary_frequencies(self.head_dim, self.base, self.pre_weight.device)
        return self

    def cache(self, pages, page_size=64):
        """An empty ops.KvCache of ``pages`` pages for this block, on its device."""
        return ops.KvCache.empty(pages, self.kv_heads, self.head_dim, page_size, self.pre_weight.device)

    def forward(self, x, cache, pages, lengths, starts=None, gate=None, scale=None, shift=None):
        rows = x.detach()
        weights = [None if w is None else w.detach() for w in (self.q_weight, self.k_weight)]
        normed = ops.block_norm(rows, self.pre_weight.detach(), None, scale, shift, self.norm, self.eps, quantize=True)
        heads = self.qkv.product(normed, dtype=x.dtype).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = torch.split(heads, [self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = ops.kv_append(cache, k, v, pages, lengths, starts, self._frequencies, k_weight=weights[1], q=q, q_weight=weights[0],
                          kind="rms" if self.q_weight is not None else "none", eps=self.eps)
        a = ops.kv_attention(q, cache, pages, lengths, starts, window=self.window)
        h = self.out.product(a.view(-1, self.heads * self.head_dim))
        return ops.block_norm_add(h, rows, self.post_weight.detach(), gate=gate, residual_scale=self.residual_scale, kind=self.norm,
                                  eps=self.eps)


def patch_conv2d():
    """Replace torch.nn.Conv2d with TraceaConv2d for modules constructed afterwards
    (tracea-python/python/tracea/__init__.py:19-26)."""
    torch.nn.Conv2d = TraceaConv2d
