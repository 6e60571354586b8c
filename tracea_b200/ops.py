"""The reference's Python operator surface for Conv2d, on torch tensors, over the C ABI.

Mirrors (paths relative to the reference project's root):
  * ``tracea.ops.conv2d(x, w, bias, residual, epilogue, stride, padding, dilation)`` with x in
    NHWC and w in KRSC memory (tracea-python/python/tracea/ops.py:39-70);
  * ``Context.conv2d(x, w, o, n, c, h, w_in, k, r, s, stride, pad, dilation, epilogue, bias,
    residual)`` and its epilogue grammar ``"bias+relu"``, ``"bias+residual+relu"``
    (src/interface/python.rs:41-87, 367-462);
  * the NCHW / OIHW call the C++ header documents (include/tracea.hpp:101-105) as ``conv2d_nchw``.

torch is used for device memory and streams only. Every call goes through ``tracea_conv2d`` in
libtracea_b200.so; nothing here computes a convolution itself. The calls below hand their tensors to the library through
the ``_ops_native`` module, which builds the C tensor views (csrc/py_ops.cpp); ``ffi`` is the same ABI through ctypes, for
callers that hold raw pointers.
"""
import ctypes
import functools

import torch

from . import ffi

_DTYPES = {torch.float32: ffi.DTYPE_FLOAT32, torch.float16: ffi.DTYPE_FLOAT16,
           torch.bfloat16: ffi.DTYPE_BFLOAT16, torch.int32: ffi.DTYPE_INT32, torch.int8: ffi.DTYPE_INT8}

_ACTS = ("relu", "gelu", "silu")

_native_module = None


def _native():
    """The tensor front end of the library, loaded with it on first use (raises if either has not been built, or the front end
    for another torch)."""
    global _native_module
    if _native_module is None:
        ffi.load()
        from . import _ops_native
        if _ops_native.torch_version != torch.__version__.split("+")[0]:
            raise ImportError("_ops_native was built for torch %s, this is torch %s: build it again with `python -m "
                              "tracea_b200.build`" % (_ops_native.torch_version, torch.__version__))
        _native_module = _ops_native
    return _native_module


@functools.lru_cache(maxsize=256)
def _epilogue_ops(epilogue):
    """The ops of an epilogue string, as a tuple; ValueError on an unknown one."""
    ops = []
    for part in epilogue.split("+"):
        op = part.strip().lower()
        if op == "identity":
            continue
        if op in _ACTS or op in ("bias", "residual"):
            ops.append(op)
        else:
            raise ValueError("Unknown epilogue op: %s" % part)
    return tuple(ops)


_EPILOGUE_KINDS = {
    (): ffi.EPILOGUE_IDENTITY,
    ("bias",): ffi.EPILOGUE_BIAS_ADD,
    ("relu",): ffi.EPILOGUE_RELU,
    ("gelu",): ffi.EPILOGUE_GELU,
    ("silu",): ffi.EPILOGUE_SILU,
    ("bias", "relu"): ffi.EPILOGUE_BIAS_RELU,
    ("bias", "silu"): ffi.EPILOGUE_BIAS_SILU,
    ("residual",): ffi.EPILOGUE_RESIDUAL,
    ("residual", "relu"): ffi.EPILOGUE_RESIDUAL_RELU,
    ("bias", "residual", "relu"): ffi.EPILOGUE_BIAS_RESIDUAL_RELU,
    ("bias", "residual"): ffi.EPILOGUE_BIAS_RESIDUAL,
}


def parse_epilogue(epilogue, bias=None, residual=None):
    """Epilogue string -> TraceaEpilogueKind, with the grammar and the errors of
    src/interface/python.rs:41-87: '+'-separated, case-insensitive ops out of identity, relu, gelu,
    silu, bias, residual; 'bias' / 'residual' without the matching tensor is a ValueError, so is an
    unknown op. The kernel applies bias -> residual -> activation, the order the reference's graph
    fusion produces (tests/fusion_verification.rs:110-170); other orders are rejected."""
    if epilogue is None:
        return ffi.EPILOGUE_IDENTITY
    ops = _epilogue_ops(epilogue)
    if "bias" in ops and bias is None:
        raise ValueError("Epilogue contains 'bias' but no bias argument provided")
    if "residual" in ops and residual is None:
        raise ValueError("Epilogue contains 'residual' but no reference provided")
    kind = _EPILOGUE_KINDS.get(ops)
    if kind is None:
        raise ValueError("Unsupported epilogue sequence %r (supported: %s)" % (
            epilogue, ", ".join("+".join(k) or "identity" for k in _EPILOGUE_KINDS)))
    return kind


def _pair(v):
    if isinstance(v, (tuple, list)):
        return int(v[0]), int(v[1])
    return int(v), int(v)


def _device_id(t):
    return t.device.index if t.is_cuda else -1


def _view(t, shape=None, stride=None):
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise TypeError("unsupported dtype %s" % t.dtype)
    return ffi.View(t.data_ptr(), t.shape if shape is None else shape, t.stride() if stride is None else stride, dt,
                    t.device.index if t.is_cuda else -1)


def _stream_of(t):
    return torch.cuda.current_stream(t.device).cuda_stream if t.is_cuda else 0


def conv2d_into(x, w, out, bias=None, residual=None, stride=1, padding=0, dilation=1, groups=1,
                epilogue=ffi.EPILOGUE_IDENTITY, stream=None):
    """out <- epilogue(conv2d(x, w)) with logical NCHW / OIHW tensors of any strides (a
    ``channels_last`` torch tensor is consumed in place). Enqueues on torch's current stream."""
    if stream is None:
        sh, sw = _pair(stride)
        ph, pw = _pair(padding)
        dh, dw = _pair(dilation)
        return _native().conv2d(x, w, bias, residual, out, False, int(epilogue), sh, sw, ph, pw, dh, dw, groups)
    ffi.conv2d_raw(_view(x), _view(w), _view(bias) if bias is not None else None,
                   _view(residual) if residual is not None else None, _view(out),
                   _pair(stride), _pair(padding), _pair(dilation), groups, epilogue, stream)
    return out


def conv2d_nchw(x, w, bias=None, residual=None, stride=1, padding=0, dilation=1, groups=1, epilogue=None,
                channels_last_out=None):
    """Logical-NCHW convolution (include/tracea.hpp:101-105). The output takes the memory format of
    ``x`` unless ``channels_last_out`` says otherwise."""
    kind = epilogue if isinstance(epilogue, int) else parse_epilogue(epilogue, bias, residual)
    sh, sw = _pair(stride)
    ph, pw = _pair(padding)
    dh, dw = _pair(dilation)
    n, _, h, wi = x.shape
    k, _, r, s = w.shape
    ho = (h + 2 * ph - dh * (r - 1) - 1) // sh + 1
    wo = (wi + 2 * pw - dw * (s - 1) - 1) // sw + 1
    if channels_last_out is None:
        channels_last_out = x.stride(1) == 1 and x.shape[1] > 1
    fmt = torch.channels_last if channels_last_out else torch.contiguous_format
    out = torch.empty((n, k, ho, wo), dtype=x.dtype, device=x.device, memory_format=fmt)
    return _native().conv2d(x, w, bias, residual, out, False, kind, sh, sw, ph, pw, dh, dw, groups)


def conv2d(x, w, bias=None, residual=None, epilogue=None, stride=1, padding=0, dilation=1):
    """tracea.ops.conv2d: x (N, H, W, C) channels-last, w (K, R, S, C), optional bias (K) and
    residual (N, Ho, Wo, K); returns (N, Ho, Wo, K). Same shape checks and messages as
    tracea-python/python/tracea/ops.py:52-61."""
    if x.ndim != 4 or w.ndim != 4:
        raise ValueError("Expected NHWC input and KRSC weight")
    n_batch, h, w_in, c = x.shape
    k, r, s, c_w = w.shape
    if c != c_w:
        raise ValueError(f"Channel mismatch: x({c}) vs w({c_w})")
    sh, sw = _pair(stride)
    ph, pw = _pair(padding)
    dh, dw = _pair(dilation)
    h_out = (h + 2 * ph - dh * (r - 1) - 1) // sh + 1
    w_out = (w_in + 2 * pw - dw * (s - 1) - 1) // sw + 1
    o = torch.empty((n_batch, h_out, w_out, k), dtype=x.dtype, device=x.device)
    kind = parse_epilogue(epilogue, bias, residual)
    return _native().conv2d(x, w, bias, residual, o, True, kind, sh, sw, ph, pw, dh, dw, 1)


def gemm(x, w, bias=None, epilogue=None, residual=None):
    """tracea.ops.gemm (tracea-python/python/tracea/ops.py:12-35): x (M, K) @ w (K, N) -> (M, N) with the conv
    epilogue. Any strides; a ``w`` whose memory is [N][K] (``weight.t()`` of a Linear layer, or the result of
    ``prepack_gemm_b``) is read in place, and so is a row-major one of 16-bit elements whose rows start on 16-byte
    boundaries; any other is transposed into scratch on every call."""
    if x.ndim != 2 or w.ndim != 2:
        raise ValueError("Expected 2D tensors: x (M, K), w (K, N)")
    if x.shape[1] != w.shape[0]:
        raise ValueError(f"Inner dimension mismatch: x({x.shape[1]}) vs w({w.shape[0]})")
    kind = parse_epilogue(epilogue, bias, residual)
    out = torch.empty((x.shape[0], w.shape[1]), dtype=x.dtype, device=x.device)
    return _native().gemm(x, w, bias, residual, out, kind)


def conv_transpose2d(x, w, bias=None, residual=None, epilogue=None, stride=1, padding=0, output_padding=0,
                     dilation=1):
    """tracea.ops.conv_transpose2d (tracea-python/python/tracea/ops.py:72-88): x (N, H, W, C), w (K, R, S, C),
    optional bias (K) and residual (N, Ho, Wo, K); returns (N, Ho, Wo, K) with
    Ho = (H-1)*stride - 2*padding + R + output_padding."""
    if x.ndim != 4 or w.ndim != 4:
        raise ValueError("Expected NHWC input and KRSC weight")
    n_batch, h, w_in, c = x.shape
    k, r, s, c_w = w.shape
    if c != c_w:
        raise ValueError(f"Channel mismatch: x({c}) vs w({c_w})")
    sh, sw = _pair(stride)
    ph, pw = _pair(padding)
    oh, ow = _pair(output_padding)
    h_out = (h - 1) * sh - 2 * ph + r + oh
    w_out = (w_in - 1) * sw - 2 * pw + s + ow
    kind = parse_epilogue(epilogue, bias, residual)
    o = torch.empty((n_batch, h_out, w_out, k), dtype=x.dtype, device=x.device)
    dh, dw = _pair(dilation)
    return _native().conv_transpose2d(x, w, bias, residual, o, kind, sh, sw, ph, pw, oh, ow, dh, dw)


def prepack_conv2d_weight(w):
    """OIHW-shaped weights of any strides -> a tensor of the same logical shape (channels rounded up to 16 bytes)
    whose memory is the dense [K][R][S][C] layout the kernel reads in place (tracea_conv2d_prepack)."""
    lib = ffi.load()
    v = _view(w)
    nbytes = lib.tracea_conv2d_prepack_bytes(v.c)
    shape = (ctypes.c_uint64 * 4)()
    stride = (ctypes.c_int64 * 4)()
    buf = torch.empty(nbytes // w.element_size(), dtype=w.dtype, device=w.device)
    st = lib.tracea_conv2d_prepack(v.c, buf.data_ptr(), nbytes, shape, stride, _stream_of(w))
    if st != ffi.SUCCESS:
        raise ffi.TraceaError(st, ffi.last_error(), "tracea_conv2d_prepack")
    return torch.as_strided(buf, tuple(int(d) for d in shape), tuple(int(d) for d in stride))


def prepack_gemm_b(b):
    """(K, N) matrix of any strides -> a (K, N) tensor whose memory is [N][K] (tracea_gemm_prepack_b)."""
    lib = ffi.load()
    v = _view(b)
    nbytes = lib.tracea_gemm_prepack_b_bytes(v.c)
    stride = (ctypes.c_int64 * 2)()
    buf = torch.empty(nbytes // b.element_size(), dtype=b.dtype, device=b.device)
    st = lib.tracea_gemm_prepack_b(v.c, buf.data_ptr(), nbytes, stride, _stream_of(b))
    if st != ffi.SUCCESS:
        raise ffi.TraceaError(st, ffi.last_error(), "tracea_gemm_prepack_b")
    return torch.as_strided(buf, tuple(b.shape), (int(stride[0]), int(stride[1])))


class MxTensor:
    """A (rows, cols) matrix in the 4-bit microscaled format of include/tracea_b200.h (TraceaMxMatrix): ``data``, uint8 of shape
    (rows, 16 * ceil(cols / 32)), and ``scales``, uint8 of shape (ceil(rows / 128), ceil(cols / 128), 512)."""

    __slots__ = ("data", "scales", "shape")

    def __init__(self, data, scales, shape):
        self.data, self.scales, self.shape = data, scales, shape

    @property
    def device(self):
        return self.data.device

    def dequantize(self, dtype=torch.bfloat16):
        return mx_dequantize(self, dtype)

    def __repr__(self):
        return "MxTensor(%d x %d, device=%s)" % (self.shape[0], self.shape[1], self.data.device)


def mx_quantize(x):
    """x (M, K), any strides -> MxTensor: blocks of 32 columns with a power-of-two scale and 4-bit elements, a quarter of the
    memory of 16-bit values and a bit. The scale is the largest power of two whose quadruple does not pass the block's largest
    value; elements are rounded to nearest, ties to even, and saturate at 6 scales. A block with a NaN or an infinity becomes
    NaN."""
    data, scales = _native().mx_quantize(x)
    return MxTensor(data, scales, tuple(x.shape))


def mx_dequantize(q, dtype=torch.bfloat16):
    """The values of an MxTensor; exact in bfloat16 and float32."""
    return _native().mx_dequantize(q.data, q.scales, q.shape[0], q.shape[1], _DTYPES.get(dtype, -1))


def mx_gemm(a, w, bias=None, epilogue=None, residual=None, dtype=None, quantize=False):
    """a (M, K) times the transpose of w (N, K) -> (M, N), with the epilogue of ``gemm``, on the block-scaled tensor cores.

    w is an MxTensor, a Linear layer's weight as it lies; a is an MxTensor or a tensor that the call quantises first. The output
    has ``dtype`` (default: the type of a, bfloat16 for an MxTensor), or with ``quantize`` is an MxTensor itself, quantised from
    the fp32 results. ``bias`` (N): float32 or the output's type; ``residual`` (M, N): the output's type, not with ``quantize``."""
    kind = parse_epilogue(epilogue, bias, residual)
    if not isinstance(w, MxTensor):
        raise TypeError("w must be an MxTensor")
    n, k = w.shape
    if len(a.shape) != 2:
        raise ValueError("Expected a 2D tensor: a (M, K)")
    m, k_a = a.shape
    if k_a != k:
        raise ValueError(f"Inner dimension mismatch: a({k_a}) vs w({k})")
    if isinstance(a, MxTensor):
        data, scales, out = a.data, a.scales, torch.bfloat16
    else:
        data, scales, out = a, None, a.dtype
    if dtype is not None:
        if quantize:
            raise ValueError("either dtype or quantize")
        out = dtype
    r = _native().mx_gemm(data, scales, m, w.data, w.scales, n, k, bias, residual, kind, None if quantize else _DTYPES.get(out, -1))
    return MxTensor(*r, (m, n)) if quantize else r


_NORM_KINDS = {"none": ffi.NORM_NONE, "rms": ffi.NORM_RMS, "layer": ffi.NORM_LAYER}


def _norm_kind(kind):
    if kind not in _NORM_KINDS:
        raise ValueError("Unknown norm: %s (supported: %s)" % (kind, ", ".join(_NORM_KINDS)))
    return _NORM_KINDS[kind]


def block_norm(x, weight=None, bias=None, scale=None, shift=None, kind="rms", eps=1e-6, quantize=False):
    """The norm in front of a block: (norm(x) * weight + bias) * (1 + scale) + shift for x (M, C), in one pass.

    kind "rms": v / sqrt(mean(v^2) + eps), "layer": (v - mean) / sqrt(var + eps), "none": v. weight, bias (C); scale, shift
    (G, C) where G divides M: each row of them serves M / G consecutive rows of x, an image's positions for example. All float32
    or x's type. Returns x's type, or with ``quantize`` an MxTensor for ``mx_gemm``."""
    r = _native().block_norm(x, weight, bias, scale, shift, _norm_kind(kind), eps, quantize)
    return MxTensor(*r, tuple(x.shape)) if quantize else r


def block_norm_add(h, x, weight=None, bias=None, scale=None, shift=None, gate=None, residual_scale=1.0, kind="rms", eps=1e-6,
                   following=None):
    """The join behind a block: r = residual_scale * x + gate * block_norm(h, ...), h the block's output, x the stream it started
    from, both (M, C) of one type; gate (G, C) as scale, or None. kind "none" joins h as it is.

    following: the next block's norm, a dict of the keyword arguments of ``block_norm``; then (r, y) is returned, with
    y = block_norm(r, **following), from the same pass over the rows. The same bits where the rows of h and x are 16-byte aligned,
    as r's are where C is a multiple of 8 (or C is not one); else the sums of y's norm are taken in another order."""
    if following is None:
        return _native().block_norm_add(h, x, weight, bias, scale, shift, _norm_kind(kind), eps, gate, residual_scale, 0)
    return _norm_add_following(h, x, (weight, bias, scale, shift, _norm_kind(kind), eps, gate, residual_scale), **following)


def _norm_add_following(h, x, first, weight=None, bias=None, scale=None, shift=None, kind="rms", eps=1e-6, quantize=False):
    r, y = _native().block_norm_add(h, x, *first, 2 if quantize else 1, weight, bias, scale, shift, _norm_kind(kind), eps)
    return r, MxTensor(*y, tuple(x.shape)) if quantize else y


def rotary_frequencies(columns, base=10000.0, device=None):
    """The usual angles per position of a rotation of ``columns`` columns, base^(-2i / columns) for pair i: float64, (columns / 2)."""
    if columns % 2 != 0:
        raise ValueError("a rotation takes an even number of columns")
    return torch.pow(float(base), -torch.arange(0, columns, 2, dtype=torch.float64, device=device) / columns)


def head_norm_rotate(q, k, positions=None, frequencies=None, interleaved=False, q_weight=None, k_weight=None, kind="rms", eps=1e-6):
    """Queries and keys between their projections and attention: each head's columns normalised, times a weight, and rotated by the
    token's position, in one pass. Returns new (q, k).

    q (T, H, D) and k (T, H', D), either may be None; their columns are contiguous, other strides any (slices of one projection, say);
    float32, float16 or bfloat16, D even and at most 256. kind "rms" or "none"; weights (D), float32 or the rows' type, with either kind.
    positions (T), int32, and frequencies, float64 radians per position (``rotary_frequencies``): pair i of the first
    2 * len(frequencies) columns, columns 2i and 2i + 1 if ``interleaved`` and i and i + len(frequencies) if not, is turned by
    positions * frequencies[i], an angle that is computed in 64 bits."""
    return _native().head_norm_rotate(q, k, positions, frequencies, interleaved, q_weight, k_weight, _norm_kind(kind), eps)


class KvCache:
    """Keys and values in 8 bits, in pages (TraceaKvCache of include/tracea_b200.h): ``k`` and ``v``, float8_e4m3fn of shape (pages,
    heads, page_size, head_dim), and ``k_scales``, ``v_scales``, uint8 of shape (pages, heads): a page's and head's elements stand for
    2^(byte - 127) times themselves. ``kv_append`` fills it, ``kv_attention`` reads it; a sequence's pages are the caller's to hand out."""

    __slots__ = ("k", "v", "k_scales", "v_scales")

    def __init__(self, k, v, k_scales, v_scales):
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales

    @classmethod
    def empty(cls, pages, heads, head_dim, page_size=64, device="cuda"):
        """A cache of ``pages`` pages of ``page_size`` (16, 32, 64 or 128) tokens, ``head_dim`` a multiple of 16 up to 128. All zeros."""
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128")
        if head_dim % 16 != 0 or not 16 <= head_dim <= 128:
            raise ValueError("head_dim must be a multiple of 16 up to 128")
        k, v = (torch.zeros((pages, heads, page_size, head_dim), dtype=torch.uint8, device=device) for _ in "kv")
        ks, vs = (torch.full((pages, heads), 87, dtype=torch.uint8, device=device) for _ in "kv")
        return cls(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs)

    @property
    def device(self):
        return self.k.device

    @property
    def page_size(self):
        return self.k.shape[2]

    def __repr__(self):
        return "KvCache(%d pages of %d tokens, %d heads of %d, device=%s)" % (self.k.shape[0], self.k.shape[2], self.k.shape[1],
                                                                             self.k.shape[3], self.k.device)


def kv_append(cache, k, v, pages, lengths, starts=None, frequencies=None, interleaved=False, k_weight=None, q=None, q_weight=None,
              kind="none", eps=1e-6):
    """Puts new tokens' keys and values into ``cache``, the keys normalised and rotated on the way as ``head_norm_rotate`` does, by the
    tokens' positions in their sequences. With ``q``, the queries of the same tokens, (T, H, D) with H a multiple of the cache's heads,
    returns them normalised and rotated, from the same launch.

    k, v (T, heads, D): the last tokens of the sequences. int32 tensors, read on the device: ``lengths`` (B), each sequence's tokens, the
    new ones included; ``pages`` (B, width), its pages: token j lies in row j % page_size of page pages[s, j // page_size], and is dropped
    where that is no page of the cache; ``starts`` (B + 1): rows starts[s] .. starts[s + 1] - 1 belong to sequence s -- None: row s is
    the one new token of sequence s. A page that a call writes to stands in one place of one sequence; such as are only read may be shared.
    Rows of no sequence are not read, and not set in the result.

    A block, the tokens of a page and head, has one scale: the smallest power of two 2^e of which 448 reach its largest value,
    -40 <= e <= 40. It grows when a larger value is appended, and the block's older tokens are then rounded anew; a page's first token
    starts it afresh. A token with a key or value in a head that is not finite is kept there as a NaN key and a zero value."""
    return _native().kv_append(cache.k, cache.v, cache.k_scales, cache.v_scales, pages, lengths, starts, k, v, k_weight, q, q_weight,
                               frequencies, interleaved, _norm_kind(kind), eps)


def kv_attention(q, cache, pages, lengths, starts=None, scale=None, causal=True, window=0):
    """Attention of queries (T, H, D), float16 or bfloat16, to the tokens of their sequences in ``cache``; ``pages``, ``lengths`` and
    ``starts`` as in ``kv_append``, after which it is called. H a multiple of the cache's heads: H / heads consecutive heads of q share
    one of the cache. scale: 1 / sqrt(D) unless given.

    Rows see their sequence up to their own position (``causal``) or all of it, and with ``window`` no tokens more than window - 1
    positions in front of their own. A row that sees no token gives 0.

    Scores, softmax and sums are held in float32, two factors of the products in halves: q, whose elements below 2^-14 of their row's
    largest are off by up to 2^-25 of it, and the tokens' weights times their values' scales, to 11 bits or by up to 2^-32 of the row's
    largest. float16 results are off by 1.0 - 1.4 times as much as with all in float32, bfloat16 results by the same."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _native().kv_attention(q, cache.k, cache.v, cache.k_scales, cache.v_scales, pages, lengths, starts, scale, causal, window)


class Context:
    """Stand-in for the reference's ``tracea.Context`` (src/interface/python.rs:367-462), Conv2d only.
    The reference builds an IR, generates CUDA text and compiles it here; this one forwards to the
    precompiled library."""

    def conv2d(self, x, w, o, n, c, h, w_in, k, r, s, stride=1, pad=0, dilation=1, epilogue=None, bias=None,
               residual=None):
        kind = parse_epilogue(epilogue, bias, residual)
        if tuple(x.shape) != (n, h, w_in, c) or tuple(w.shape) != (k, r, s, c):
            raise ValueError("x must be (n, h, w_in, c) and w must be (k, r, s, c)")
        sh, sw = _pair(stride)
        ph, pw = _pair(pad)
        dh, dw = _pair(dilation)
        _native().conv2d(x, w, bias, residual, o, True, kind, sh, sw, ph, pw, dh, dw, 1)
        return 0

    def synchronize(self):
        torch.cuda.synchronize()
