"""The 4-bit microscaled operators and the norms around them, as cases to be timed: quantisation, matrix products of
quantised operands, the norm in front of a block, the gated join behind it, and a feed-forward block made of all four.

Format ("mx"): blocks of 32 consecutive columns share a power-of-two scale, 2^(byte - 127) with byte 255 for NaN; an element
is a sign, two exponent bits and one mantissa bit (0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte, the even column in the low half.
A matrix of M rows and K columns is `data`, M rows of 16 * ceil(K / 32) bytes, and `scales`, tiles of 128 rows x 4 blocks: the
byte of row r, block b is byte 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4 of tile [r // 128][b // 4].

Sizes are those of the repository's own benchmark configurations and layer table (14 x 14 maps of 1024 channels, the 2048-wide
classifier head, the 8192-wide product) or generic ones. The framework computes forward passes only, so there is one direction.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}

# Bounds of a drawn case: below the largest listed ones.
_MAX_BYTES = 3e8
_MAX_FLOPS = 3e11


# ------------------------------------------------------------------------------------------------------------ the cases
def _quantize(name, dtype, m, k, pad=0):
    return {"name": name, "kind": "quantize", "dtype": dtype, "m": m, "k": k, "pad": pad}


def _gemm(name, dtype, m, n, k, epilogue, quantized_input):
    return {"name": name, "kind": "gemm", "dtype": dtype, "m": m, "n": n, "k": k, "epilogue": epilogue,
            "quantized_input": quantized_input}


def _norm(name, dtype, m, c, norm, groups, affine, pad=0):
    return {"name": name, "kind": "norm", "dtype": dtype, "m": m, "c": c, "norm": norm, "groups": groups, "affine": affine,
            "pad": pad}


def _join(name, dtype, m, c, norm, groups, affine, residual_scale, following, pad=0):
    return {"name": name, "kind": "join", "dtype": dtype, "m": m, "c": c, "norm": norm, "groups": groups, "affine": affine,
            "residual_scale": residual_scale, "following": following, "pad": pad}


def listed():
    return [
        # one pooled feature vector in front of the classifier head: the smallest call, where latency counts
        _quantize("quantize_row_f16", "f16", 1, 2048),
        # fp32 features that are a slice of a wider buffer, columns no multiple of a block: user-written networks
        _quantize("quantize_odd_f32", "f32", 777, 1000, 3),
        # activations of a large batch on their way into a 4-bit layer
        _quantize("quantize_large_bf16", "bf16", 16384, 4096),
        # a single token through a linear layer: 16-bit activations in, 4-bit weights, as when answers are generated
        _gemm("gemm_token_bf16", "bf16", 1, 4096, 4096, "bias", False),
        # the classifier head on a small batch
        _gemm("gemm_head_f16", "f16", 64, 1000, 2048, "bias", True),
        # nothing is a multiple of anything, fp32 in and out of the epilogue with a skip connection
        _gemm("gemm_odd_f32", "f32", 1500, 1030, 777, "bias+residual", True),
        # the benchmark's large square product: the largest case
        _gemm("gemm_square_bf16", "bf16", 8192, 8192, 8192, "", True),
        # the norm in front of a block for a single token
        _norm("norm_row_bf16", "bf16", 1, 4096, "rms", 0, "weight"),
        # 64 images of 14 x 14 positions, 1024 channels, the norm modulated per image by its conditioning
        _norm("norm_images_bf16", "bf16", 12544, 1024, "layer", 64, ""),
        # the join behind a block on an odd number of odd rows in fp32, affine layer norm, a gate per sample
        _join("join_odd_f32", "f32", 333, 1001, "layer", 3, "weight+bias", 1.0, "", 5),
        # the join of a large batch with a scaled residual and the next block's norm in the same pass
        _join("join_next_bf16", "bf16", 16384, 2048, "rms", 1, "weight", 0.5, "rms"),
        # a whole feed-forward block on 64 images: norm, up with SiLU, down, join; both products read 4-bit operands
        {"name": "feed_forward_bf16", "kind": "block", "dtype": "bf16", "m": 12544, "c": 1024, "hidden": 4096, "groups": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Half of them multiples of 128, a quarter multiples of 8, a quarter anything."""
    u, v = rng.random(), _log(rng, lo, hi)
    return 128 * max(1, v // 128) if u < 0.5 else 8 * max(1, v // 8) if u < 0.75 else v


def _draw_once(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kind = rng.choice(["quantize", "gemm", "gemm", "gemm", "norm", "join", "block"])
    if kind == "quantize":
        return _quantize("", dtype, _log(rng, 1, 16384), _width(rng, 8, 8192), rng.choice([0, 0, 1, 8]))
    if kind == "gemm":
        return _gemm("", dtype, _log(rng, 1, 8192), _width(rng, 16, 8192), _width(rng, 16, 8192),
                     rng.choice(["", "bias", "bias+relu", "bias+silu", "gelu", "residual", "bias+residual"]), rng.random() < 0.6)
    if kind == "block":
        c = _width(rng, 32, 2048)
        groups = rng.choice([1, 1, 2, 8])
        return {"kind": "block", "dtype": rng.choice(["bf16", "f16"]), "m": groups * _log(rng, 1, 2048), "c": c, "hidden": _width(rng, c, 4 * c),
                "groups": groups}
    groups = rng.choice([0, 1, 1, 3, 16])
    m = max(1, groups) * _log(rng, 1, 16384 // max(1, groups))
    args = ("", dtype, m, _width(rng, 8, 8192), rng.choice(["rms", "layer"]), groups, rng.choice(["", "weight", "weight+bias"]))
    if kind == "norm":
        return _norm(*args, rng.choice([0, 0, 1, 8]))
    return _join(*args, rng.choice([1.0, 0.5, 0.25]), rng.choice(["", "rms", "layer"]), rng.choice([0, 0, 1, 8]))


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS:
            case.pop("name", None)
            return case


# ----------------------------------------------------------------------------------------------------------- the inputs
def _features(gen, m, c, dtype, pad=0):
    """Rows as networks have them: normal values whose channels differ in size, a few of them by far."""
    spread = torch.exp(0.7 * torch.randn(c, generator=gen, device="cuda"))
    x = (torch.randn(m, c, generator=gen, device="cuda") * spread).to(_DT[dtype])
    if not pad:
        return x
    wide = torch.zeros(m, c + pad, dtype=_DT[dtype], device="cuda")
    wide[:, :c] = x
    return wide[:, :c]


def _stored(values):
    """A float32 matrix as a checkpoint in this format holds it: (data, scales)."""
    m, k = values.shape
    blocks, tiles = -(-k // 32), -(-k // 128)
    x = torch.nn.functional.pad(values, (0, 32 * blocks - k)).view(m, blocks, 32)
    peak = x.abs().amax(-1)
    e = torch.where(peak > 0, torch.frexp(peak).exponent - 3, torch.full_like(peak, -127, dtype=torch.int32)).clamp(-127, 125)
    a = torch.ldexp(x.abs(), -e[..., None])
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.searchsorted(torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device), q.contiguous())
    code = (code + 8 * (x < 0)).to(torch.uint8).view(m, 16 * blocks, 2)
    data = code[..., 0] | (code[..., 1] << 4)
    rows = -(-m // 128)
    s = torch.zeros(rows * 128, tiles * 4, dtype=torch.uint8, device=x.device)
    s[:m, :blocks] = (e + 127).to(torch.uint8)
    scales = s.view(rows, 4, 32, tiles, 4).permute(0, 3, 2, 1, 4).reshape(rows, tiles, 512)
    return data.contiguous(), scales.contiguous()


def _weights(gen, n, k):
    return _stored(torch.randn(n, k, generator=gen, device="cuda") * (2.0 / k) ** 0.5)


def _vector(gen, c, mean, size):
    return mean + size * torch.randn(c, generator=gen, device="cuda")


def _affine(gen, case, s):
    s["weight"] = _vector(gen, case["c"], 1.0, 0.1) if "weight" in case["affine"] else None
    s["bias"] = _vector(gen, case["c"], 0.0, 0.1) if "bias" in case["affine"] else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    kind, dtype, m = case["kind"], case["dtype"], case["m"]
    if kind == "quantize":
        s["x"] = _features(gen, m, case["k"], dtype, case["pad"])
    elif kind == "gemm":
        n, k = case["n"], case["k"]
        x = _features(gen, m, k, dtype)
        s["x"] = None if case["quantized_input"] else x
        s["x_mx"] = _stored(x.float()) if case["quantized_input"] else None
        s["w_mx"] = _weights(gen, n, k)
        s["bias"] = _vector(gen, n, 0.0, 0.1) if "bias" in case["epilogue"] else None
        s["residual"] = torch.randn(m, n, generator=gen, device="cuda").to(_DT[dtype]) if "residual" in case["epilogue"] else None
    elif kind == "norm":
        s["x"] = _features(gen, m, case["c"], dtype, case["pad"])
        _affine(gen, case, s)
        s["scale"] = 0.3 * torch.randn(case["groups"], case["c"], generator=gen, device="cuda") if case["groups"] else None
        s["shift"] = 0.3 * torch.randn(case["groups"], case["c"], generator=gen, device="cuda") if case["groups"] else None
    elif kind == "join":
        s["x"] = _features(gen, m, case["c"], dtype, case["pad"])
        s["h"] = _features(gen, m, case["c"], dtype)
        _affine(gen, case, s)
        s["gate"] = 0.3 * torch.randn(case["groups"], case["c"], generator=gen, device="cuda") if case["groups"] else None
        s["next_weight"] = _vector(gen, case["c"], 1.0, 0.1) if case["following"] else None
    else:
        c, hidden = case["c"], case["hidden"]
        s["x"] = _features(gen, m, c, dtype)
        s["weight"], s["post_weight"] = _vector(gen, c, 1.0, 0.1), _vector(gen, c, 1.0, 0.1)
        s["gate"] = 0.3 * torch.randn(case["groups"], c, generator=gen, device="cuda")
        s["up_mx"], s["up_bias"] = _weights(gen, hidden, c), _vector(gen, hidden, 0.0, 0.1)
        s["down_mx"], s["down_bias"] = _weights(gen, c, hidden), _vector(gen, c, 0.0, 0.1)
    return s


# ------------------------------------------------------------------------------------------------------- the plain forms
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _plain_values(x):
    """x as the format holds it, in float32."""
    m, k = x.shape
    blocks = -(-k // 32)
    v = torch.nn.functional.pad(x.float(), (0, 32 * blocks - k)).view(m, blocks, 32)
    peak = v.abs().amax(-1, keepdim=True)
    e = torch.where(peak > 0, torch.frexp(peak).exponent - 3, torch.full_like(peak, -127, dtype=torch.int32)).clamp(-127, 125)
    v = torch.ldexp(v, -e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)
    return torch.ldexp(q, e).view(m, 32 * blocks)[:, :k]


def _plain_unpack(stored, k):
    data, scales = stored
    m, blocks = data.shape[0], data.shape[1] // 16
    codes = torch.stack((data & 15, data >> 4), dim=-1).view(m, 32 * blocks)
    v = torch.tensor(_VALUES, device=data.device)[codes.long()].view(m, blocks, 32)
    rows, tiles = scales.shape[:2]
    e = scales.view(rows, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(128 * rows, 4 * tiles)[:m, :blocks].to(torch.int32) - 127
    return torch.ldexp(v, e[..., None]).view(m, 32 * blocks)[:, :k]


def _plain_norm(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    y = y * weight.to(y.dtype) if weight is not None else y
    return y + bias.to(y.dtype) if bias is not None else y


def _per_row(t, m):
    return t.repeat_interleave(m // t.shape[0], dim=0)


def _plain_epilogue(y, epilogue, bias, residual):
    if bias is not None:
        y = y + bias.to(y.dtype)
    if residual is not None:
        y = y + residual.to(y.dtype)
    if "relu" in epilogue:
        y = torch.clamp(y, min=0)
    elif "silu" in epilogue:
        y = y / (1 + torch.exp(-y))
    elif "gelu" in epilogue:
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain(s):
    case = s["case"]
    kind, out, m = case["kind"], _DT[case["dtype"]], case["m"]
    if kind == "quantize":
        return _plain_values(s["x"]).to(torch.bfloat16)
    if kind == "gemm":
        x = _plain_values(s["x"]) if s["x"] is not None else _plain_unpack(s["x_mx"], case["k"])
        return _plain_epilogue(x @ _plain_unpack(s["w_mx"], case["k"]).t(), case["epilogue"], s["bias"], s["residual"]).to(out)
    if kind == "norm":
        y = _plain_norm(s["x"].float(), case["norm"], s["weight"], s["bias"])
        if s["scale"] is not None:
            y = y * (1 + _per_row(s["scale"], m)) + _per_row(s["shift"], m)
        return y.to(out)
    if kind == "join":
        y = _plain_norm(s["h"].float(), case["norm"], s["weight"], s["bias"])
        if s["gate"] is not None:
            y = y * _per_row(s["gate"], m)
        r = (case["residual_scale"] * s["x"].float() + y).to(out)
        if not case["following"]:
            return r
        return r, _plain_norm(r.float(), case["following"], s["next_weight"], None).to(out)
    y = _plain_values(_plain_norm(s["x"].float(), "rms", s["weight"], None))
    u = _plain_epilogue(y @ _plain_unpack(s["up_mx"], case["c"]).t(), "bias+silu", s["up_bias"], None)
    h = (_plain_values(u) @ _plain_unpack(s["down_mx"], case["hidden"]).t() + s["down_bias"]).to(out)
    y = _plain_norm(h.float(), "rms", s["post_weight"], None) * _per_row(s["gate"], m)
    return (s["x"].float() + y).to(out)


# --------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from tracea_b200 import ops
    case = s["case"]
    kind, dtype, m = case["kind"], _DT[case["dtype"]], case["m"]
    if kind == "quantize":
        return ops.mx_dequantize(ops.mx_quantize(s["x"]))
    if kind == "gemm":
        x = s["x"] if s["x"] is not None else ops.MxTensor(*s["x_mx"], (m, case["k"]))
        return ops.mx_gemm(x, ops.MxTensor(*s["w_mx"], (case["n"], case["k"])), s["bias"], case["epilogue"] or None,
                           s["residual"], dtype=dtype)
    if kind == "norm":
        return ops.block_norm(s["x"], s["weight"], s["bias"], scale=s["scale"], shift=s["shift"], kind=case["norm"])
    if kind == "join":
        following = {"weight": s["next_weight"], "kind": case["following"]} if case["following"] else None
        return ops.block_norm_add(s["h"], s["x"], s["weight"], s["bias"], gate=s["gate"],
                                  residual_scale=case["residual_scale"], kind=case["norm"], following=following)
    q = ops.block_norm(s["x"], s["weight"], kind="rms", quantize=True)
    u = ops.mx_gemm(q, ops.MxTensor(*s["up_mx"], (case["hidden"], case["c"])), s["up_bias"], "bias+silu", quantize=True)
    h = ops.mx_gemm(u, ops.MxTensor(*s["down_mx"], (case["c"], case["hidden"])), s["down_bias"], "bias", dtype=dtype)
    return ops.block_norm_add(h, s["x"], s["post_weight"], gate=s["gate"], kind="rms")


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------- work and truth
def _mx_bytes(rows, cols):
    return rows * cols * (0.5 + 1.0 / 32)


def work(case):
    kind, m, es = case["kind"], case["m"], _SIZE[case["dtype"]]
    if kind == "quantize":
        return {"bytes": m * case["k"] * (es + 2), "flops": 0}
    if kind == "gemm":
        n, k = case["n"], case["k"]
        x = _mx_bytes(m, k) if case["quantized_input"] else m * k * es
        res = m * n * es if "residual" in case["epilogue"] else 0
        return {"bytes": x + _mx_bytes(n, k) + m * n * es + res, "flops": 2.0 * m * n * k}
    c = case["c"]
    if kind == "norm":
        return {"bytes": 2 * m * c * es + 8 * case["groups"] * c, "flops": 0}
    if kind == "join":
        return {"bytes": (4 if case["following"] else 3) * m * c * es + 4 * case["groups"] * c, "flops": 0}
    hidden = case["hidden"]
    return {"bytes": 2 * m * c * es + 2 * _mx_bytes(hidden, c), "flops": 4.0 * m * c * hidden}


def _exact_values(x):
    """Nearest of the format's values, found by comparing with the borders between them; a tie goes to the even code."""
    m, k = x.shape
    blocks = -(-k // 32)
    full = torch.zeros(m, 32 * blocks, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    v = full.view(m, blocks, 32)
    scale = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().amax(-1, keepdim=True).clamp(min=1e-300))) - 2, -127, 125))
    # log2 may be off by an ulp next to a power of two
    scale = torch.where(v.abs().amax(-1, keepdim=True) >= 8 * scale, 2 * scale, scale)
    scale = torch.where((v.abs().amax(-1, keepdim=True) < 4 * scale) & (scale > 2.0 ** -127), scale / 2, scale)
    a = (v / scale).abs()
    code = (a > 0.25).long() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    q = torch.tensor(_VALUES[:8], dtype=torch.float64, device=x.device)[code] * torch.sign(v) * scale
    return q.view(m, 32 * blocks)[:, :k]


def _exact_unpack(stored, k):
    """What (data, scales) stand for, element by element from where the format says it lies."""
    data, scales = stored
    m = data.shape[0]
    r = torch.arange(m, device=data.device)[:, None]
    col = torch.arange(k, device=data.device)[None, :]
    code = (data[:, :(k + 1) // 2].repeat_interleave(2, dim=1)[:, :k].long() >> (4 * (col % 2))) & 15
    power, half = (code & 7) >> 1, code & 1
    size = torch.where(power == 0, 0.5 * half, (1 + 0.5 * half) * torch.exp2((power - 1).double()))
    b = col // 32
    at = ((r // 128) * scales.shape[1] + b // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4
    scale = torch.exp2(scales.reshape(-1)[at].double() - 127)
    return torch.where(code >= 8, -size, size) * scale


def _exact_norm(x, kind, weight, bias, m):
    mean = x.mean(1, keepdim=True) if kind == "layer" else 0.0
    d = x - mean
    y = d / torch.sqrt((d * d).sum(1, keepdim=True) / x.shape[1] + 1e-6)
    y = y if weight is None else y * weight.double()
    return y if bias is None else y + bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    kind, m = case["kind"], case["m"]

    def rows(t):
        return t.double()[torch.arange(m, device=t.device) // (m // t.shape[0])]

    def finish(y, epilogue, bias, residual):
        y = y if bias is None else y + bias.double()
        y = y if residual is None else y + residual.double()
        if "relu" in epilogue:
            return torch.where(y > 0, y, torch.zeros_like(y))
        if "silu" in epilogue:
            return y * torch.sigmoid(y)
        if "gelu" in epilogue:
            return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y

    if kind == "quantize":
        return _exact_values(s["x"].double())
    if kind == "gemm":
        x = _exact_values(s["x"].double()) if s["x"] is not None else _exact_unpack(s["x_mx"], case["k"])
        w = _exact_unpack(s["w_mx"], case["k"])
        return finish(torch.matmul(x, w.t()), case["epilogue"], s["bias"], s["residual"])
    if kind == "norm":
        y = _exact_norm(s["x"].double(), case["norm"], s["weight"], s["bias"], m)
        return y if s["scale"] is None else y + y * rows(s["scale"]) + rows(s["shift"])
    if kind == "join":
        y = _exact_norm(s["h"].double(), case["norm"], s["weight"], s["bias"], m)
        r = case["residual_scale"] * s["x"].double() + (y if s["gate"] is None else y * rows(s["gate"]))
        if not case["following"]:
            return r
        # the next norm reads what is stored
        return r, _exact_norm(r.to(_DT[case["dtype"]]).double(), case["following"], s["next_weight"], None, m)
    y = _exact_values(_exact_norm(s["x"].double(), "rms", s["weight"], None, m))
    u = finish(y @ _exact_unpack(s["up_mx"], case["c"]).t(), "silu", s["up_bias"], None)
    h = _exact_values(u) @ _exact_unpack(s["down_mx"], case["hidden"]).t() + s["down_bias"].double()
    h = h.to(_DT[case["dtype"]]).double()   # a product is stored in the data type
    return s["x"].double() + _exact_norm(h, "rms", s["post_weight"], None, m) * rows(s["gate"])
