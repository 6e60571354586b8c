"""The 4-bit microscaled format, its products and the norms around a block, in numpy and 64 bits, from their definitions: what
test_mx_*.py and test_block_norm_*.py compare with. Nothing here calls the library."""
import numpy as np

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
BORDERS = (VALUES[:-1] + VALUES[1:]) / 2          # a tie goes to the neighbour with the even code


def encode(x):
    """(codes (M, 32 * blocks), scale bytes (M, blocks)) of a float matrix."""
    x = np.asarray(x, dtype=np.float64)
    m, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((m, 32 * blocks))
    v[:, :k] = x
    v = v.reshape(m, blocks, 32)
    bad = ~np.isfinite(v).all(-1)
    with np.errstate(invalid="ignore"):
        peak = np.abs(np.where(bad[..., None], 0.0, v)).max(-1)
    e = np.where(peak > 0, np.frexp(peak)[1] - 1 - 2, -127)
    e = np.clip(e, -127, 125)
    a = np.abs(np.where(bad[..., None], 0.0, v)) / np.exp2(e)[..., None]
    code = np.zeros(a.shape, dtype=np.int64)
    for i, b in enumerate(BORDERS):               # code i + 1 from border i on: inclusive where i + 1 is even
        code += (a >= b) if (i + 1) % 2 == 0 else (a > b)
    code = code + 8 * np.signbit(v)
    code[bad] = 0
    return code.reshape(m, 32 * blocks).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes, scales):
    """Values of (M, 32 * blocks) codes and (M, blocks) scale bytes."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=1)


def pack(codes, scales):
    """(data, scales) bytes as TraceaMxMatrix lays them out; scale bytes of rows past the last one are 255 here, NaN, so that a
    result that depended on them would show it."""
    m, blocks = scales.shape
    data = (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)
    rows, tiles = -(-m // 128), -(-blocks // 4)
    out = np.full((rows, tiles, 512), 255, dtype=np.uint8)
    for r in range(rows * 128):
        for b in range(4 * tiles):
            if r < m:
                out[r // 128, b // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4] = scales[r, b] if b < blocks else 0
    return data, out


def unpack(data, scales, m, k):
    """The inverse of pack: (codes, scale bytes (M, blocks), the scale bytes behind the last block)."""
    blocks, tiles = -(-k // 32), -(-k // 128)
    codes = np.empty((m, 32 * blocks), dtype=np.uint8)
    codes[:, 0::2] = data & 15
    codes[:, 1::2] = data >> 4
    r = np.arange(m)[:, None]
    b = np.arange(4 * tiles)[None, :]
    s = scales.reshape(-1)[((r // 128) * tiles + b // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4]
    return codes, s[:, :blocks], s[:, blocks:]


def values(x):
    """x as the format holds it."""
    k = np.asarray(x).shape[1]
    return decode(*encode(x))[:, :k]


def activation(y, act):
    if act == "relu":
        return np.maximum(y, 0)
    if act == "silu":
        with np.errstate(over="ignore"):
            return y / (1 + np.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + np.tanh(np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3)))
    return y


def norm(x, kind, eps, weight=None, bias=None, scale=None, shift=None):
    """(result, bound on the error of an fp32 computation of it, before the output's rounding).

    The bound: sums over a row are of at most 32 terms in a thread and 5 + 4 steps across threads, so a sum of C terms is off by
    less than 64 half steps (2^-24) of the sum of its terms' sizes. That shifts the mean by 64 2^-24 mean|x|, and the factor
    1 / sqrt(.) by as much relative to itself, with 8 more for the divisions and the square root; every later product and sum adds
    half a step of its result, counted as 8 of the largest term."""
    x = np.asarray(x, dtype=np.float64)
    m = x.shape[0]
    per = lambda t: np.repeat(np.asarray(t, dtype=np.float64), m // len(t), axis=0)
    u = 2.0 ** -24
    d, mean_err = x, 0.0
    if kind == "layer":
        d = x - x.mean(1, keepdims=True)
        mean_err = 64 * u * np.abs(x).mean(1, keepdims=True) + u * np.abs(x)
    inv = 1.0 if kind == "none" else 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    y = d * inv
    # a shift of the mean by t changes mean(d^2) by t^2 only, and 1 / sqrt(.) by (t inv)^2 / 2
    err = (mean_err * inv) * (1 + np.abs(y)) + 72 * u * np.abs(y) if kind != "none" else 0 * y
    a, b = np.ones((1, x.shape[1])), np.zeros((1, x.shape[1]))
    if weight is not None:
        a = a * np.asarray(weight, dtype=np.float64)
    if bias is not None:
        b = b + np.asarray(bias, dtype=np.float64)
    size = np.abs(b)
    if scale is not None:
        a, b, size = a * (1 + per(scale)), b * (1 + per(scale)), size * (1 + np.abs(per(scale)))
        err = err + 0 * a
    if shift is not None:
        b, size = b + per(shift), size + np.abs(per(shift))
    grown = np.abs(a) if scale is None else np.abs(np.asarray(weight, dtype=np.float64) if weight is not None else 1.0) * (1 + np.abs(per(scale)))
    return y * a + b, err * np.abs(a) + 8 * u * (np.abs(y) * grown + size)
