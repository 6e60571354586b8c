"""Rows of heads, the paged cache in 8 bits and attention over it, in 64 bits and from their definitions: what test_heads_gpu.py and
test_kv_*.py compare with. Plain torch on whatever device the arguments are; nothing here calls the library."""
import torch

U = 2.0 ** -24                                   # half a step of fp32, relative


def rotate(x, positions=None, frequencies=None, interleaved=False, weight=None, kind="none", eps=1e-6):
    """(result, bound on the error of an fp32 computation of it, before the output's rounding) for x (T, H, D).

    The bound: a lane sums 16 squares or fewer and five steps across lanes follow, at most 24 half steps of the sum and so 12 of the
    factor 1 / sqrt(.), with 8 more for the division, the square root and the two products: 20 of the value. Cosine and sine are off
    by 2 half steps of 1 and by the angle's, at most pi/4 half steps; a rotation's two products and sum add 3 of |a| + |b|: in all
    fewer than 32 half steps of |a| + |b|."""
    y = x.double()
    if kind == "rms":
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    if weight is not None and kind != "none":
        y = y * weight.double()
    size = y.abs()
    if frequencies is not None:
        n = frequencies.numel()
        angle = positions.double()[:, None, None] * frequencies.double()
        c, s = torch.cos(angle), torch.sin(angle)
        first = torch.arange(0, 2 * n, 2) if interleaved else torch.arange(n)
        second = first + 1 if interleaved else first + n
        a, b = y[..., first], y[..., second]
        y, both = y.clone(), a.abs() + b.abs()
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size = size.clone()
        size[..., first] = size[..., second] = both
    return y, 32 * U * size


def e4m3(v):
    """The nearest element, ties to even, saturated, as a float64; NaN stays NaN."""
    v = v.double()
    e = (torch.frexp(torch.where(torch.isfinite(v), v, 0.0)).exponent - 1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def half_step(v):
    """Half the distance of elements around v."""
    e = (torch.frexp(v.double()).exponent - 1).clamp(min=-6, max=8)
    return torch.ldexp(torch.ones_like(v, dtype=torch.float64), e - 4)


def exponent(peak):
    """The smallest e in -40..40 of which 448 reach `peak`."""
    e = torch.full_like(peak, -40, dtype=torch.float64)
    for i in range(-40, 40):
        e = torch.where(peak > 448 * 2.0 ** i, i + 1.0, e)
    return e


def places(pages, lengths, starts, rows, size, total):
    """For each row (sequence, position, page or -1, row in the page)."""
    b = len(lengths)
    starts = list(range(b + 1)) if starts is None else [int(s) for s in starts]
    out = [(-1, 0, -1, 0)] * rows
    for s in range(b):
        n = starts[s + 1] - starts[s]
        for i in range(n):
            p = int(lengths[s]) - n + i
            slot = p // size
            page = int(pages[s][slot]) if 0 <= slot < len(pages[s]) else -1
            out[starts[s] + i] = (s, p, page if 0 <= page < total else -1, p % size)
    return out


def append(elements, scales, values, err, bad, where):
    """What appending leaves in a cache (elements (pages, heads, P, D) as float64, scale bytes (pages, heads)): a list of (page, first
    new row, {row of the page: row of values}, least exponents, greatest exponents) of the pages touched, the exponents (heads) with
    the values' error taken into account; values, err (T, heads, D); bad (T, heads)."""
    touched = {}
    for row, (_, _, page, at) in enumerate(where):
        if page >= 0:
            touched.setdefault(page, {})[at] = row
    out = []
    for page, rows in touched.items():
        index = torch.tensor(sorted(rows.values()), device=values.device)
        v = torch.where(bad[index][..., None], 0.0, values[index].abs())
        e = torch.where(bad[index][..., None], 0.0, err[index])
        low, high = exponent((v - e).clamp(min=0).amax((0, 2))), exponent((v + e).amax((0, 2)))
        first = min(rows)
        if first > 0:
            old = scales[page].double() - 127
            low, high = torch.maximum(low, old), torch.maximum(high, old)
        out.append((page, first, rows, low, high))
    return out


def dequantized(elements, scales):
    return elements.double() * torch.exp2(scales.double() - 127)[..., None, None]


def attention(q, elements_k, elements_v, scales_k, scales_v, pages, lengths, starts, scale, causal, window, out_eps):
    """(result, bound on the error of the kernels, their output's rounding included) for q (T, H, D).

    The bound. Scores: q is rounded to 11 bits of its row's largest value at least, which changes nothing in an input of 11 bits or
    fewer but elements 2^-14 of the largest and smaller, those by 2^-25 of it; D products are added in fp32, by at most D additions
    that drop up to a step: 2 D half steps of the sum of the products' sizes. Twice as much in a weight's logarithm, since its
    denominator is off likewise. Weights: 2^-11 from their rounding to halves, and for weights too small for that 2^-25 of the largest
    weight times scale, for each value; 2^-20 for the exponential, which takes its argument, of up to 2^8, in fp32, and the sums."""
    t, heads, d = q.shape
    kv, size = elements_k.shape[1], elements_k.shape[2]
    y, bound = torch.zeros(t, heads, d, dtype=torch.float64, device=q.device), torch.zeros(t, heads, d, dtype=torch.float64, device=q.device)
    starts = list(range(len(lengths) + 1)) if starts is None else [int(s) for s in starts]
    total = elements_k.shape[0]
    for s, length in enumerate(int(x) for x in lengths):
        rows = slice(starts[s], starts[s + 1])
        n = starts[s + 1] - starts[s]
        if n == 0:
            continue
        there = [p if 0 <= p < total else -1 for p in (int(x) for x in pages[s])][:-(-length // size)]
        used = torch.tensor([max(p, 0) for p in there], dtype=torch.long, device=q.device)
        tokens = len(there) * size
        at = torch.arange(tokens, device=q.device)
        held = (at < length) & torch.tensor([p >= 0 for p in there], device=q.device, dtype=torch.bool).repeat_interleave(size)
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        seen = held[None, :].expand(n, tokens)
        if causal:
            seen = seen & (at[None, :] <= pos)
        if window:
            seen = seen & (at[None, :] > pos - window)
        for h in range(heads):
            block = (used, torch.full_like(used, h // (heads // kv)))
            kk = (elements_k[block].double() * torch.exp2(scales_k[block].double() - 127)[:, None, None]).reshape(tokens, d)
            ve = elements_v[block].double().reshape(tokens, d)
            ev = torch.exp2(scales_v[block].double() - 127).repeat_interleave(size)
            ve = torch.where(held[:, None], ve, 0.0)
            x = q[rows, h].double()
            a = torch.where(seen, scale * (x @ kk.t()), -torch.inf)
            slip = 2 * d * U * (x.abs() @ kk.abs().t()) + 2.0 ** -25 * x.abs().amax(1, keepdim=True) * kk.abs().sum(1)[None, :]
            slip = torch.where(seen, abs(scale) * slip, 0.0)
            top = a.amax(1, keepdim=True) if tokens else a.new_zeros(n, 1)
            p = torch.where(seen, torch.exp(a - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            weight = p.sum(1, keepdim=True)
            safe = torch.where(weight == 0, 1.0, weight)
            y[rows, h] = (p @ (ve * ev[:, None])) / safe
            relative = 2 * slip.amax(1, keepdim=True) + 2.0 ** -11 + 2.0 ** -20 if tokens else a.new_zeros(n, 1)
            big = (p * ev).amax(1, keepdim=True) if tokens else a.new_zeros(n, 1)
            bound[rows, h] = (relative * (p @ (ve.abs() * ev[:, None])) + 2.0 ** -25 * big * (seen.double() @ ve.abs())) / safe
    return y, bound + out_eps / 2 * (y.abs() + bound)
