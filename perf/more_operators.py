"""Attention over a paged cache in 8 bits and what stands in front of it, as cases to be timed: norms of queries and keys per
head with the rotation by position, appending keys and values to the cache, attention over it, and a step of generation made of
the last two.

The cache: pages of P tokens. The keys of a page and head are P x D elements of e4m3 and one power of two that scales them, and so
are the values; a sequence's tokens lie in the pages that its row of a table lists. The scale of a block is the smallest 2^e,
-40 <= e <= 40, of which 448 reach its largest value; it only grows while tokens are appended to a page, and the page's older
elements are then rounded anew. A token whose key or value is not finite is kept as a NaN key and a zero value and counts for no
scale.

Sizes are generic: 128 or fewer columns a head, a few queries' heads to a head of keys. The framework computes forward passes
only, so there is one direction: prompts, and single tokens.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}

# Bounds of a drawn case: below the largest listed ones.
_MAX_BYTES = 4e8
_MAX_SCORES = 1.2e9


# ------------------------------------------------------------------------------------------------------------ the cases
def _rotate(name, dtype, tokens, heads, kv_heads, d, rotated, interleaved, norm, fused):
    return {"name": name, "kind": "rotate", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "d": d,
            "rotated": rotated, "interleaved": interleaved, "norm": norm, "fused": fused}


def _cached(name, kind, dtype, batch, old, new, heads, kv_heads, d, page, window=0, norm=False):
    """old, new: (least, most) of the tokens that sequences have in the cache before the call and get by it; new None: one each."""
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "old_low": old[0], "old_high": old[1], "ragged": new is not None,
            "new_low": new[0] if new else 1, "new_high": new[1] if new else 1, "heads": heads, "kv_heads": kv_heads, "d": d, "page": page,
            "window": window, "norm": norm}


def listed():
    return [
        # one token's queries and keys between a fused projection and attention: the smallest call, where latency counts
        _rotate("rotate_token_f16", "f16", 1, 32, 8, 128, 128, False, True, True),
        # fp32 rows of a user-written network, few odd heads, half of the columns rotated, neighbours paired
        _rotate("rotate_odd_f32", "f32", 777, 5, 1, 80, 40, True, False, True),
        # queries and keys of long prompts
        _rotate("rotate_large_bf16", "bf16", 16384, 32, 8, 128, 128, False, True, True),
        # a step of generation for 64 sequences: one token each goes behind what the cache holds
        _cached("append_tokens_bf16", "append", "bf16", 64, (100, 2000), None, 32, 8, 128, 64, norm=True),
        # pieces of prompts of odd lengths, behind odd lengths, in small pages of narrow heads
        _cached("append_ragged_f16", "append", "f16", 7, (0, 333), (1, 700), 10, 5, 80, 16),
        # eight long prompts into an empty cache
        _cached("append_prompts_bf16", "append", "bf16", 8, (0, 0), (1500, 2500), 32, 8, 128, 64, norm=True),
        # the next token of one short conversation
        _cached("attend_token_bf16", "attend", "bf16", 1, (700, 700), None, 32, 8, 128, 64),
        # the next tokens of 64 conversations of very different lengths
        _cached("attend_tokens_bf16", "attend", "bf16", 64, (0, 8191), None, 32, 8, 128, 64),
        # two conversations that are long: the work has to be split along the cache
        _cached("attend_long_f16", "attend", "f16", 2, (100000, 131071), None, 32, 8, 128, 64),
        # a long prompt, each token sees those in front of it: the largest case
        _cached("attend_prompt_bf16", "attend", "bf16", 1, (0, 0), (8192, 8192), 32, 8, 128, 64),
        # pieces of prompts behind what the cache holds, odd lengths, narrow heads, small pages, a sliding window
        _cached("attend_ragged_f16", "attend", "f16", 5, (0, 1500), (1, 900), 10, 2, 80, 16, window=500),
        # a step of generation: projections normalised and rotated, keys and values appended, attention
        _cached("step_tokens_bf16", "step", "bf16", 32, (500, 4000), None, 32, 8, 128, 64, norm=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["rotate", "append", "attend", "attend", "attend", "step"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    if kind == "rotate":
        d = rng.choice([32, 64, 72, 80, 96, 128, 128, 192, 256])
        return _rotate("", rng.choice(["bf16", "bf16", "f16", "f32"]), _log(rng, 1, 16384), heads, kv_heads, d,
                       rng.choice([d, d, d // 2]), rng.random() < 0.3, rng.random() < 0.6, rng.random() < 0.7)
    d, page = rng.choice([64, 80, 96, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    window = rng.choice([0, 0, 0, 100, 1000]) if kind != "append" else 0
    if kind == "step" or rng.random() < 0.5:
        most = _log(rng, 1, 16384)
        return _cached("", kind, dtype, _log(rng, 1, 128), (rng.choice([0, most // 2, most]), most), None, heads, kv_heads, d, page, window,
                       rng.random() < 0.5 and kind != "attend")
    old, new = rng.choice([0, 0, _log(rng, 1, 4000)]), _log(rng, 2, 2500)
    return _cached("", kind, dtype, _log(rng, 1, 8), (old // 2, old), (rng.choice([1, new // 2 + 1, new]), new), heads, kv_heads, d, page, window,
                   rng.random() < 0.5 and kind != "attend")


def draw(rng):
    while True:
        case = _draw_once(rng)
        scores = 0
        if case["kind"] != "rotate":
            scores = case["batch"] * case["heads"] * case["new_high"] * (case["old_high"] + case["new_high"])
        if work(case)["bytes"] <= _MAX_BYTES and scores <= _MAX_SCORES:
            case.pop("name", None)
            return case


def _lengths(case):
    """(tokens in the cache before, new ones) of each sequence; the same in every run of a case."""
    rng = random.Random(case["batch"] * 7919 + case["old_high"] * 31 + case["new_high"])
    return [(rng.randint(case["old_low"], case["old_high"]), rng.randint(case["new_low"], case["new_high"])) for _ in range(case["batch"])]


# ----------------------------------------------------------------------------------------------------------- the inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _heads(gen, tokens, heads, d, size):
    """Rows of heads as projections make them: channels differ in size, a few of them by far."""
    return _randn(gen, tokens, heads, d) * (size * torch.exp(0.5 * _randn(gen, heads, d)))


def _rows(gen, tokens, heads, kv_heads, d, dtype, fused):
    """Queries, keys and values, as slices of the rows of one projection if `fused`."""
    parts = [_heads(gen, tokens, heads, d, 1.0), _heads(gen, tokens, kv_heads, d, 1.0), _heads(gen, tokens, kv_heads, d, 0.7)]
    if not fused:
        return [p.to(_DT[dtype]) for p in parts]
    whole = torch.cat([p.to(_DT[dtype]) for p in parts], dim=1)
    return list(torch.split(whole, [heads, kv_heads, kv_heads], dim=1))


def _stored(x):
    """A cache's blocks as the format holds them: (elements, scale bytes) of x (pages, heads, P, D)."""
    peak = x.abs().amax((2, 3))
    e = (torch.frexp(peak / 448).exponent).clamp(-40, 40)        # an exact power of two may get one more than it needs
    return torch.ldexp(x, -e[..., None, None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    d, heads, kv_heads, dtype = case["d"], case["heads"], case["kv_heads"], case["dtype"]
    if case["kind"] == "rotate":
        tokens = case["tokens"]
        s["q"], s["k"], _ = _rows(gen, tokens, heads, kv_heads, d, dtype, case["fused"])
        s["positions"] = torch.randint(0, 131072, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
        rotated = case["rotated"]
    else:
        lengths, page, rotated = _lengths(case), case["page"], d
        tokens = sum(new for _, new in lengths)
        s["lengths"] = torch.tensor([old + new for old, new in lengths], dtype=torch.int32, device="cuda")
        if case["ragged"]:
            s["starts"] = torch.tensor([sum(new for _, new in lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")
        else:
            s["starts"] = None
        s["longest"] = max(new for _, new in lengths)
        width = max(-(-(old + new) // page) for old, new in lengths)
        pages = case["batch"] * width + 3
        s["pages"] = torch.randperm(pages, generator=gen, device="cuda")[:case["batch"] * width].view(case["batch"], width).to(torch.int32)
        spread = torch.exp(0.5 * _randn(gen, kv_heads, 1, d))
        s["k_cache"], s["k_scales"] = _stored(_randn(gen, pages, kv_heads, page, d) * spread)
        s["v_cache"], s["v_scales"] = _stored(0.7 * _randn(gen, pages, kv_heads, page, d))
        s["q"], s["k"], s["v"] = _rows(gen, tokens, heads, kv_heads, d, dtype, case["kind"] != "attend")
    s["frequencies"] = torch.exp(-math.log(10000.0) * torch.arange(0, rotated, 2, device="cuda", dtype=torch.float64) / rotated)
    s["q_weight"] = 1 + 0.1 * _randn(gen, d) if case["norm"] else None
    s["k_weight"] = 1 + 0.1 * _randn(gen, d) if case["norm"] else None
    return s


# ------------------------------------------------------------------------------------------------------- the plain forms
def _plain_rotate(x, weight, positions, frequencies, interleaved):
    """Heads x (T, H, D), normalised if there is a weight, and rotated, in float32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    angle = positions.double()[:, None, None] * frequencies
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    r = 2 * frequencies.numel()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _places(s):
    """Sequence and position of each row."""
    rows = torch.arange(s["q"].shape[0], device=s["q"].device)
    if s["starts"] is None:
        return rows, s["lengths"].long() - 1
    seq = torch.searchsorted(s["starts"].long(), rows, right=True) - 1
    return seq, s["lengths"].long()[seq] - s["starts"].long()[seq + 1] + rows


def _plain_append(values, bad, cache, scales, offset, touched, at, zero_bad):
    """New tokens' values (T, H, D) into the blocks (pages, H, P, D); `touched`: the pages that get some, `at`: the place in it of each
    token's page."""
    size = cache.shape[2]
    peak = torch.where(bad[..., None], 0.0, values).abs().amax(-1)
    peak = torch.zeros(touched.numel(), values.shape[1], device=values.device).index_reduce_(0, at, peak, "amax")
    first = torch.full((touched.numel(),), size, device=values.device).index_reduce_(0, at, offset, "amin")
    # the smallest exponent of which 448 reach the peak: 448 = 0.875 * 2^9
    mantissa, exponent = torch.frexp(peak)
    e = torch.where(peak > 0, exponent - 9 + (mantissa > 0.875), -40).clamp(-40, 40)
    old = scales[touched].int() - 127
    e = torch.where((first > 0)[:, None], torch.maximum(e, old), e)
    block = torch.ldexp(cache[touched].float(), (old - e)[..., None, None])
    kept = torch.arange(size, device=values.device) < first[:, None]
    block = torch.where(kept[:, None, :, None], block, cache[touched].float())
    new = torch.ldexp(values, -e[at][..., None]).clamp(-448, 448)
    block[at, :, offset] = torch.where(bad[..., None], 0.0 if zero_bad else math.nan, new)
    cache[touched] = block.to(torch.float8_e4m3fn)
    scales[touched] = (e + 127).to(torch.uint8)


def _plain_cache(s):
    seq, position = _places(s)
    size = s["case"]["page"]
    page_of, offset = s["pages"].long()[seq, position // size], position % size
    k, v = _plain_rotate(s["k"], s["k_weight"], position, s["frequencies"], False), s["v"].float()
    bad = ~(torch.isfinite(k) & torch.isfinite(v)).all(-1)
    touched, at = torch.unique(page_of, return_inverse=True)
    _plain_append(k, bad, s["k_cache"], s["k_scales"], offset, touched, at, False)
    _plain_append(v, bad, s["v_cache"], s["v_scales"], offset, touched, at, True)
    return _plain_rotate(s["q"], s["q_weight"], position, s["frequencies"], False).to(s["q"].dtype)


def _plain_attend(s, q):
    case = s["case"]
    b, kv, d, group = case["batch"], case["kv_heads"], case["d"], case["heads"] // case["kv_heads"]
    table = s["pages"].long()
    tokens = table.shape[1] * case["page"]
    lengths = s["lengths"].long()
    held = torch.arange(tokens, device=q.device) < lengths[:, None]

    def gathered(cache, scales):
        x = torch.ldexp(cache[table].float(), (scales[table].int() - 127)[..., None, None])       # b, pages, kv, P, d
        return torch.where(held[:, None, :, None], x.transpose(1, 2).reshape(b, kv, tokens, d), 0.0)

    seq, position = _places(s)
    rows = s["longest"]
    row = position - lengths[seq] + (1 if s["starts"] is None else (s["starts"][1:] - s["starts"][:-1]).long()[seq])
    padded = torch.zeros(b, rows, kv, group, d, device=q.device)
    padded[seq, row] = q.float().view(-1, kv, group, d)
    at = torch.full((b, rows), -1, device=q.device, dtype=torch.long)
    at[seq, row] = position
    scores = padded.permute(0, 2, 3, 1, 4).reshape(b, kv, group * rows, d) @ gathered(s["k_cache"], s["k_scales"]).transpose(2, 3)
    scores = scores.view(b, kv, group, rows, tokens) * d ** -0.5
    j = torch.arange(tokens, device=q.device)
    seen = held[:, None, :] & (j <= at[..., None])
    if case["window"]:
        seen = seen & (j > at[..., None] - case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.exp_().view(b, kv, group * rows, tokens)
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered(s["v_cache"], s["v_scales"]) / torch.where(total > 0, total, 1.0)).view(b, kv, group, rows, d)
    return out.permute(0, 3, 1, 2, 4)[seq, row].reshape(q.shape).to(q.dtype)


def _plain(s):
    case = s["case"]
    if case["kind"] == "rotate":
        return tuple(_plain_rotate(s[x], s[x + "_weight"], s["positions"], s["frequencies"], case["interleaved"]).to(s[x].dtype) for x in "qk")
    if case["kind"] == "attend":
        return _plain_attend(s, s["q"])
    q = _plain_cache(s)
    return q if case["kind"] == "append" else _plain_attend(s, q)


def _with_cache(s, first):
    """The outputs of a call that writes to the cache: elements and scales as the numbers that they are."""
    return first, s["k_cache"], s["v_cache"], s["k_scales"].view(torch.float8_e8m0fnu), s["v_scales"].view(torch.float8_e8m0fnu)


# --------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from tracea_b200 import ops
    case = s["case"]
    if case["kind"] == "rotate":
        return ops.head_norm_rotate(s["q"], s["k"], s["positions"], s["frequencies"], case["interleaved"], s["q_weight"], s["k_weight"],
                                    kind="rms" if case["norm"] else "none")
    cache = ops.KvCache(s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"])
    q = s["q"]
    if case["kind"] != "attend":
        q = ops.kv_append(cache, s["k"], s["v"], s["pages"], s["lengths"], s["starts"], s["frequencies"], k_weight=s["k_weight"],
                          q=q, q_weight=s["q_weight"], kind="rms" if case["norm"] else "none")
        if case["kind"] == "append":
            return q
    return ops.kv_attention(q, cache, s["pages"], s["lengths"], s["starts"], window=case["window"])


def run(state):
    out = _own(state) if own else _plain(state)
    return out if state["case"]["kind"] in ("rotate", "attend") else _with_cache(state, out)


# ---------------------------------------------------------------------------------------------------------- work and truth
def _visible(case):
    """(tokens of the cache that some row sees, row-token pairs) over all sequences."""
    tokens, pairs, window = 0, 0, case["window"]
    for old, new in _lengths(case):
        tokens += min(old + new, window + new - 1) if window else old + new
        full = lambda n: n * (n + 1) // 2        # noqa: E731  1 + .. + n
        if not window:
            pairs += full(old + new) - full(old)
        else:
            grow = max(0, min(new, window - old))          # rows that see less than a window
            pairs += full(old + grow) - full(old) + (new - grow) * window if grow else new * window
    return tokens, pairs


def work(case):
    es, d, heads, kv = _SIZE[case["dtype"]], case["d"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotate":
        return {"bytes": 2 * case["tokens"] * (heads + kv) * d * es, "flops": 0}
    new = sum(n for _, n in _lengths(case))
    queries = 2 * new * heads * d * es
    appended = 2 * new * kv * d * (es + 1)
    if case["kind"] == "append":
        return {"bytes": queries + appended, "flops": 0}
    tokens, pairs = _visible(case)
    read = 2 * tokens * kv * d
    if case["kind"] == "step":
        return {"bytes": queries + appended + read, "flops": 4.0 * pairs * heads * d}
    return {"bytes": queries + read, "flops": 4.0 * pairs * heads * d}


def _exact_rotate(x, weight, positions, frequencies, interleaved):
    """As products of complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    turn = torch.polar(torch.ones_like(frequencies), positions.double()[:, None] * frequencies)[:, None]
    n = frequencies.numel()
    pairs = x[..., :2 * n].unflatten(-1, (n, 2)) if interleaved else x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2)
    return torch.cat((turned, x[..., 2 * n:]), dim=-1)


def _exact_e4m3(v):
    """The nearest element, a tie to the even one, as a float64: steps of 2^(floor(log2 |v|) - 3), no finer than 2^-9."""
    e = (torch.frexp(v).exponent - 1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_append(values, cache, scales, pages, lengths, size):
    """Sequence by sequence, page by page; values[i]: the new tokens of sequence i, (n, H, D)."""
    out, bytes_out = cache.double(), scales.double()
    for i, (old, new) in enumerate(lengths):
        for slot in range(old // size, (old + new - 1) // size + 1):
            page, first, last = int(pages[i, slot]), max(old - slot * size, 0), min(old + new - slot * size, size)
            part = values[i][slot * size + first - old:slot * size + last - old].transpose(0, 1)       # H, n, D
            need = part.abs().amax((1, 2)) / 448
            e = torch.ceil(torch.log2(need.clamp(min=1e-300))).clamp(-40, 40)
            e = torch.where(need > torch.exp2(e), e + 1, e)
            before = bytes_out[page] - 127
            if first > 0:
                e = torch.maximum(e, before)
                out[page, :, :first] = _exact_e4m3(out[page, :, :first] * torch.exp2(before - e)[:, None, None])
            out[page, :, first:last] = _exact_e4m3(part * torch.exp2(-e)[:, None, None])
            bytes_out[page] = e + 127
    return out, torch.exp2(bytes_out - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return tuple(_exact_rotate(s[x], s[x + "_weight"], s["positions"], s["frequencies"], case["interleaved"]) for x in "qk")
    lengths, size = _lengths(case), case["page"]
    rows, at = [], 0
    for _, new in lengths:
        rows.append(slice(at, at + new))
        at += new
    q, k, v = s["q"].double(), s["k_cache"].double(), s["v_cache"].double()
    k_scale, v_scale = (torch.exp2(s[x].double() - 127) for x in ("k_scales", "v_scales"))
    if case["kind"] != "attend":
        if sum(1 + new // size for _, new in lengths) > 4000:
            return None
        place = torch.cat([torch.arange(old, old + new) for old, new in lengths]).to(q.device)
        q = _exact_rotate(q, s["q_weight"], place, s["frequencies"], False)
        new_k = _exact_rotate(s["k"], s["k_weight"], place, s["frequencies"], False)
        pages = s["pages"].cpu()
        k, k_scale = _exact_append([new_k[r] for r in rows], s["k_cache"], s["k_scales"], pages, lengths, size)
        v, v_scale = _exact_append([s["v"][r].double() for r in rows], s["v_cache"], s["v_scales"], pages, lengths, size)
        cache = (k, v, k_scale, v_scale)
        if case["kind"] == "append":
            return (q, *cache)
        q = q.to(_DT[case["dtype"]]).double()            # the queries are stored between the two calls
    out, group = torch.empty_like(q), case["heads"] // case["kv_heads"]
    for i, (old, new) in enumerate(lengths):
        n = old + new
        used = s["pages"][i, :-(-n // size)].long()
        place = torch.arange(old, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None, :]
        hidden = (j > place) | (j <= place - case["window"]) if case["window"] else j > place
        for h in range(case["heads"]):
            kk, vv = ((x[used, h // group] * z[used, h // group][:, None, None]).reshape(-1, case["d"])[:n] for x, z in ((k, k_scale), (v, v_scale)))
            a = q[rows[i], h] @ kk.t() / math.sqrt(case["d"])
            a.masked_fill_(hidden, -math.inf)
            out[rows[i], h] = torch.softmax(a, dim=-1) @ vv
    return out if case["kind"] == "attend" else (out, *cache)
