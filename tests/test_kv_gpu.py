"""The paged cache in 8 bits on a B200: appending, and attention over it, against 64 bits. Elements are rounded to nearest, so what is
not rotated is compared bit by bit; what is, within half a step and the bound on the fp32 computation (kvref.rotate); attention within
the bound that kvref.attention derives."""
import pytest
import torch

import kvref
from tracea_b200 import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def random_cache(pages, heads, size, d, seed, spread=2.0):
    """A cache whose blocks hold anything but NaN, with scales that differ by far."""
    g = torch.Generator().manual_seed(seed)
    bytes_ = [torch.randint(0, 256, (pages, heads, size, d), generator=g, dtype=torch.uint8) for _ in "kv"]
    for b in bytes_:
        b[(b & 127) == 127] = 0x3c
    scales = [torch.clamp(118 + spread * torch.randn(pages, heads, generator=g), 87, 167).to(torch.uint8).cuda() for _ in "kv"]
    return ops.KvCache(*(b.cuda().view(torch.float8_e4m3fn) for b in bytes_), *scales)


def tables(lengths, size, total, seed, extra=1):
    """Distinct pages in any order; entries past a sequence's are -1."""
    width = max(-(-n // size) for n in lengths) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    out = [[-1] * width for _ in lengths]
    for s, n in enumerate(lengths):
        for i in range(-(-n // size)):
            out[s][i] = order.pop()
    return out


def rows(t, heads, d, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + t)
    return (size * torch.randn(t, heads, d, generator=g) * torch.exp(0.5 * torch.randn(1, heads, d, generator=g))).to(DT[dtype]).cuda()


def copies(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]


def check_append(cache, before, k, v, pages, lengths, starts, rotation=None, weight=None, kind="none", interleaved=False):
    """The whole cache after appending, from the one before."""
    size, total = cache.page_size, cache.k.shape[0]
    where = kvref.places(pages, lengths, starts, k.shape[0], size, total)
    positions = torch.tensor([w[1] for w in where], device="cuda")
    vk, ek = kvref.rotate(k, positions, rotation, interleaved, weight, kind)
    vv, ev = v.double(), torch.zeros_like(v, dtype=torch.float64)
    bad = ~(torch.isfinite(vk) & torch.isfinite(vv)).all(-1)
    exact = rotation is None and kind == "none"
    if exact:
        ek = torch.zeros_like(ek)
    for values, err, old, scales, now, now_scales, fill in ((vk, ek, before[0], before[2], cache.k, cache.k_scales, float("nan")),
                                                            (vv, ev, before[1], before[3], cache.v, cache.v_scales, 0.0)):
        want = old.double()
        slack = torch.zeros_like(want)
        want_scales = scales.clone()
        for page, first, at, low, high in kvref.append(want, scales, values, err, bad, where):
            e = now_scales[page].double() - 127
            assert bool(((low <= e) & (e <= high)).all()), (page, low, e, high)
            want_scales[page] = now_scales[page]
            one = torch.exp2(e)[:, None]
            if first > 0:
                shrink = torch.exp2(scales[page].double() - 127 - e)[:, None, None]
                want[page, :, :first] = torch.where(shrink == 1, want[page, :, :first], kvref.e4m3(want[page, :, :first] * shrink))
            for r, row in at.items():
                x = values[row] / one
                lost = bad[row][:, None]
                if err.any():
                    want[page, :, r] = torch.where(lost, fill, x.clamp(-448, 448))
                    off = err[row] / one
                    slack[page, :, r] = torch.where(lost, 0.0, off + torch.maximum(kvref.half_step(x), kvref.half_step(x.abs() + off)))
                else:
                    want[page, :, r] = torch.where(lost, fill, kvref.e4m3(x))
        assert torch.equal(now_scales, want_scales)
        got = now.double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        off = torch.nan_to_num((got - want).abs(), nan=0.0)
        assert bool((off <= slack).all()), "%d of %d" % (int((off > slack).sum()), off.numel())


# heads of keys, columns, page, (tokens before, new ones) of each sequence; None: one new token each
APPENDS = [(1, 16, 16, [(0, 1)]), (8, 128, 64, [(0, 200), (63, 1), (64, 65), (100, 0), (5, 30)]), (3, 80, 32, [(31, 2), (0, 33), (7, 90)]),
           (2, 64, 128, [(0, 300), (127, 2), (50, 77)]), (2, 128, 128, [(0, 128), (1, 129)]), (5, 96, 16, [(15, 50), (0, 16), (16, 16)]),
           (4, 48, 64, [(70, 11), (0, 1)]), (2, 112, 64, [(10, 1), (0, 64)])]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, d, size, sequences", APPENDS)
def test_append_prompts(heads, d, size, sequences, dtype):
    lengths = [a + b for a, b in sequences]
    starts = [sum(n for _, n in sequences[:i]) for i in range(len(sequences) + 1)]
    total = sum(-(-n // size) for n in lengths) + 2
    pages = tables(lengths, size, total, d)
    k, v = rows(starts[-1], heads, d, dtype, 1), rows(starts[-1], heads, d, dtype, 2, 0.7)
    for rotation, weight, kind in ((None, None, "none"), (ops.rotary_frequencies(d, device="cuda"), None, "none"),
                                   (ops.rotary_frequencies(d // 2 // 2 * 2, device="cuda"), 1 + 0.2 * rows(1, 1, d, "f32", 3)[0, 0], "rms")):
        cache = random_cache(total, heads, size, d, size)
        before = copies(cache)
        q = rows(starts[-1], 2 * heads, d, dtype, 4)
        got = ops.kv_append(cache, k, v, ints(pages), ints(lengths), ints(starts), rotation, k_weight=weight, q=q, q_weight=weight, kind=kind)
        check_append(cache, before, k, v, pages, lengths, starts, rotation, weight, kind)
        where = kvref.places(pages, lengths, starts, starts[-1], size, total)
        y, err = kvref.rotate(q, torch.tensor([w[1] for w in where], device="cuda"), rotation, False, weight, kind)
        f = torch.finfo(got.dtype)
        assert bool(((got.double() - y).abs() <= err + f.eps / 2 * (y.abs() + err) + f.smallest_normal * f.eps).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, d, size", [(8, 128, 64), (1, 64, 16), (3, 80, 32), (2, 128, 128)])
def test_append_single_tokens(heads, d, size, dtype):
    """Token by token across a page's end: what the pages hold is what each step leaves of the one before."""
    lengths = [1, size - 1, size, 3 * size + 7, 40]
    total = 20 + sum(-(-(n + 4) // size) for n in lengths)
    pages = tables([n + 4 for n in lengths], size, total, d)
    cache = random_cache(total, heads, size, d, d)
    freq = ops.rotary_frequencies(d, device="cuda")
    for step in range(3):
        now = [n + step for n in lengths]
        k, v = rows(5, heads, d, dtype, step, 4.0 ** step), rows(5, heads, d, dtype, 10 + step, 3.0 ** step)
        before = copies(cache)
        assert ops.kv_append(cache, k, v, ints(pages), ints(now), None, freq) is None
        check_append(cache, before, k, v, pages, now, None, freq)
        again = copies(cache)
        ops.kv_append(cache, k, v, ints(pages), ints(now), None, freq)            # the same once more changes nothing
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(again, copies(cache)))


@pytest.mark.parametrize("size", [16, 64])
def test_append_extremes(size):
    """Largest and smallest scales, zeros, elements that saturate, values that are not finite, pages that are not there."""
    heads, d = 2, 64
    cache = random_cache(6, heads, size, d, 9)
    before = copies(cache)
    k, v = rows(5, heads, d, "f32", 1), rows(5, heads, d, "f32", 2)
    k[0], v[0] = 1e30, -1e-30                    # beyond 448 * 2^40; below half of the smallest element
    k[1], v[1] = 0.0, 448.0                      # the largest scale that 448 needs is 2^0
    v[1, 0, 3] = 449.0
    k[2, 0, 1], v[2, 1, 0] = float("nan"), float("inf")
    pages, lengths = [[0], [1], [2], [99], [-1]], [3, 2, 5, 4, 1]
    ops.kv_append(cache, k, v, ints(pages), ints(lengths))
    check_append(cache, before, k, v, pages, lengths, None)
    assert cache.k_scales[0].tolist() == [167, 167] and int(cache.v_scales[1, 1]) >= 127
    assert torch.isnan(cache.k[2, :, 4].float()).all() and not cache.v[2, :, 4].float().any()     # one by its key, one by its value


def test_append_fresh_page_forgets_and_rows_behind_stay():
    cache = random_cache(2, 1, 16, 16, 3)
    before = copies(cache)
    cache.k_scales.fill_(160)
    k, v = rows(3, 1, 16, "f16", 1), rows(3, 1, 16, "f16", 2)
    ops.kv_append(cache, k, v, ints([[1]]), ints([3]), ints([0, 3]))
    assert int(cache.k_scales[1]) < 140 and int(cache.k_scales[0]) == 160
    assert torch.equal(cache.k[1, 0, 3:].view(torch.uint8), before[0][1, 0, 3:].view(torch.uint8))
    assert torch.equal(cache.v[0].view(torch.uint8), before[1][0].view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------ attention
def check_attention(q, cache, pages, lengths, starts, causal=True, window=0, scale=None, got=None):
    if got is None:
        got = ops.kv_attention(q, cache, ints(pages), ints(lengths), None if starts is None else ints(starts), scale, causal, window)
    eps = torch.finfo(q.dtype).eps
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    y, bound = kvref.attention(q, cache.k, cache.v, cache.k_scales, cache.v_scales, pages, lengths, starts, scale, causal, window, eps)
    off = (got.double() - y).abs()
    tiny = torch.finfo(q.dtype).smallest_normal * eps
    assert bool((off <= bound + tiny).all()), "%d of %d off, worst %g of the bound" % (
        int((off > bound + tiny).sum()), off.numel(), float((off / (bound + tiny)).max()))


# heads, heads of keys, columns, page, lengths
TOKENS = [(1, 1, 16, 16, [1]), (32, 8, 128, 64, [1, 700, 64, 65, 4097]), (10, 2, 80, 16, [15, 16, 17, 333]), (6, 6, 64, 32, [100, 0, 31]),
          (40, 2, 128, 128, [129, 1000]), (7, 1, 48, 16, [50, 2000]), (16, 1, 112, 64, [9, 640]), (33, 1, 96, 32, [77, 1500]),
          (8, 8, 128, 64, [20000])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h, kv, d, size, lengths", TOKENS)
def test_attention_of_single_tokens(h, kv, d, size, lengths, dtype):
    total = sum(-(-n // size) for n in lengths) + 2
    pages = tables(lengths, size, total, h)
    cache = random_cache(total, kv, size, d, d + h)
    q = rows(len(lengths), h, d, dtype, 1)
    for window in (0, 1, 40):
        check_attention(q, cache, pages, lengths, None, window=window)
    check_attention(q, cache, pages, lengths, None, causal=False, scale=0.3)


# heads, heads of keys, columns, page, (tokens before, new ones)
PROMPTS = [(4, 1, 128, 64, [(0, 3), (10, 5), (1000, 2)]), (8, 2, 128, 64, [(0, 300)]), (10, 2, 80, 16, [(0, 1), (5, 130), (200, 77), (40, 0)]),
           (3, 3, 64, 32, [(0, 129), (127, 256)]), (32, 8, 128, 128, [(0, 513), (300, 20)]), (5, 1, 48, 16, [(17, 90), (0, 400)]),
           (2, 2, 96, 64, [(640, 640)]), (48, 1, 64, 64, [(30, 9)])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h, kv, d, size, sequences", PROMPTS)
def test_attention_of_prompts(h, kv, d, size, sequences, dtype):
    lengths = [a + b for a, b in sequences]
    starts = [sum(n for _, n in sequences[:i]) for i in range(len(sequences) + 1)]
    total = sum(-(-n // size) for n in lengths) + 2
    pages = tables(lengths, size, total, h)
    cache = random_cache(total, kv, size, d, d + h)
    q = rows(starts[-1], h, d, dtype, 1)
    for causal, window in ((True, 0), (False, 0), (True, 70), (False, 100), (True, 1)):
        check_attention(q, cache, pages, lengths, starts, causal, window)


@pytest.mark.parametrize("n", [1, 200])
def test_attention_of_rows_that_see_nothing(n):
    """Lengths of zero or short of the rows, tables too short, pages that are not there."""
    cache = random_cache(8, 2, 16, 64, 5)
    q = rows(4 * n, 4, 64, "bf16", 2)
    starts = [i * n for i in range(5)]
    pages, lengths = [[0, 1], [-1, 2], [3, 77], [-5, -1]], [0, 30 + n, 32 + n // 2, 20 + n]
    for causal in (True, False):
        got = ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts), causal=causal)
        check_attention(q, cache, pages, lengths, starts, causal, got=got)
        assert not got[:n].any() and not got[3 * n:].any() and got[n:3 * n].any()


@pytest.mark.parametrize("n", [1, 150])
def test_attention_of_unseen_nan_and_extreme_scales(n):
    """NaN keys are seen only by rows behind them; what lies behind the last token may be anything; scales at both ends of their range
    side by side, and blocks of zeros."""
    size, d = 16, 64
    cache = random_cache(20, 1, size, d, 6)
    length = 10 * size + 5
    pages = [list(range(11))]
    cache.k.view(torch.uint8)[10, :, 5:] = 0x7f
    cache.v.view(torch.uint8)[10, :, 5:] = 0xff
    for page, byte in ((0, 167), (1, 87), (2, 167), (3, 87)):
        cache.v_scales[page] = byte
    cache.v[4:6] = 0
    cache.v_scales[4] = 87
    cache.k[1] = 0
    cache.k_scales[1] = 87
    q = rows(n, 4, d, "bf16", 3, 0.2)
    check_attention(q, cache, pages, [length], [0, n])
    if n > 1:
        cache.k.view(torch.uint8)[9, 0, 9] = 0x7f
        got = ops.kv_attention(q, cache, ints(pages), ints([length]), ints([0, n]))
        bad = torch.isnan(got).all(-1).all(-1)
        first = 9 * size + 9 - (length - n)
        assert bad.tolist() == [i >= first for i in range(n)] and not torch.isnan(got[:first]).any()


def test_attention_of_large_and_small_queries():
    """Rows of q whose elements are at the ends of their types, and with elements 2^-20 of the largest."""
    cache = random_cache(8, 1, 64, 128, 7)
    for dtype, sizes in (("f16", (6e4, 1e-7, 1.0)), ("bf16", (1e30, 1e-30, 1.0))):
        for size in sizes:
            q = rows(2, 2, 128, dtype, 4, 0.1)
            q = (q.float() / q.float().abs().max() * size).to(DT[dtype])
            q[:, :, ::3] *= 2.0 ** -20 if dtype == "bf16" else 2.0 ** -9
            check_attention(q, cache, [list(range(8))] * 2, [500, 511], None, scale=0.01 / size)


@pytest.mark.parametrize("n", [1, 130])
def test_strided_rows_of_a_projection(n):
    whole = rows(3 * n, 4 + 2, 72, "f16", 5)
    q = whole[:, :4, 3:67]
    cache = random_cache(60, 2, 16, 64, 8)
    lengths = [n, n + 15, 2 * n]
    pages = tables(lengths, 16, 60, 1)
    check_attention(q, cache, pages, lengths, [0, n, 2 * n, 3 * n])


def test_a_step_of_generation_in_a_graph_and_on_two_streams():
    """Prompts, then steps: appended, attended to; captured once and replayed, with lengths that grow on the device; beside it the same on
    another stream and another cache. All bits are those of the calls made one by one."""
    h, kv, d, size, b = 8, 2, 128, 64, 3
    freq = ops.rotary_frequencies(d, device="cuda")
    pages = ints(tables([200] * b, size, 20, 2))
    lengths0, starts = [60, 3, 100], [0, 60, 63, 163]
    prompt = rows(163, h + 2 * kv, d, "bf16", 6)
    steps = [rows(b, h + 2 * kv, d, "bf16", 7 + i) for i in range(5)]

    def step(cache, x, lengths, starts=None):
        q, k, v = torch.split(x, [h, kv, kv], dim=1)
        q = ops.kv_append(cache, k, v, pages, lengths, starts, freq, q=q)
        return ops.kv_attention(q, cache, pages, lengths, starts)

    def eager():
        cache = ops.KvCache.empty(20, kv, d, size)
        out = [step(cache, prompt, ints(lengths0), ints(starts))]
        return cache, out + [step(cache, x, ints([n + 1 + i for n in lengths0])) for i, x in enumerate(steps)]

    want_cache, want = eager()
    cache = ops.KvCache.empty(20, kv, d, size)
    lengths = ints(lengths0)
    got = [step(cache, prompt, lengths, ints(starts))]
    x = steps[0].clone()
    scratch = ops.KvCache.empty(20, kv, d, size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(scratch, x, lengths)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths += 1
        y = step(cache, x, lengths)
    with torch.cuda.stream(side):
        other_cache, other = eager()
    for s in steps:
        x.copy_(s)
        graph.replay()
        got.append(y.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b_) for a, b_ in zip(want, got)) and all(torch.equal(a, b_) for a, b_ in zip(want, other))
    assert all(torch.equal(a.view(torch.uint8), b_.view(torch.uint8)) for a, b_ in zip(copies(want_cache), copies(cache)))


def test_results_do_not_change_from_call_to_call():
    cache = random_cache(300, 2, 64, 128, 11)
    q = rows(3, 16, 128, "bf16", 9)
    lengths = [4000, 5000, 1234]
    pages = ints(tables(lengths, 64, 300, 3))
    first = ops.kv_attention(q, cache, pages, ints(lengths))
    assert all(torch.equal(first, ops.kv_attention(q, cache, pages, ints(lengths))) for _ in range(20))


def test_offsets_beyond_32_bits():
    """A cache of over 4 GB a tensor, its last pages used."""
    heads, d, size = 8, 128, 128
    pages = 2 ** 32 // (heads * d * size) + 300
    cache = ops.KvCache(*(torch.zeros(pages, heads, size, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv"),
                        *(torch.full((pages, heads), 120, dtype=torch.uint8, device="cuda") for _ in "kv"))
    table = [[pages - 1, 0, pages - 2]]
    k, v = rows(300, heads, d, "bf16", 1), rows(300, heads, d, "bf16", 2)
    ops.kv_append(cache, k, v, ints(table), ints([300]), ints([0, 300]))
    assert torch.equal(cache.v[pages - 1].double() * torch.exp2(cache.v_scales[pages - 1].double() - 127)[:, None, None],
                       torch.stack([kvref.e4m3(v[:128, h].double() / 2.0 ** (int(cache.v_scales[pages - 1, h]) - 127)) *
                                    2.0 ** (int(cache.v_scales[pages - 1, h]) - 127) for h in range(heads)]))
    assert not cache.k[1:pages - 2].view(torch.uint8).any()
    q = rows(300, heads, d, "bf16", 3)
    small = [0, pages - 2, pages - 1]
    sub = ops.KvCache(cache.k[small], cache.v[small], cache.k_scales[small], cache.v_scales[small])
    check_attention(q, sub, [[2, 0, 1]], [300], [0, 300],
                    got=ops.kv_attention(q, cache, ints(table), ints([300]), ints([0, 300])))
    check_attention(q[:1], sub, [[2, 0, 1]], [300], None, got=ops.kv_attention(q[:1], cache, ints(table), ints([300])))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h, kv, d, size, sequences", [(8, 2, 128, 64, [(4000, 130)]), (4, 1, 64, 32, [(0, 2500), (3000, 70)]),
                                                       (6, 2, 80, 128, [(9000, 45), (100, 3), (2000, 90)])])
def test_attention_of_pieces_of_prompts_behind_long_ones(h, kv, d, size, sequences, dtype):
    """Few blocks of rows and many tokens: the tokens are split over CTAs, and some of a block's parts are seen by none of its rows."""
    lengths = [a + b for a, b in sequences]
    starts = [sum(n for _, n in sequences[:i]) for i in range(len(sequences) + 1)]
    total = sum(-(-n // size) for n in lengths) + 2
    pages = tables(lengths, size, total, h, extra=20)
    pages[0][3] = -1
    cache = random_cache(total, kv, size, d, d + h)
    q = rows(starts[-1], h, d, dtype, 1)
    for causal, window in ((True, 0), (False, 0), (True, 900), (True, 33)):
        check_attention(q, cache, pages, lengths, starts, causal, window)
