"""Heads, the cache and attention on a B200 where single values, rows or warps go their own way: waits that run out for some warps of a
block and not for others, weights without a norm, scores that vanish beside masked ones, rows that are not finite and see nothing,
values that are not finite beside columns that are copied, small weights beside large ones, scores of
any size."""
import pytest
import torch

import kvref
from test_heads_gpu import DT, assert_near, make, weights
from test_kv_gpu import check_append, check_attention, copies, ints, random_cache, rows, tables
from tracea_b200 import ffi, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stop", [0, 1, 2, 3, 5])
def test_waits_that_run_out_behind_one_silent_warp(stop):
    """One of the four warps that widen the cache's elements leaves: the products wait in vain for its part, the other three for the
    products. All give up as whole warps, the kernel returns, and the next call is right."""
    lib = ffi.load()
    cache = random_cache(40, 2, 64, 128, 5)
    pages, lengths, starts = [list(range(20))], [1200], [0, 1200]
    q = rows(1200, 4, 128, "bf16", 6)
    assert lib.tracea_b200_device_status(0) == 0
    try:
        lib.tracea_b200_test_hooks(400000, 65536 + stop)
        ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts))
        torch.cuda.synchronize()
    finally:
        lib.tracea_b200_test_hooks(0, -1)
    assert lib.tracea_b200_device_status(0) != 0
    assert lib.tracea_b200_device_status(0) == 0
    check_attention(q, cache, pages, lengths, starts)


def weighted(x, weight, positions=None, frequencies=None, interleaved=False):
    """kvref.rotate of the weighted rows: the weight's product, rounded, is a half step more of what its bound of 32 counts 5 of."""
    return kvref.rotate(x.double() * weight.double(), positions, frequencies, interleaved)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t, h, kv, d, rotated", [(1, 32, 8, 128, 128), (9, 3, 2, 64, 32), (7, 4, 1, 72, 40), (5, 2, 1, 250, 0), (33, 6, 3, 80, 0)])
def test_a_weight_counts_without_a_norm(t, h, kv, d, rotated, dtype):
    """Lanes of 16 columns and column by column, all, some and none of them rotated."""
    q, k, _ = make(t, h, kv, d, dtype, 11)
    positions = torch.arange(t, dtype=torch.int32).cuda() * 1001 + 5
    freq = ops.rotary_frequencies(rotated, device="cuda") if rotated else None
    for w in (weights(d, torch.float32, 2), weights(d, DT[dtype], 3)):
        for interleaved in (False, True):
            got = ops.head_norm_rotate(q, k, positions, freq, interleaved, *w, kind="none")
            for x, y, weight in zip((q, k), got, w):
                assert_near(y, *weighted(x, weight, positions, freq, interleaved))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_a_weight_counts_without_a_norm_when_appending(shift, dtype):
    """What kv_append does by default; rows on a 16-byte boundary and off it."""
    heads, d, size = 2, 64, 32
    lengths, starts = [40, 3, 101], [0, 40, 41, 100]
    pages = tables(lengths, size, 12, 1)
    part = lambda n, seed: rows(100, n, d + 8, dtype, seed)[:, :, shift:shift + d]      # noqa: E731
    k, v, q = part(heads, 1), part(heads, 2), part(3 * heads, 3)
    kw, qw = weights(d, torch.float32, 4)
    freq = ops.rotary_frequencies(48, device="cuda")
    where = torch.tensor([w[1] for w in kvref.places(pages, lengths, starts, 100, size, 12)], device="cuda")
    cache = random_cache(12, heads, size, d, 5)
    before = copies(cache)
    got = ops.kv_append(cache, k, v, ints(pages), ints(lengths), ints(starts), freq, k_weight=kw, q=q, q_weight=qw)
    check_append(cache, before, k.double() * kw.double(), v, pages, lengths, starts, freq)
    assert_near(got, *weighted(q, qw, where, freq))
    one = random_cache(12, heads, size, d, 6)
    before = copies(one)
    got = ops.kv_append(one, k[:3], v[:3], ints(pages), ints(lengths), None, None, k_weight=torch.full_like(kw, 0.5), q=q[:3], q_weight=qw)
    check_append(one, before, k[:3].double() * 0.5, v[:3], pages, lengths, None)      # by a power of two: exactly
    assert_near(got, *weighted(q[:3], qw))


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("n, old", [(3, 40), (70, 0), (150, 90), (100, 6000)])
def test_scores_that_vanish_and_masks(n, old, d):
    """A scale of zero, or queries so small that all products underflow, over pages of the smallest scale and of zeros: the mean of what
    a row sees, and no NaN out of what it does not. Few rows, many, and many with their tokens split."""
    length = old + n
    total = -(-length // 16) + 1
    cache = random_cache(total, 2, 16, d, 7)
    cache.k_scales[::2] = 87
    cache.k[::4] = 0
    pages, starts = tables([length], 16, total, 3), [0, n]
    for dtype in ("f16", "bf16"):
        q = rows(n, 8, d, dtype, 8)
        smallest = (q.float() * (1e-37 if dtype == "bf16" else 1e-6)).to(q.dtype)
        for window in (0, 33):
            for x, scale in ((q, 0.0), (q, -0.2), (q, 1e-30), (smallest, 0.1), (smallest, 0.0), (torch.zeros_like(q), 0.1)):
                check_attention(x, cache, pages, [length], starts, window=window, scale=scale)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [1, 90, 300])
def test_rows_of_anything_that_see_no_page_are_zero(n, value):
    """Pages that are not there, under rows that are not finite (what a padded batch may hold): 0, in every form; NaN where there is one."""
    size, d = 16, 64
    cache = random_cache(300, 2, size, d, 9)
    cache.k[7] = 1.0
    width = 400
    pages = [[-1] * width, [-1, 3] + [300] * (width - 2), [-1] * width]
    pages[2][250] = 7
    lengths, starts = [n + 5, 2 * size + n, 300 * size], [0, n, 2 * n, 3 * n]
    for dtype in ("f16", "bf16"):
        q = rows(3 * n, 4, d, dtype, 2)
        q[:, 1] = value
        q[:, 3, 5] = value
        got = ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts))
        assert not got[:n].any()
        clean = torch.nan_to_num(q, nan=0.0, posinf=0.0)
        check_attention(clean[:, ::2], cache, pages, lengths, starts, got=got[:, ::2])
        if value != value:
            assert torch.isnan(got[n:, 1::2]).all()
        near = ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts), window=size)
        assert not near[:n].any() and not near[n + size:2 * n].any() and not near[2 * n:].any()


def same(got, y, err):
    """As assert_near, element by element where the formula gives no finite value."""
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    assert torch.equal(torch.isinf(got), torch.isinf(y)) and torch.equal(got[torch.isinf(got)].double(), y[torch.isinf(y)])
    finite = torch.isfinite(y)
    assert_near(got[finite], y[finite], err[finite])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d, rotated", [(64, 32), (64, 0), (128, 128), (72, 40), (250, 0), (80, 16), (96, 2)])
def test_columns_that_are_not_rotated_keep_to_themselves(d, rotated, dtype):
    q, k, _ = make(40, 2, 1, d, dtype, 12)
    positions = torch.arange(40, dtype=torch.int32).cuda() + 1
    freq = ops.rotary_frequencies(rotated, device="cuda") if rotated else None
    for i in range(40):
        q[i, i % 2, (7 * i) % d] = (float("nan"), float("inf"), -float("inf"))[i % 3]
        k[i, 0, d - 1 - i] = (float("inf"), float("nan"))[i % 2]
    w = weights(d, torch.float32, 5)
    for interleaved in (False, True):
        for qw, kw in ((None, None), w):
            got = ops.head_norm_rotate(q, k, positions, freq, interleaved, qw, kw, kind="none")
            for x, y, weight in zip((q, k), got, (qw, kw)):
                same(y, *kvref.rotate(x if weight is None else x.double() * weight.double(), positions, freq, interleaved))
    if d % 16 == 0:
        cache = ops.KvCache.empty(10, 1, min(d, 128), 16)
        got = ops.kv_append(cache, k.nan_to_num(0.0, 0.0, 0.0), k.nan_to_num(0.0, 0.0, 0.0), ints([list(range(10))]), ints([41]), ints([0, 40]),
                            freq, q=q)
        same(got, *kvref.rotate(q, positions, freq))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, d", [(1, 64), (3, 128), (100, 64), (100, 128)])
def test_small_weights_count(n, d, dtype):
    """Weights of 2^-24.5 beside largest ones whose values are 0: as halves that reach no lower than 2^-24 they would be off by a third.
    Bound: 2^-11 of a weight's rounding, 2^-20 of exponential and sums, twice a score's 24.5 times 8 half steps of 2^-24 (q, scale and
    key are exact but for the scale's own rounding and its product with log2 e); and 2^-32 of the largest weight for each token."""
    size, length = 64, 8192
    cache = ops.KvCache.empty(length // size, 1, d, size)
    cache.k_scales.fill_(127)
    cache.v_scales.fill_(127)
    one = torch.tensor(1.0, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    k[..., 3] = one | 128
    v.fill_(int(one))
    k[:, :, ::16], v[:, :, ::16] = 0, 0
    q = torch.zeros(n, 2, d, dtype=DT[dtype], device="cuda")
    q[:, :, 3] = 24.5
    got = ops.kv_attention(q, cache, ints([list(range(length // size))]), ints([length]), ints([0, n]), scale=0.6931471805599453, causal=False)
    low = length * 15 / 16 * 2.0 ** -24.5
    want = low / (length / 16 + low)
    bound = (2.0 ** -11 + 2.0 ** -20 + 2 * 24.5 * 2.0 ** -21) * want + 2.0 ** -32 * length * 15 / 16 / (length / 16)
    f = torch.finfo(got.dtype)
    assert float((got.double() - want).abs().max()) <= bound + f.eps / 2 * (want + bound) + f.smallest_normal * f.eps


@pytest.mark.parametrize("n, length", [(1, 300), (1, 4096), (2, 30000), (3, 700), (200, 300), (100, 6000), (600, 600)])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_any_size(n, length, d):
    """Values that are all 1: whatever the scores, every row's result is 1, a weighted mean. Weights in halves are off by 2^-11 at most,
    the denominator, of as many exponentials in fp32, by less, the result's rounding by half a step."""
    size = 64
    total = -(-length // size)
    cache = random_cache(total, 2, size, d, 3, 0.0)
    cache.v[:] = 1.0
    cache.v_scales.fill_(127)
    table = ints([list(range(total))])
    for dtype in ("f16", "bf16"):
        q = rows(n, 8, d, dtype, 4)
        off = 2.0 ** -11 + 2.0 ** -20 + torch.finfo(q.dtype).eps / 2
        for e in (0, 10, 18, 20, 21, 22, 24, 26, 28, 30, 34, 40, 60):
            for sign in (1, -1):
                got = ops.kv_attention(q, cache, table, ints([length]), ints([0, n]), scale=sign * 2.0 ** e * d ** -0.5)
                assert float((got.double() - 1).abs().max()) <= off, (dtype, e, sign)


@pytest.mark.parametrize("n, length", [(1, 4096), (3, 30000), (100, 4196)])
@pytest.mark.parametrize("power", [18, 20, 24, 26, 27, 28])
def test_maxima_a_step_of_fp32_apart(n, length, power):
    """Scores of 1.5 2^power in 64 tokens and a step of 8 or more, up to 2^5, above that in the 64 behind them, and so on: the larger ones'
    values are 1, the others' 0. scale log2(e) is 1 in fp32, and all scores, sums and differences are exact."""
    size, d = 64, 64
    total = -(-length // size)
    cache = ops.KvCache.empty(total, 1, d, size)
    cache.k_scales.fill_(127)
    cache.v_scales.fill_(127)
    cache.k[:, :, :, 0] = 1.0
    cache.k[1::2, :, :, 1] = 1.0
    cache.v[1::2] = 1.0
    step = max(8.0, 2.0 ** (power - 23))
    q = torch.zeros(n, 2, d, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0], q[:, :, 1] = 1.5 * 2.0 ** power, step
    got = ops.kv_attention(q, cache, ints([list(range(total))]), ints([length]), ints([0, n]), scale=0.6931471824645996, causal=False)
    full = 64 * (total // 2) - (64 * total - length if total % 2 == 0 else 0)      # tokens of the larger score
    less = length - full
    want = full / (full + less * 2.0 ** -step)
    assert float((got.double() - want).abs().max()) <= 2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8
