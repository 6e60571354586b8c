"""Appending and attention on a B200 through what the Python calls do not reach -- outputs with strides, in place -- and in the rarer forms:
pairs of neighbours, parts of a head rotated, odd pairs, narrow heads in long pages, weights in 16 bits, one sequence after another."""
import ctypes

import pytest
import torch

import kvref
from test_heads_gpu import assert_near, make, weights
from test_kv_gpu import DT, check_append, check_attention, copies, ints, random_cache, rows, tables
from test_mx_gpu import status_ok
from tracea_b200 import ffi, ops

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def c_cache(cache):
    pages, heads, size, d = cache.k.shape
    return ffi.KvCache(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scales.data_ptr(), cache.v_scales.data_ptr(), pages, heads, size, d, 0)


def c_sequences(pages, lengths, starts):
    views = [ops._view(t) for t in (pages, lengths)] + ([ops._view(starts)] if starts is not None else [])
    s = ffi.Sequences(views[0].c, views[1].c, ctypes.pointer(views[2].c) if starts is not None else None)
    return s, views


@pytest.mark.parametrize("gap", [1, 4, 8])
@pytest.mark.parametrize("n, old", [(1, 700), (1, 20000), (150, 30), (70, 3000)])
def test_attention_into_strided_outputs(n, old, gap):
    """Heads of the output 2, 8 and 16 bytes apart from a 16-byte boundary, in every form; what lies between them stays."""
    cache = random_cache(700, 2, 64, 64, 3)
    lengths, pages = [old + n], tables([old + n], 64, 700, 5)
    starts = [0, n]
    q = rows(n, 8, 64, "bf16", 4)
    wide = torch.full((n, 8, 64 + gap), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, :, :64]
    s, alive = c_sequences(ints(pages), ints(lengths), ints(starts))
    st = ffi.load().tracea_kv_attention(ops._view(q).c, c_cache(cache), s, ctypes.byref(ops._view(out).c), ffi.KvAttentionParams(0.125, 1, 0, stream()))
    assert st == ffi.SUCCESS, ffi.last_error()
    check_attention(q, cache, pages, lengths, starts, got=out)
    assert bool((wide[:, :, 64:] == 7).all())
    status_ok()


def test_norm_and_rotation_in_place_and_into_slices():
    freq, positions = ops.rotary_frequencies(64, device="cuda"), torch.arange(50, dtype=torch.int32, device="cuda") * 37
    q, k, _ = make(50, 6, 2, 64, "f16", 8)
    want = [kvref.rotate(x, positions, freq, False, None, "rms") for x in (q, k)]
    wide = torch.zeros(50, 2, 67, dtype=torch.float16, device="cuda")
    out = wide[:, :, 1:65]
    vq, vk, vy = ops._view(q), ops._view(k), ops._view(out)
    hq = ffi.Heads(vq.c, None, ctypes.pointer(vq.c))
    hk = ffi.Heads(vk.c, None, ctypes.pointer(vy.c))
    vp = ops._view(positions)
    rot = ffi.Rotation(freq.data_ptr(), 32, 0)
    assert ffi.load().tracea_head_norm_rotate(ctypes.byref(hq), ctypes.byref(hk), 1, 1e-6, ctypes.byref(rot), ctypes.byref(vp.c), stream()) == ffi.SUCCESS
    torch.cuda.synchronize()
    assert_near(q, *want[0])
    assert_near(out, *want[1])
    assert not wide[:, :, 0].any() and not wide[:, :, 65:].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, d, size, rotated", [(2, 32, 128, 32), (3, 16, 128, 16), (2, 48, 64, 24), (1, 128, 32, 64), (2, 80, 128, 20), (4, 64, 16, 2)])
def test_append_of_neighbouring_pairs_and_parts(heads, d, size, rotated, dtype):
    sequences = [(0, 150), (5, 3), (size - 1, 40), (0, 1)]
    lengths = [a + b for a, b in sequences]
    starts = [sum(n for _, n in sequences[:i]) for i in range(5)]
    total = sum(-(-n // size) for n in lengths) + 1
    pages = tables(lengths, size, total, d)
    freq = ops.rotary_frequencies(rotated, device="cuda")
    k, v, q = (rows(starts[-1], h, d, dtype, i) for i, h in enumerate((heads, heads, 3 * heads)))
    kw, qw = weights(d, DT[dtype], 5)
    for interleaved in (False, True):
        cache = random_cache(total, heads, size, d, size)
        before = copies(cache)
        got = ops.kv_append(cache, k, v, ints(pages), ints(lengths), ints(starts), freq, interleaved, kw, q, qw, "rms", 1e-5)
        where = torch.tensor([w[1] for w in kvref.places(pages, lengths, starts, starts[-1], size, total)], device="cuda")
        vk, _ = kvref.rotate(k, where, freq, interleaved, kw, "rms", 1e-5)
        assert bool(torch.isfinite(vk).all())
        original = kvref.rotate

        def with_eps(x, positions, f, inter, w, kind):
            return original(x, positions, f, inter, w, kind, 1e-5)

        kvref.rotate = with_eps
        try:
            check_append(cache, before, k, v, pages, lengths, starts, freq, kw, "rms", interleaved)
        finally:
            kvref.rotate = original
        assert_near(got, *kvref.rotate(q, where, freq, interleaved, qw, "rms", 1e-5))


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(seed):
    """Prompts, pieces and tokens in one batch, with holes in the tables, against 64 bits."""
    r = __import__("random").Random(seed)
    kv = r.choice([1, 2, 3])
    h, d, size = kv * r.choice([1, 2, 5, 8, 12]), r.choice([16, 48, 64, 80, 128]), r.choice([16, 32, 64, 128])
    b = r.randint(1, 6)
    new = [r.choice([0, 1, 1, 2, r.randint(1, 40), r.randint(1, 300)]) for _ in range(b)]
    lengths = [n + r.choice([0, r.randint(0, 50), r.randint(0, 1500)]) for n in new]
    starts = [sum(new[:i]) for i in range(b + 1)]
    if starts[-1] == 0:
        new[0] = lengths[0] = 1
        starts = [0] + [1] * b
    total = sum(-(-n // size) for n in lengths) + 2
    pages = tables([max(n, 1) for n in lengths], size, total + b, seed)
    for row in pages:
        if r.random() < 0.4 and len(row) > 2:
            row[r.randrange(len(row) - 1)] = r.choice([-1, 10 ** 6])
    cache = random_cache(total + b, kv, size, d, seed)
    q = rows(starts[-1], h, d, r.choice(["f16", "bf16"]), seed)
    for causal, window in ((True, 0), (r.random() < 0.5, r.randint(1, 400))):
        check_attention(q, cache, pages, lengths, starts, causal, window)
    status_ok()


@pytest.mark.parametrize("h, kv", [(8, 2), (48, 1)])
def test_sequences_that_share_pages(h, kv):
    """A prefix that several sequences have in common, and a page that stands twice in one of them, are only read."""
    cache = random_cache(12, kv, 32, 64, 9)
    pages = [[3, 4, 5, 0], [3, 4, 6, 7], [3, 3, 4, -1], [5, 4, 3, 2]]
    lengths = [100, 128, 70, 96]
    check_attention(rows(4, h, 64, "f16", 1), cache, pages, lengths, None)
    check_attention(rows(185, h, 64, "f16", 2), cache, pages, lengths, [0, 90, 91, 155, 185], window=77)


@pytest.mark.parametrize("n, old", [(1, 500), (1, 30000), (20, 100), (150, 30), (100, 6000)])
def test_attention_in_place_with_rows_behind_the_last_sequence(n, old):
    """Every form reads what it needs of q before it writes there, and leaves the rows that belong to no sequence."""
    cache = random_cache(520, 2, 64, 128, 4)
    lengths, pages = [old + n], tables([old + n], 64, 520, 5)
    q = rows(n + 3, 10, 128, "bf16", 6)
    out = q.clone()
    s, alive = c_sequences(ints(pages), ints(lengths), ints([0, n]))
    v = ops._view(out)
    st = ffi.load().tracea_kv_attention(v.c, c_cache(cache), s, ctypes.byref(v.c), ffi.KvAttentionParams(128 ** -0.5, 1, 0, stream()))
    assert st == ffi.SUCCESS, ffi.last_error()
    check_attention(q[:n], cache, pages, lengths, [0, n], got=out[:n])
    assert torch.equal(out[n:], q[n:])
    status_ok()


def test_many_sequences_few_of_which_have_rows():
    new = [0] * 150
    new[3], new[31], new[32], new[100], new[149] = 40, 1, 200, 7, 1
    lengths = [n + 20 * (i % 3) for i, n in enumerate(new)]
    starts = [sum(new[:i]) for i in range(151)]
    pages = tables([max(n, 1) for n in lengths], 16, 1000, 2)
    cache = random_cache(1000, 2, 16, 80, 7)
    check_attention(rows(starts[-1], 8, 80, "f16", 3), cache, pages, lengths, starts)


def test_calls_of_no_rows_and_no_sequences():
    cache = random_cache(4, 2, 16, 64, 1)
    before = copies(cache)
    none, x, kv = ints([]), torch.empty(0, 4, 64, dtype=torch.float16, device="cuda"), torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    for pages, lengths, starts in ((ints([[0], [1]]), ints([3, 0]), ints([0, 0, 0])), (torch.empty(0, 3, dtype=torch.int32, device="cuda"), none, None)):
        assert ops.kv_append(cache, kv, kv, pages, lengths, starts, q=x).shape == x.shape
        assert ops.kv_attention(x, cache, pages, lengths, starts).shape == x.shape
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(copies(cache), before))
    q, k = ops.head_norm_rotate(x, kv)
    assert q.shape == x.shape and k.shape == kv.shape
