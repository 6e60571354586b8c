"""Norm and rotation of heads on a B200 against 64 bits. The tolerance is the bound that kvref.rotate derives for an fp32 computation,
plus the output's rounding, half a step."""
import pytest
import torch

import kvref
from tracea_b200 import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def assert_near(got, y, err):
    f = torch.finfo(got.dtype)
    err = err + f.eps / 2 * (y.abs() + err) + f.smallest_normal * f.eps
    off = (got.double() - y).abs()
    assert bool((off <= err).all()), "%d of %d, worst %g of the bound" % (int((off > err).sum()), off.numel(), float((off / err).max()))


def make(t, h, kv, d, dtype, seed, fused=False):
    g = torch.Generator().manual_seed(seed)
    whole = (torch.randn(t, h + 2 * kv, d, generator=g) * torch.exp(torch.randn(1, h + 2 * kv, 1, generator=g))).to(DT[dtype]).cuda()
    parts = torch.split(whole, [h, kv, kv], dim=1)
    return parts if fused else [p.contiguous() for p in parts]


def weights(d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype).cuda() for _ in range(2)]


# tokens, heads, heads of keys, columns, rotated columns: every number of lanes a row takes, odd columns, parts rotated, one row
SHAPES = [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 5, 1, 80, 80), (7, 4, 2, 64, 32), (2, 3, 3, 16, 16), (5, 2, 1, 32, 16), (9, 6, 2, 96, 48),
          (4, 2, 2, 256, 256), (3, 1, 1, 192, 64), (6, 3, 1, 72, 40), (11, 7, 1, 250, 130), (513, 12, 4, 128, 64), (2000, 2, 1, 48, 16)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t, h, kv, d, rotated", SHAPES)
def test_norm_and_rotation(t, h, kv, d, rotated, dtype):
    freq = ops.rotary_frequencies(rotated, device="cuda")
    positions = torch.randint(0, 200000, (t,), generator=torch.Generator().manual_seed(t), dtype=torch.int32).cuda()
    for fused in (False, True):
        q, k, _ = make(t, h, kv, d, dtype, d + t, fused)
        qw, kw = weights(d, torch.float32 if t % 2 else DT[dtype], d)
        for interleaved in (False, True):
            for kind, w in (("rms", (qw, kw)), ("rms", (None, None)), ("none", (None, None))):
                got = ops.head_norm_rotate(q, k, positions, freq, interleaved, *w, kind=kind)
                for x, y, weight in zip((q, k), got, w):
                    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
                    assert_near(y, *kvref.rotate(x, positions, freq, interleaved, weight, kind))


def test_the_norm_alone_and_one_of_the_two():
    q, k, _ = make(10, 4, 2, 64, "bf16", 3)
    w = weights(64, torch.float32, 1)[0]
    got, none = ops.head_norm_rotate(q, None, q_weight=w)
    assert none is None
    assert_near(got, *kvref.rotate(q, weight=w, kind="rms"))
    none, got = ops.head_norm_rotate(None, k, torch.arange(10, dtype=torch.int32).cuda(), ops.rotary_frequencies(64, device="cuda"), kind="none")
    assert none is None
    assert_near(got, *kvref.rotate(k, torch.arange(10).cuda(), ops.rotary_frequencies(64, device="cuda")))


@pytest.mark.parametrize("shift", [1, 4, 8])
def test_rows_on_any_boundary_and_strides(shift):
    """Heads that start on 2-, 8- and 16-byte boundaries, tokens of odd strides, heads in front of tokens."""
    g = torch.Generator().manual_seed(shift)
    flat = torch.randn(40 * 1000, generator=g).to(torch.float16).cuda()
    positions = torch.arange(8, dtype=torch.int32).cuda() * 1000
    freq = ops.rotary_frequencies(64, device="cuda")
    for stride in ((64 * 3 + shift, 64, 1), (64, 64 * 8 + shift, 1)):
        q = torch.as_strided(flat, (8, 3, 64), stride, shift)
        got, _ = ops.head_norm_rotate(q, None, positions, freq, kind="none")
        assert_near(got, *kvref.rotate(q, positions, freq))


def test_far_and_negative_positions():
    """Angles of 2^31 turn in 64 bits: the float64 product itself is off by 2^-53 of the angle, 2^-21 here, times |a| + |b|."""
    q, _, _ = make(4, 2, 1, 128, "f32", 5)
    positions = torch.tensor([2 ** 31 - 1, -(2 ** 31), -1, 1 << 24], dtype=torch.int32).cuda()
    freq = ops.rotary_frequencies(128, device="cuda")
    got, _ = ops.head_norm_rotate(q, None, positions, freq, kind="none")
    y, err = kvref.rotate(q, positions, freq)
    assert_near(got, y, err + 4 * 2.0 ** -21 / U32 * err)


U32 = 32 * kvref.U      # kvref.rotate's bound, of |a| + |b|


def test_empty_and_not_finite_rows():
    q, k, _ = make(3, 2, 1, 64, "bf16", 6)
    empty = ops.head_norm_rotate(q[:0], k[:0])
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 1, 64)
    q[1, 0, 5] = float("nan")
    q[2, 1, 7] = float("inf")
    got, _ = ops.head_norm_rotate(q, None)
    bad = torch.isnan(got).any(-1)
    assert bad.tolist() == [[False, False], [True, False], [False, True]]


def test_streams_and_graphs():
    q, k, _ = make(100, 8, 2, 128, "bf16", 7)
    positions = torch.arange(100, dtype=torch.int32).cuda()
    freq = ops.rotary_frequencies(128, device="cuda")
    want = ops.head_norm_rotate(q, k, positions, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.head_norm_rotate(q, k, positions, freq)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.head_norm_rotate(q, k, positions, freq)
    q += 1
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    assert torch.equal(captured[0], ops.head_norm_rotate(q, k, positions, freq)[0]) and torch.equal(captured[1], want[1])
