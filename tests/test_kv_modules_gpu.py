"""nn.MxAttention on a B200: the calls it makes, prompts and tokens in turn, graphs, and the kernels' failure path."""
import copy

import pytest
import torch

from test_kv_gpu import check_attention, copies, ints, random_cache, rows, tables
from test_mx_gpu import status_ok
from tracea_b200 import ffi, nn, ops

pytestmark = pytest.mark.gpu


def by_hand(block, x, cache, pages, lengths, starts, gate=None, scale=None, shift=None):
    w = lambda t: None if t is None else t.detach()      # noqa: E731
    n = ops.block_norm(x, w(block.pre_weight), scale=scale, shift=shift, kind=block.norm, eps=block.eps, quantize=True)
    h = ops.mx_gemm(n, ops.mx_quantize(w(block.qkv.weight)), dtype=x.dtype).view(x.shape[0], -1, block.head_dim)
    q, k, v = torch.split(h, [block.heads, block.kv_heads, block.kv_heads], dim=1)
    positions = torch.cat([torch.arange(int(m) - (b - a), int(m)) for m, a, b in zip(lengths, starts[:-1], starts[1:])]).int().cuda()
    kind = "none" if block.q_weight is None else "rms"
    turned, _ = ops.head_norm_rotate(q, None, positions, block._frequencies, q_weight=w(block.q_weight), kind=kind, eps=block.eps)
    ops.kv_append(cache, k, v, ints(pages), ints(lengths), ints(starts), block._frequencies, k_weight=w(block.k_weight), kind=kind, eps=block.eps)
    a = ops.kv_attention(turned, cache, ints(pages), ints(lengths), ints(starts), window=block.window)
    o = ops.mx_gemm(a.reshape(x.shape[0], -1), ops.mx_quantize(w(block.out.weight)))
    return ops.block_norm_add(o, x, w(block.post_weight), gate=gate, residual_scale=block.residual_scale, kind=block.norm, eps=block.eps)


@pytest.mark.parametrize("options", [{}, {"kv_heads": 2, "window": 33, "residual_scale": 0.5}, {"head_norm": False, "norm": "layer"}])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_module_is_the_calls_by_hand(options, dtype):
    """The queries of kv_append and of head_norm_rotate are computed by the same operations on the same values: the same bits, and so is
    the rest."""
    torch.manual_seed(0)
    block = nn.MxAttention(256, 4, device="cuda", **options)
    for p in (block.q_weight, block.k_weight):
        if p is not None:
            p.data += 0.1 * torch.randn_like(p)
    lengths, starts = [40, 17, 90], [0, 40, 57, 147]
    pages = tables([100] * 3, 16, 30, 1)
    x = torch.randn(147, 256, device="cuda").to(dtype)
    mine, other = block.cache(30, 16), block.cache(30, 16)
    g = 0.5 * torch.randn(3, 1, 256, device="cuda")
    extra = {"gate": g[0], "scale": g[1], "shift": g[2]}
    got = block(x, mine, ints(pages), ints(lengths), ints(starts), **extra)
    want = by_hand(block, x, other, pages, lengths, starts, **extra)
    assert torch.equal(got, want) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(copies(mine), copies(other)))
    status_ok()


def test_prompt_in_pieces_tokens_and_a_graph():
    """A layer of attention and feed-forward: pieces of a prompt, then tokens, eagerly and from a graph; copies of the module agree."""
    torch.manual_seed(1)
    layer = [nn.MxAttention(256, 4, 2, device="cuda"), nn.MxFeedForward(256, 512, device="cuda")]
    pages = ints(tables([80, 80], 32, 10, 3))
    x = [torch.randn(n, 256, device="cuda").bfloat16() for n in (33, 20, 2, 2, 2)]
    calls = [([20, 13], [0, 20, 33]), ([30, 23], [0, 10, 20]), ([31, 24], None), ([32, 25], None), ([33, 26], None)]

    def run(attention, feed, cache):
        return [feed(attention(v, cache, pages, ints(n), None if s is None else ints(s))) for v, (n, s) in zip(x, calls)]

    want = run(*layer, layer[0].cache(10, 32))
    twin = copy.deepcopy(layer)
    assert all(torch.equal(a, b) for a, b in zip(want, run(*twin, twin[0].cache(10, 32))))
    cache = layer[0].cache(10, 32)
    for v, (n, s) in list(zip(x, calls))[:2]:
        layer[1](layer[0](v, cache, pages, ints(n), ints(s)))
    token, lengths = x[2].clone(), ints([30, 23])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths += 1
        y = layer[1](layer[0](token, cache, pages, lengths))
    for i in (2, 3, 4):
        token.copy_(x[i])
        graph.replay()
        assert torch.equal(y, want[i])
    status_ok()


def test_two_graphs_and_an_eager_call_at_once():
    """Captured calls own what they join their sums in: two graphs on two streams and eager calls beside them keep to their own."""
    cache = random_cache(2100, 1, 64, 128, 4)
    pages, lengths = ints([list(range(1000)), list(range(1000, 2000))]), ints([64000, 50001])      # long: split over all CTAs
    qs = [rows(2, 8, 128, "bf16", 20 + i) for i in range(3)]
    want = [ops.kv_attention(q, cache, pages, lengths) for q in qs]
    graphs, outs = [], []
    for q in qs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv_attention(q, cache, pages, lengths))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        got = ops.kv_attention(qs[2], cache, pages, lengths)
    torch.cuda.synchronize()
    assert torch.equal(got, want[2]) and all(torch.equal(a, b) for a, b in zip(outs, want))


def test_every_form_of_attention_is_taken():
    """One token of a short sequence, of a long one, a prompt, and a batch with both: cluster, line, tiles of rows, two kernels."""
    cache = random_cache(400, 2, 64, 64, 8)
    few, many = (lambda: ffi.launch_count_of(12)), (lambda: ffi.launch_count_of(13))
    for lengths, starts, expect in (([100], None, (1, 0)), ([20000], None, (2, 0)), ([100], [0, 100], (0, 1)), ([100, 300], [0, 1, 101], (1, 1)),
                                    ([100], [0, 3], (1, 0))):
        pages = tables(lengths, 64, 400, 1)
        q = rows(len(lengths) if starts is None else starts[-1], 8, 64, "f16", 3)
        before = few(), many()
        got = ops.kv_attention(q, cache, ints(pages), ints(lengths), None if starts is None else ints(starts))
        assert (few() - before[0], many() - before[1]) == expect, (lengths, starts)
        check_attention(q, cache, pages, lengths, starts, got=got)


def test_a_wait_that_runs_out_is_reported_and_the_device_stays_usable():
    """The warps that widen the cache's elements go silent after two steps: the waits behind them run out, the kernel returns."""
    lib = ffi.load()
    cache = random_cache(40, 2, 64, 128, 5)
    pages, lengths, starts = [list(range(20))], [1200], [0, 1200]
    q = rows(1200, 4, 128, "bf16", 6)
    check_attention(q, cache, pages, lengths, starts)
    assert lib.tracea_b200_device_status(0) == 0
    try:
        lib.tracea_b200_test_hooks(400000, 2)
        ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts))
        torch.cuda.synchronize()
    finally:
        lib.tracea_b200_test_hooks(0, -1)
    with pytest.raises(ffi.TraceaError, match="gave up a bounded wait"):
        ops.kv_attention(q, cache, ints(pages), ints(lengths), ints(starts))
    assert lib.tracea_b200_device_status(0) == 0
    check_attention(q, cache, pages, lengths, starts)
