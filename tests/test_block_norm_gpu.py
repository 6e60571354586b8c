"""The norms around a block on a B200 against 64-bit ones. Tolerances are the bounds that mxref.norm derives for an fp32 computation,
plus the output's rounding, half a step."""
import ctypes

import numpy as np
import pytest
import torch

import mxref
from test_mx_gpu import DT, assert_quantized, status_ok
from tracea_b200 import ffi, ops

pytestmark = pytest.mark.gpu

EPS = 1e-6


def rows(m, c, dtype, seed, far=0.0):
    g = torch.Generator().manual_seed(seed * 1000003 + m * 1009 + c)
    return (torch.randn(m, c, generator=g) * torch.exp(torch.randn(m, 1, generator=g)) + far).to(DT[dtype]).cuda()


def vectors(c, groups, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    v = {"weight": 1 + 0.2 * torch.randn(c, generator=g), "bias": 0.3 * torch.randn(c, generator=g)}
    if groups:
        v.update({k: 0.3 * torch.randn(groups, c, generator=g) for k in ("scale", "shift", "gate")})
    return {k: t.to(dtype).cuda() for k, t in v.items()}


def d(t):
    return None if t is None else t.double().cpu().numpy()


def assert_rows(got, y, err):
    f = torch.finfo(got.dtype)
    err = err + f.eps / 2 * np.abs(y) + f.smallest_normal * f.eps
    off = np.abs(d(got) - y)
    assert (off <= err).all(), "%d of %d, worst %g of the bound" % ((off > err).sum(), off.size, (off / err).max())


def stage(v, names):
    return {k: v.get(k) for k in names}


# widths of every form -- a warp's, several rows to a CTA, one row to a CTA, the widest -- odd ones and ones a vector is not
SHAPES = [(1, 1), (5, 2), (7, 31), (300, 32), (33, 200), (64, 256), (9, 257), (40, 512), (65, 513), (20, 1000), (130, 1001), (12, 1024),
          (3, 2047), (50, 2048), (6, 4096), (5, 4097), (4, 8192), (3, 8200), (2, 16384), (2, 16383), (2000, 48)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, c", SHAPES)
def test_norm(m, c, dtype):
    x = rows(m, c, dtype, 1)
    groups = next(g for g in (5, 3, 2, 1) if m % g == 0)
    v = vectors(c, groups, torch.float32 if c % 3 else DT[dtype], c)
    for kind in ("rms", "layer", "none"):
        for names in ((), ("weight",), ("weight", "bias"), ("scale", "shift"), ("weight", "bias", "scale", "shift"), ("shift",)):
            s = stage(v, names)
            y, err = mxref.norm(d(x), kind, EPS, **{k: d(t) for k, t in s.items()})
            assert_rows(ops.block_norm(x, **s, kind=kind), y, err)
        s = stage(v, ("weight", "scale", "shift"))
        y, err = mxref.norm(d(x), kind, EPS, **{k: d(t) for k, t in s.items()})
        assert_quantized(ops.block_norm(x, **s, kind=kind, quantize=True), torch.from_numpy(y), torch.from_numpy(err))
    status_ok()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, c", SHAPES)
def test_join(m, c, dtype):
    h, x = rows(m, c, dtype, 2), rows(m, c, dtype, 3)
    groups = next(g for g in (4, 3, 1) if m % g == 0)
    v = vectors(c, groups, torch.float32 if c % 2 else DT[dtype], c + 1)
    for kind, names, gate, rs in (("rms", ("weight",), True, 1.0), ("layer", ("weight", "bias", "scale", "shift"), True, 0.5),
                                  ("none", (), True, 2.0), ("layer", (), False, 0.25), ("none", ("bias",), False, 1.0)):
        s = stage(v, names)
        y, err = mxref.norm(d(h), kind, EPS, **{k: d(t) for k, t in s.items()})
        g = np.repeat(d(v["gate"]), m // groups, axis=0) if gate else 1.0
        want = rs * d(x) + g * y
        # the products with gate and scale and their sum: half a step each, of terms no larger than these
        bound = err * np.abs(g) + 8 * 2.0 ** -24 * (np.abs(g * y) + np.abs(rs * d(x)))
        if s.get("scale") is not None or s.get("bias") is not None or s.get("shift") is not None:
            bound = bound + 8 * 2.0 ** -24 * np.abs(g) * (np.abs(y) + 4)
        args = dict(**s, gate=v["gate"] if gate else None, residual_scale=rs, kind=kind)
        r = ops.block_norm_add(h, x, **args)
        assert_rows(r, want, bound)
        # the next norm in the same pass: the bits of two calls
        for following in ({"kind": "rms", "weight": v["weight"]}, {"kind": "layer", "scale": v["scale"], "shift": v["shift"]}):
            r2, y2 = ops.block_norm_add(h, x, **args, following=following)
            assert torch.equal(r2, r) and torch.equal(y2, ops.block_norm(r, **following))
            r3, q = ops.block_norm_add(h, x, **args, following={**following, "quantize": True})
            q2 = ops.block_norm(r, **following, quantize=True)
            assert torch.equal(r3, r) and torch.equal(q.data, q2.data)
            assert torch.equal(q.dequantize(torch.float32), q2.dequantize(torch.float32))
    status_ok()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, c", [(600, 1024), (1001, 520), (1500, 1000), (640, 1001)])
def test_rows_of_a_warp(m, c, dtype):
    test_norm(m, c, dtype)
    test_join(m, c, dtype)


@pytest.mark.parametrize("dtype, far", [("f32", 1e4), ("f32", -1e6), ("bf16", 300.0)])
def test_rows_far_from_zero_keep_their_spread(dtype, far):
    x = rows(40, 1000, dtype, 4, far)
    y, err = mxref.norm(d(x), "layer", EPS)
    assert_rows(ops.block_norm(x, kind="layer"), y, err)


def test_constant_zero_and_broken_rows():
    for c in (40, 1000, 3000):
        x = rows(12, c, "f32", 5)
        x[1] = 0
        x[2] = 7.25
        clean = ops.block_norm(x, kind="layer")
        assert (clean[1] == 0).all() and (clean[2] == 0).all()
        assert (ops.block_norm(x)[1] == 0).all()
        x[3, 0], x[4, c - 1], x[5, c // 2] = float("nan"), float("inf"), float("-inf")
        for kind in ("rms", "layer"):
            got = ops.block_norm(x, kind=kind)
            assert got[3].isnan().all() and got[4].isnan().any() and got[5].isnan().any()
            q = ops.block_norm(x, kind=kind, quantize=True).dequantize(torch.float32)
            assert q[3].isnan().all() and q[4, -1].isnan() and not q[6:].isnan().any()
        rest = [0, 1, 2, 6, 7, 8, 9, 10, 11]
        assert torch.equal(ops.block_norm(x, kind="layer")[rest], clean[rest])
    assert (ops.block_norm(torch.zeros(2, 64, device="cuda"), eps=0.0)).isnan().all()     # 0 / 0


@pytest.mark.parametrize("c", [48, 1000, 2048, 2051])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_and_in_place(c, dtype):
    m = 30
    base = rows(m, c + 13, dtype, 6)
    h, x = base[:, 5:5 + c], rows(m, 2 * c, dtype, 7)[:, :c]
    v = vectors(c, 2, torch.float32, 1)
    w = v["weight"].repeat(2)[c // 2:c // 2 + c]                 # not at the start of its memory
    # rows that are 16-byte aligned are summed in another order than others, so each form is held to the bound, not to the other's bits
    y64, err = mxref.norm(d(h), "rms", EPS, d(w))
    gate = np.repeat(d(v["gate"]), m // 2, axis=0)
    want_r, bound_r = d(x) + gate * y64, err * np.abs(gate) + 8 * 2.0 ** -24 * (np.abs(gate * y64) + np.abs(d(x)))

    def right(r, y):
        assert_rows(r, want_r, bound_r)
        assert_rows(y, *mxref.norm(d(r), "rms", EPS, d(w)))

    right(*ops.block_norm_add(h.contiguous(), x.contiguous(), w.clone(), gate=v["gate"], following={"weight": w.clone()}))
    right(*ops.block_norm_add(h, x, w, gate=v["gate"], following={"weight": w}))
    # into views, the rest of which stays; r over x; the gate a slice of a wider matrix
    whole_x, whole_y = torch.full((m, c + 8), 3.0, device="cuda").to(DT[dtype]), torch.full((m + 1, c + 1), 3.0, device="cuda").to(DT[dtype])
    xr, yv = whole_x[:, 8:], whole_y[1:, 1:]
    xr.copy_(x)
    wide_gate = torch.zeros(2, c + 9, device="cuda")
    wide_gate[:, 9:] = v["gate"]
    as_view = lambda t: ffi.View(t.data_ptr(), t.shape, t.stride(), ops._DTYPES[t.dtype], 0)
    vh, vx, vy, vw, vg = (as_view(t) for t in (h, xr, yv, w, wide_gate[:, 9:]))
    n = ffi.Norm(ffi.NORM_RMS, EPS, ctypes.pointer(vw.c))
    stream = torch.cuda.current_stream().cuda_stream
    st = ffi.load().tracea_block_norm_add(vh.c, vx.c, ctypes.byref(n), ctypes.byref(vg.c), 1.0, ctypes.byref(vx.c), ctypes.byref(n),
                                          ctypes.byref(vy.c), None, stream)
    assert st == ffi.SUCCESS, ffi.last_error()
    torch.cuda.synchronize()
    right(xr, yv)
    assert (whole_x[:, :8] == 3).all() and (whole_y[0] == 3).all() and (whole_y[:, 0] == 3).all()
    before = xr.clone()
    st = ffi.load().tracea_block_norm(vx.c, ctypes.byref(n), ctypes.byref(vx.c), None, stream)
    assert st == ffi.SUCCESS, ffi.last_error()
    torch.cuda.synchronize()
    assert_rows(xr, *mxref.norm(d(before), "rms", EPS, d(w)))


@pytest.mark.parametrize("c", [40, 333, 1024, 2051, 5000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("quantize", [False, True])
def test_result_over_the_blocks_output(c, dtype, quantize):
    """r over h, with a norm behind it, more rows than the grid has CTAs; and an x that is one row for all."""
    m = 700
    h, x = rows(m, c, dtype, 10), rows(1, c, dtype, 11).expand(m, c)
    s = stage(vectors(c, 7, torch.float32, 3), ("scale", "shift"))
    want_r, want_y = ops.block_norm_add(h, x, **s, kind="layer", following={"kind": "rms", "quantize": quantize})
    y64, err = mxref.norm(d(h), "layer", EPS, scale=d(s["scale"]), shift=d(s["shift"]))
    assert_rows(want_r, d(x) + y64, err + 8 * 2.0 ** -24 * (2 * np.abs(y64) + 4 + np.abs(d(x))))
    as_view = lambda t: ffi.View(t.data_ptr(), t.shape, t.stride(), ops._DTYPES[t.dtype], 0)
    over, y = h.clone(), torch.empty_like(h)
    vh, vx, vs, vt, vy = (as_view(t) for t in (over, x, s["scale"], s["shift"], y))
    n = ffi.Norm(ffi.NORM_LAYER, EPS, None, None, ctypes.pointer(vs.c), ctypes.pointer(vt.c))
    f = ffi.Norm(ffi.NORM_RMS, EPS)
    q = ops.mx_quantize(h)
    mq = ffi.MxMatrix(q.data.data_ptr(), q.scales.data_ptr(), m, c, 0)
    st = ffi.load().tracea_block_norm_add(vh.c, vx.c, ctypes.byref(n), None, 1.0, ctypes.byref(vh.c), ctypes.byref(f),
                                          None if quantize else ctypes.byref(vy.c), ctypes.byref(mq) if quantize else None,
                                          torch.cuda.current_stream().cuda_stream)
    assert st == ffi.SUCCESS, ffi.last_error()
    torch.cuda.synchronize()
    assert torch.equal(over, want_r)
    assert torch.equal(q.data, want_y.data) if quantize else torch.equal(y, want_y)


def test_quantized_rows_leave_the_scales_of_rows_behind_them():
    x = rows(130, 300, "bf16", 8)
    lib = ffi.load()
    data = torch.full((130, 160), 255, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, 3, 512), 77, dtype=torch.uint8, device="cuda")
    q = ffi.MxMatrix(data.data_ptr(), scales.data_ptr(), 130, 300, 0)
    n = ffi.Norm(ffi.NORM_RMS, EPS)
    vx = ffi.View(x.data_ptr(), x.shape, x.stride(), ffi.DTYPE_BFLOAT16, 0)
    assert lib.tracea_block_norm(vx.c, ctypes.byref(n), None, ctypes.byref(q), None) == ffi.SUCCESS
    torch.cuda.synchronize()
    s = scales[1].cpu().numpy().reshape(3, 32, 4, 4)                       # rows 128 ..: 130 and on are untouched
    assert (s[:, 2:] == 77).all() and (s[:, :, 1:] == 77).all()
    codes, got, rest = mxref.unpack(data.cpu().numpy(), scales.cpu().numpy(), 130, 300)
    assert (rest == 0).all() and (codes[:, 300:] == 0).all()


def test_graph_replay_and_many_groups():
    x = rows(600, 1024, "bf16", 9)
    v = vectors(1024, 600, torch.float32, 2)
    s = stage(v, ("scale", "shift"))
    y, err = mxref.norm(d(x), "layer", EPS, scale=d(s["scale"]), shift=d(s["shift"]))
    assert_rows(ops.block_norm(x, **s, kind="layer"), y, err)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.block_norm(x, kind="layer")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = ops.block_norm(x, **s, kind="layer", quantize=True)
        out = ops.block_norm_add(q.dequantize(), x, gate=v["gate"], kind="none")
    for seed in range(3):
        x.copy_(rows(600, 1024, "bf16", 20 + seed))
        g.replay()
        torch.cuda.synchronize()
        q2 = ops.block_norm(x, **s, kind="layer", quantize=True)
        assert torch.equal(out, ops.block_norm_add(q2.dequantize(), x, gate=v["gate"], kind="none"))


def test_offsets_past_32_bits():
    m, c = 150000, 16384                              # 2.5 G elements
    x = torch.zeros(m, c, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, c, device="cuda").bfloat16()
    r, q = ops.block_norm_add(x, x, following={"quantize": True})
    want_r, want_q = ops.block_norm_add(x[-3:], x[-3:], following={"quantize": True})
    assert torch.equal(r[-3:], want_r) and torch.equal(q.data[-3:], want_q.data) and (r[:-3] == 0).all()
    status_ok()
