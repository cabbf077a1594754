"""ngp_hip_gated_ffn_forward / _backward on the GPU against 64-bit values, element by element, within the bounds that tests/ffn_reference.py derives."""
import numpy as np
import pytest
import torch

import capi
import ffn_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": (torch.float16, 0), "bf16": (torch.bfloat16, 1)}
SENTINEL = 1234.0


def block(d, f, o, dtype, act):
    b = np.zeros(1, capi.GATED_FFN)
    b["n_in"], b["n_hidden"], b["n_out"], b["dtype"], b["activation"] = d, f, o, TYPES[dtype][1], R.ACTS[act]
    return b


def inputs(rows, d, f, o, dtype, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)   # noqa: E731
    t = TYPES[dtype][0]
    return (r(rows, d).to(t), (r(f, d) * d ** -0.5).to(t), (r(f, d) * d ** -0.5).to(t), (r(o, f) * f ** -0.5).to(t), (r(rows, o) * max(rows, 1) ** -0.5).to(t))


def strided(t, stride, offset=0):
    """t with another row stride and base offset (in elements), sentinels around it"""
    buf = torch.full((t.shape[0] * stride + offset + 64,), SENTINEL, dtype=t.dtype, device=t.device)
    v = buf.as_strided(t.shape, (stride, 1), offset)
    v.copy_(t)
    return buf, v


def guarded(rows, cols, stride, dtype, offset=0):
    return strided(torch.zeros(rows, cols, dtype=dtype, device="cuda"), stride, offset)


def untouched(buf, view):
    seen = torch.ones_like(buf, dtype=torch.bool)
    seen.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
    assert (buf[seen] == SENTINEL).all(), "a value outside the output was written"


def workspace(ngp, b, rows, flags, extra=0):
    n = ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, rows, flags)
    ws = torch.full((n + 256,), 0xff, dtype=torch.uint8, device="cuda")   # NaNs: nothing may rely on what was there
    return ws, n


def forward(ngp, b, x, wg, wu, wd, y, ws, n, stream=None):
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    capi.check(ngp.ngp_hip_gated_ffn_forward(s, b.ctypes.data, x.shape[0], x.data_ptr(), x.stride(0), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), y.data_ptr(), y.stride(0), ws.data_ptr(), n))


def backward(ngp, b, x, wg, wu, wd, dy, dx, grads, ws, n, stream=None):
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    g = [None if grads is None else t.data_ptr() for t in (grads or (0, 0, 0))]
    capi.check(ngp.ngp_hip_gated_ffn_backward(s, b.ctypes.data, x.shape[0], x.data_ptr(), x.stride(0), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dy.data_ptr(), dy.stride(0),
                                              None if dx is None else dx.data_ptr(), 0 if dx is None else dx.stride(0), g[0], g[1], g[2], ws.data_ptr(), n))


# (rows, n_in, n_hidden, n_out): single rows and columns, widths around the vector and tile sizes, k that ends inside a step, rows that end inside a tile, split sums,
# few rows (the row-streaming kernels), narrow blocks over many rows, and sizes whose tiles fill the chip for each product
SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (1, 64, 128, 64), (1, 520, 1032, 264), (3, 7, 5, 9), (2, 333, 77, 130), (16, 72, 264, 40), (17, 256, 96, 48), (1, 136, 264, 136), (33, 129, 130, 131), (64, 300, 500, 200), (65, 300, 500, 200), (24, 1024, 2056, 520), (9, 2000, 130, 24), (33, 64, 64, 64), (20, 8200, 8200, 40), (33, 2001, 8011, 131), (64, 1030, 4100, 72),
          (64, 32, 64, 16), (65, 33, 65, 17), (129, 128, 96, 257), (300, 40, 200, 3), (513, 264, 328, 136), (4097, 32, 64, 16), (5000, 16, 32, 8), (3000, 64, 128, 64),
          (2500, 96, 160, 32), (4500, 8, 64, 16), (6200, 136, 1000, 2056), (6200, 136, 1400, 72), (3000, 1200, 2600, 1100), (40000, 72, 136, 72), (200, 1600, 4104, 3000)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_against_64_bits(ngp, cuda, shape, dtype):
    rows, d, f, o = shape
    for act in (["silu", "relu"] if rows > 1000 else sorted(R.ACTS)):
        b = block(d, f, o, dtype, act)
        x, wg, wu, wd, dy = inputs(rows, d, f, o, dtype, seed=rows + d)
        ref = R.Block(act, x, wg, wu, wd, dy)
        ybuf, y = guarded(rows, o, o, x.dtype)
        ws, n = workspace(ngp, b, rows, 0)
        forward(ngp, b, x, wg, wu, wd, y, ws, n)
        torch.cuda.synchronize()
        R.check("y " + act, y, ref.y, ref.ey)
        untouched(ybuf, y)
        assert (ws[n:] == 0xff).all()
        ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
        outs = [guarded(*s, s[1], x.dtype) for s in ((rows, d), (f, d), (f, d), (o, f))]
        backward(ngp, b, x, wg, wu, wd, dy, outs[0][1], [v for _, v in outs[1:]], ws, n)
        torch.cuda.synchronize()
        for name, (buf, v), want, bound in zip(("dx", "dw_gate", "dw_up", "dw_down"), outs, (ref.dx, ref.dwg, ref.dwu, ref.dwd), (ref.edx, ref.edwg, ref.edwu, ref.edwd)):
            R.check(name + " " + act, v, want, bound)
            untouched(buf, v)
        assert (ws[n:] == 0xff).all()


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
@pytest.mark.parametrize("widths", [(64, 96, 48), (33, 65, 17), (32, 64, 16), (136, 200, 144), (133, 161, 139), (2051, 6205, 24)], ids=lambda w: "x".join(map(str, w)))
@pytest.mark.parametrize("layout", ["aligned stride", "odd stride", "odd base"])
def test_strides_and_alignment(ngp, cuda, rows, widths, layout):
    d, f, o = widths
    extra, offset = {"aligned stride": (8, 0), "odd stride": (3, 0), "odd base": (8, 1)}[layout]
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "f16", seed=3)
    _, xs = strided(x, d + extra, offset)
    _, dys = strided(dy, o + extra, offset)
    ws_ = [strided(w, w.shape[1], offset)[1] for w in (wg, wu, wd)]
    b = block(d, f, o, "f16", "silu")
    ref = R.Block("silu", x, wg, wu, wd, dy)
    any_layout = 0 if layout == "aligned stride" else capi.FFN_ANY_LAYOUT
    ybuf, y = guarded(rows, o, o + extra, x.dtype, offset)
    ws, n = workspace(ngp, b, rows, any_layout)
    forward(ngp, b, xs, *ws_, y, ws, n)
    dxbuf, dx = guarded(rows, d, d + extra, x.dtype, offset)
    grads = [guarded(*w.shape, w.shape[1], x.dtype, offset) for w in (wg, wu, wd)]
    ws2, n2 = workspace(ngp, b, rows, any_layout | capi.FFN_BACKWARD)
    backward(ngp, b, xs, *ws_, dys, dx, [v for _, v in grads], ws2, n2)
    torch.cuda.synchronize()
    R.check("y", y, ref.y, ref.ey)
    R.check("dx", dx, ref.dx, ref.edx)
    for name, (buf, v), want, bound in zip(("dw_gate", "dw_up", "dw_down"), grads, (ref.dwg, ref.dwu, ref.dwd), (ref.edwg, ref.edwu, ref.edwd)):
        R.check(name, v, want, bound)
        untouched(buf, v)
    untouched(ybuf, y)
    untouched(dxbuf, dx)


def test_gradients_against_differences(ngp, cuda):
    """<dy, y(x + t v) - y(x - t v)> / 2t in 64 bits against <gradient, v>: the gradients' own definition, apart from the formulas of the reference"""
    rows, d, f, o = 37, 48, 72, 24
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "f16", seed=11)
    b = block(d, f, o, "f16", "gelu")
    ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    outs = [torch.empty_like(t) for t in (x, wg, wu, wd)]
    backward(ngp, b, x, wg, wu, wd, dy, outs[0], outs[1:], ws, n)
    torch.cuda.synchronize()
    ref = R.Block("gelu", x, wg, wu, wd, dy)
    t = 1e-5
    for k, (grad, bound) in enumerate(zip(outs, (ref.edx, ref.edwg, ref.edwu, ref.edwd))):
        v = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda", dtype=torch.float64)
        ends = []
        for s in (t, -t):
            args = [w.double() for w in (x, wg, wu, wd)]
            args[k] = args[k] + s * v
            g = args[0] @ args[1].T
            ends.append(((g * torch.special.ndtr(g) * (args[0] @ args[2].T)) @ args[3].T * dy.double()).sum())
        # third derivatives are of order one here: t^2 of the sum of 37 x 24 terms; 64-bit cancellation 1e-16 / t
        assert abs((ends[0] - ends[1]).item() / (2 * t) - (grad.double() * v).sum().item()) <= (bound * v.abs()).sum().item() + 1e-6


@pytest.mark.parametrize("rows", [0, 1])
def test_empty_and_single_row(ngp, cuda, rows):
    d, f, o = 40, 56, 24
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "bf16")
    b = block(d, f, o, "bf16", "silu")
    ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    grads = [guarded(*w.shape, w.shape[1], x.dtype) for w in (wg, wu, wd)]
    dx = torch.empty_like(x)
    y = torch.empty(rows, o, dtype=x.dtype, device="cuda")
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    backward(ngp, b, x, wg, wu, wd, dy, dx if rows else None, [v for _, v in grads], ws, n)
    torch.cuda.synchronize()
    ref = R.Block("silu", x, wg, wu, wd, dy)
    for (buf, v), want, bound in zip(grads, (ref.dwg, ref.dwu, ref.dwd), (ref.edwg, ref.edwu, ref.edwd)):
        untouched(buf, v)
        if rows:
            R.check("grad", v, want, bound)
        else:
            assert (v == 0).all()   # a sum over nothing, written


def test_parts_of_the_backward_pass(ngp, cuda):
    """dx alone and the weight gradients alone are the bits of the whole call"""
    rows, d, f, o = 200, 64, 136, 72
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "f16", seed=5)
    b = block(d, f, o, "f16", "relu")
    ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    whole = [torch.empty_like(t) for t in (x, wg, wu, wd)]
    part = [torch.empty_like(t) for t in (x, wg, wu, wd)]
    backward(ngp, b, x, wg, wu, wd, dy, whole[0], whole[1:], ws, n)
    backward(ngp, b, x, wg, wu, wd, dy, part[0], None, ws, n)
    backward(ngp, b, x, wg, wu, wd, dy, None, part[1:], ws, n)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(whole, part))


@pytest.mark.parametrize("shape", [(1, 64, 128, 64), (40, 64, 128, 64), (700, 32, 64, 16), (300, 256, 512, 128)], ids=lambda s: "x".join(map(str, s)))
def test_non_finite_rows_stay_in_their_rows(ngp, cuda, shape):
    rows, d, f, o = shape
    b = block(d, f, o, "f16", "silu")
    x, wg, wu, wd, _ = inputs(rows, d, f, o, "f16", seed=7)
    ws, n = workspace(ngp, b, rows, 0)
    y0, y1 = (torch.empty(rows, o, dtype=x.dtype, device="cuda") for _ in range(2))
    forward(ngp, b, x, wg, wu, wd, y0, ws, n)
    bad = rows // 2
    x[bad, 3] = float("nan")
    forward(ngp, b, x, wg, wu, wd, y1, ws, n)
    torch.cuda.synchronize()
    keep = torch.arange(rows, device="cuda") != bad
    assert torch.isnan(y1[bad]).all() and torch.equal(y0[keep], y1[keep])


@pytest.mark.parametrize("act", sorted(R.ACTS))
def test_far_arguments(ngp, cuda, act):
    """|g| up to thousands: the exponentials saturate to their limits, nothing becomes a NaN"""
    d, f, o = 8, 16, 8
    x = torch.zeros(64, d, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.linspace(-3000, 3000, 64, device="cuda")
    wg, wu = torch.zeros(f, d, device="cuda").bfloat16(), torch.zeros(f, d, device="cuda").bfloat16()
    wg[:, 0], wu[:, 0] = 1, 2.0 ** -10
    wd = torch.zeros(o, f, device="cuda").bfloat16()
    wd[:, 0] = 1
    b = block(d, f, o, "bf16", act)
    ws, n = workspace(ngp, b, 64, capi.FFN_BACKWARD)
    y, dy = torch.empty(64, o, dtype=x.dtype, device="cuda"), torch.ones(64, o, dtype=x.dtype, device="cuda")
    outs = [torch.empty_like(t) for t in (x, wg, wu, wd)]
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    backward(ngp, b, x, wg, wu, wd, dy, outs[0], outs[1:], ws, n)
    torch.cuda.synchronize()
    ref = R.Block(act, x, wg, wu, wd, dy)
    # the smallest |g| is 47, the largest 3000: the exponential is 0 or inf, or its argument's rounding moves it by 3000 x 2^-24 of values below 1e-20
    R.check("y", y, ref.y, ref.ey + 1e-18)
    for v, want, bound in zip(outs, (ref.dx, ref.dwg, ref.dwu, ref.dwd), (ref.edx, ref.edwg, ref.edwu, ref.edwd)):
        R.check("gradient", v, want, bound + 1e-15)


@pytest.mark.parametrize("shape", [(1, 256, 512, 128), (50, 64, 96, 32), (5000, 32, 64, 16), (700, 128, 320, 72)], ids=lambda s: "x".join(map(str, s)))
def test_same_bits_every_time_on_another_stream_and_in_a_graph(ngp, cuda, shape):
    rows, d, f, o = shape
    b = block(d, f, o, "bf16", "silu")
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "bf16", seed=9)
    n = max(ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, rows, k) for k in (0, capi.FFN_BACKWARD))

    def buffers():
        return torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty(rows, o, dtype=x.dtype, device="cuda"), [torch.empty_like(t) for t in (x, wg, wu, wd)]

    def step(ws, y, outs):
        forward(ngp, b, x, wg, wu, wd, y, ws, n)
        backward(ngp, b, x, wg, wu, wd, dy, outs[0], outs[1:], ws, n)

    eager, other, captured = buffers(), buffers(), buffers()
    step(*eager)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*other)
    torch.cuda.synchronize()
    assert torch.equal(eager[1], other[1]) and all(torch.equal(p, q) for p, q in zip(eager[2], other[2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*captured)
    for k in range(3):   # new inputs in the same tensors, eager work between the replays
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(100 + k), device="cuda"))
        graph.replay()
        step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(eager[1], captured[1]) and all(torch.equal(p, q) for p, q in zip(eager[2], captured[2]))


@pytest.mark.parametrize("widths", [(32, 64, 16), (136, 264, 72)], ids=lambda w: "x".join(map(str, w)))
def test_rows_whose_offsets_pass_32_bits(ngp, cuda, widths):
    """a row stride that puts the last rows behind 2^32 bytes of the first, and weights of the gradient summed over them"""
    (d, f, o), rows, stride = widths, 1100, 1 << 21
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "f16", seed=13)
    buf = torch.empty(rows * stride, dtype=torch.float16, device="cuda")   # 4.6 GB, only the rows are written
    xs = buf.as_strided((rows, d), (stride, 1))
    xs.copy_(x)
    b = block(d, f, o, "f16", "silu")
    ref = R.Block("silu", x, wg, wu, wd, dy)
    ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    y, outs = torch.empty(rows, o, dtype=x.dtype, device="cuda"), [torch.empty_like(t) for t in (x, wg, wu, wd)]
    forward(ngp, b, xs, wg, wu, wd, y, ws, n)
    backward(ngp, b, xs, wg, wu, wd, dy, outs[0], outs[1:], ws, n)
    torch.cuda.synchronize()
    R.check("y", y, ref.y, ref.ey)
    for v, want, bound in zip(outs, (ref.dx, ref.dwg, ref.dwu, ref.dwd), (ref.edx, ref.edwg, ref.edwu, ref.edwd)):
        R.check("gradient", v, want, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_gelu_far_out(ngp, cuda, dtype):
    """g = u = x up to where Phi(-x) is 1e-9: one column of everything, the weights 1.  h and y are rounded once each, the activation itself within 1e-5 of its value."""
    t = TYPES[dtype][0]
    x = torch.linspace(-6, 6, 4099, device="cuda").to(t).view(-1, 1)
    one = torch.ones(1, 1, device="cuda", dtype=t)
    b = block(1, 1, 1, dtype, "gelu")
    ws, n = workspace(ngp, b, len(x), 0)
    y = torch.empty_like(x)
    forward(ngp, b, x, one, one, one, y, ws, n)
    torch.cuda.synchronize()
    want = (x.double() ** 2 * torch.special.ndtr(x.double()))
    smallest = torch.finfo(t).tiny * torch.finfo(t).eps   # half a step of f16's subnormal values, twice
    assert ((y.double() - want).abs() <= (torch.finfo(t).eps + 1.1e-5) * want.abs() + smallest).all()


# 24 to 48 rows of the weights to a workgroup, for h and for y; x packed or not
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 40, 4500, 10001), (3, 41, 10001, 4500), (12, 40, 4500, 10001), (12, 41, 10001, 4500), (24, 40, 4500, 10001), (24, 41, 10001, 4500), (50, 40, 4500, 5001),
                                   (16, 16000, 4500, 40), (16, 12000, 10001, 40), (24, 9500, 4500, 40), (24, 4001, 10001, 40), (50, 4001, 4500, 40), (2, 30, 17000, 21000)], ids=lambda s: "x".join(map(str, s)))
def test_few_rows_through_many_columns(ngp, cuda, shape, dtype):
    rows, d, f, o = shape
    b = block(d, f, o, dtype, "silu")
    x, wg, wu, wd, dy = inputs(rows, d, f, o, dtype, seed=rows + f)
    ref = R.Block("silu", x, wg, wu, wd, dy)
    ybuf, y = guarded(rows, o, o, x.dtype)
    ws, n = workspace(ngp, b, rows, 0)
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    torch.cuda.synchronize()
    R.check("y", y, ref.y, ref.ey)
    untouched(ybuf, y)
    assert (ws[n:] == 0xff).all()


@pytest.mark.parametrize("shape", [(3, 5, 1 << 20, 2), (3, 1 << 20, 5, 2), (3, 2, 5, 1 << 20), (70, 5, 1 << 20, 2), (70, 1 << 20, 5, 2), (70, 2, 5, 1 << 20), (3000001, 8, 16, 4), (400003, 136, 72, 40)],
                         ids=lambda s: "x".join(map(str, s)))
def test_the_widest_and_longest(ngp, cuda, shape):
    rows, d, f, o = shape
    b = block(d, f, o, "f16", "relu")
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "f16", seed=rows)
    ref = R.Block("relu", x, wg, wu, wd, dy)
    y, outs = torch.empty(rows, o, dtype=x.dtype, device="cuda"), [torch.empty_like(t) for t in (x, wg, wu, wd)]
    ws, n = workspace(ngp, b, rows, 0)
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    ws2, n2 = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    backward(ngp, b, x, wg, wu, wd, dy, outs[0], outs[1:], ws2, n2)
    torch.cuda.synchronize()
    R.check("y", y, ref.y, ref.ey)
    for name, v, want, bound in zip(("dx", "dw_gate", "dw_up", "dw_down"), outs, (ref.dx, ref.dwg, ref.dwu, ref.dwd), (ref.edx, ref.edwg, ref.edwu, ref.edwd)):
        R.check(name, v, want, bound)
    assert (ws[n:] == 0xff).all() and (ws2[n2:] == 0xff).all()


@pytest.mark.parametrize("shape", [(24, 1024, 2056, 520), (700, 264, 520, 136), (3000, 32, 64, 16)], ids=lambda s: "x".join(map(str, s)))
def test_two_streams_at_once_and_graphs_that_share_a_workspace(ngp, cuda, shape):
    rows, d, f, o = shape
    b = block(d, f, o, "f16", "gelu")
    sets = [inputs(rows, d, f, o, "f16", seed=s) for s in (1, 2)]
    n = max(ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, rows, k) for k in (0, capi.FFN_BACKWARD))

    def fresh():
        return torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), torch.empty(rows, o, dtype=torch.float16, device="cuda"), [torch.empty_like(t) for t in sets[0][:4]]

    def both(i, ws, y, outs):
        x, wg, wu, wd, dy = sets[i]
        forward(ngp, b, x, wg, wu, wd, y, ws, n)
        backward(ngp, b, x, wg, wu, wd, dy, outs[0], outs[1:], ws, n)

    want, got, streams = [fresh(), fresh()], [fresh(), fresh()], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        both(i, *want[i])
    torch.cuda.synchronize()
    for _ in range(5):   # in turn, so that the two streams' kernels lie beside each other
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                both(i, *got[i])
    torch.cuda.synchronize()
    same = lambda a, c: torch.equal(a[1], c[1]) and all(torch.equal(u, v) for u, v in zip(a[2], c[2]))   # noqa: E731
    assert all(same(want[i], got[i]) for i in range(2))
    shared, graphs = fresh()[0], []
    for i in range(2):
        got[i][1].zero_()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            both(i, shared, *got[i][1:])
    for _ in range(3):
        for i in (0, 1, 0):
            got[i][1].fill_(-1.0)
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(same(want[i], got[i]) for i in range(2))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 32, 64, 16), (3, 256, 512, 128), (20, 256, 512, 128), (24, 9500, 4500, 40), (300, 256, 512, 128), (700, 2048, 4096, 256)], ids=lambda s: "x".join(map(str, s)))
def test_the_range_of_the_hidden_row(ngp, cuda, shape, dtype):
    """h = g u with g and u single products of powers of two: in f16 exact down to 2^-24 and up to 65504, infinite beyond and in its own row only; in bf16 far beyond that"""
    rows, d, f, o = shape
    t = TYPES[dtype][0]
    x, wg, wu, wd = (torch.zeros(s, device="cuda", dtype=t) for s in ((rows, d), (f, d), (f, d), (o, f)))
    wg[:, 0], wu[:, 1], wd[:, f - 1] = 1.0, 1.0, 2.0 ** -3
    x[0, 0], x[0, 1] = 2.0 ** 8, 255.0 + 0.875 if dtype == "f16" else 255.0    # f16: 65504, the largest
    x[1, 0], x[1, 1] = 2.0 ** -12, 3 * 2.0 ** -12                              # 3 steps of f16's smallest
    x[2, 0], x[2, 1] = 2.0 ** 10, -2.0 ** 10                                   # 2^20: beyond f16, and y would not be
    b = block(d, f, o, dtype, "none")
    ws, n = workspace(ngp, b, rows, 0)
    y = torch.full((rows, o), SENTINEL, device="cuda", dtype=t)
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    torch.cuda.synchronize()
    h = x[:, 0].double() * x[:, 1].double()
    want = (h / 8).to(t)   # exact in both types but for the smallest in f16: 3 2^-27 is rounded to nothing
    assert torch.equal(y[3:], torch.zeros_like(y[3:])) and (y[0] == want[0]).all() and (y[1] == want[1]).all()
    # f16: every hidden value of that row is minus infinity, and all weights of y but one are zero: a sum of infinity times zero is a NaN
    assert not torch.isfinite(y[2]).any() if dtype == "f16" else (y[2] == want[2]).all()
    wd[:, f - 1] = 2.0 ** 6   # what f16 holds of the small ones is all there
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    torch.cuda.synchronize()
    assert (y[1] == 3 * 2.0 ** -18).all()


@pytest.mark.parametrize("bad_value", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("shape", [(2, 256, 512, 128), (5, 256, 512, 128), (12, 256, 512, 128), (24, 9500, 4500, 40), (50, 9500, 4500, 40), (33, 2001, 8011, 131), (70, 300, 500, 200)], ids=lambda s: "x".join(map(str, s)))
def test_non_finite_rows_among_few(ngp, cuda, shape, bad_value):
    """the streaming kernels, rows packed and not (their packed rows behind the last are never written), and the tiles behind them; the first row, a middle one, the last"""
    rows, d, f, o = shape
    b = block(d, f, o, "f16", "silu")
    x, wg, wu, wd, _ = inputs(rows, d, f, o, "f16", seed=7)
    ws, n = workspace(ngp, b, rows, 0)
    y0, y1 = (torch.empty(rows, o, dtype=x.dtype, device="cuda") for _ in range(2))
    forward(ngp, b, x, wg, wu, wd, y0, ws, n)
    for bad in {0, rows // 2, rows - 1}:
        x1 = x.clone()
        x1[bad, 3] = bad_value
        ws.fill_(0xff)
        forward(ngp, b, x1, wg, wu, wd, y1, ws, n)
        torch.cuda.synchronize()
        keep = torch.arange(rows, device="cuda") != bad
        assert not torch.isfinite(y1[bad]).any() and torch.equal(y0[keep], y1[keep]) and torch.isfinite(y0).all()


@pytest.mark.parametrize("shape", [(40, 32, 64, 16), (5, 256, 512, 128), (70, 300, 500, 200), (700, 264, 520, 136)], ids=lambda s: "x".join(map(str, s)))
def test_a_non_finite_row_of_the_backward_pass_stays_in_its_row_of_dx(ngp, cuda, shape):
    """the weights' gradients are sums over the rows: all of them have it"""
    rows, d, f, o = shape
    b = block(d, f, o, "bf16", "gelu")
    x, wg, wu, wd, dy = inputs(rows, d, f, o, "bf16", seed=8)
    ws, n = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    runs = [[torch.empty_like(t) for t in (x, wg, wu, wd)] for _ in range(2)]
    backward(ngp, b, x, wg, wu, wd, dy, runs[0][0], runs[0][1:], ws, n)
    bad = rows // 2
    dy[bad, 1] = float("nan")
    backward(ngp, b, x, wg, wu, wd, dy, runs[1][0], runs[1][1:], ws, n)
    torch.cuda.synchronize()
    keep = torch.arange(rows, device="cuda") != bad
    assert torch.isnan(runs[1][0][bad]).all() and torch.equal(runs[0][0][keep], runs[1][0][keep])
    assert torch.isnan(runs[1][1]).all() and torch.isnan(runs[1][2]).all()
    other = torch.arange(o, device="cuda") != 1
    assert torch.isnan(runs[1][3][1]).all() and torch.equal(runs[0][3][other], runs[1][3][other])   # dw_down: the row of that output alone


def test_the_most_rows(ngp, cuda):
    """2^30 rows: positions, tiles and row offsets of the narrow kernels at their largest.  y and dx against 64 bits on rows from all over; the gradients against the sums in 64 bits, to the roundings
    of partial sums in fp32 (2^30 terms of one sign would be lost in one accumulator: here they have both, and 512 workgroups' waves have their own)"""
    rows, d, f, o = 1 << 30, 2, 3, 1
    x = torch.empty(rows, d, dtype=torch.float16, device="cuda")
    dy = torch.empty(rows, o, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    part = 1 << 26
    for i in range(0, rows, part):
        x[i:i + part] = torch.randn(part, d, generator=g, device="cuda", dtype=torch.float32)
        dy[i:i + part] = torch.randn(part, o, generator=g, device="cuda", dtype=torch.float32) * 0.5
    wg, wu, wd = (torch.randn(s, generator=g, device="cuda").half() for s in ((f, d), (f, d), (o, f)))
    b = block(d, f, o, "f16", "relu")
    y, dx = torch.empty(rows, o, dtype=torch.float16, device="cuda"), torch.empty_like(x)
    grads = [torch.empty_like(w) for w in (wg, wu, wd)]
    ws, n = workspace(ngp, b, rows, 0)
    forward(ngp, b, x, wg, wu, wd, y, ws, n)
    ws2, n2 = workspace(ngp, b, rows, capi.FFN_BACKWARD)
    backward(ngp, b, x, wg, wu, wd, dy, dx, grads, ws2, n2)
    torch.cuda.synchronize()
    for at in (0, rows // 2 - 1000, rows - 3001, rows - 1000):
        ref = R.Block("relu", x[at:at + 1000], wg, wu, wd, dy[at:at + 1000])
        R.check("y", y[at:at + 1000], ref.y, ref.ey)
        R.check("dx", dx[at:at + 1000], ref.dx, ref.edx)
    sums, magnitudes = [torch.zeros_like(w, dtype=torch.float64) for w in grads], [torch.zeros_like(w, dtype=torch.float64) for w in grads]
    part = 1 << 24   # sums of elementwise products: the library's product of such a shape, three by two over 2^26, takes two seconds
    for i in range(0, rows, part):
        xs, ys = x[i:i + part].double(), dy[i:i + part].double()
        gg, u = (sum(xs[:, j:j + 1] * w[:, j].double() for j in range(d)) for w in (wg, wu))
        on = (gg > 0).double()
        dh = ys * wd.double()
        for k, (p, q) in enumerate(((dh * u * on, xs), (dh * gg * on, xs), (ys, gg * on * u))):
            for c in range(q.shape[1]):
                t = p * q[:, c:c + 1]
                sums[k][:, c] += t.sum(0)
                magnitudes[k][:, c] += t.abs().sum(0)
    for v, want, size in zip(grads, sums, magnitudes):
        # every term is rounded once or twice to f16 and enters sums of up to 2^21 rows in one accumulator (2^30 / 512 workgroups): the roundings' signs are as random as the terms',
        # so sqrt(terms) of 2^-11 of a term, and sqrt(2^21) 2^-24 of a partial sum, which is itself of the order of sqrt(2^21) terms; 8 standard deviations, and the result's own rounding
        term = size / rows
        limit = 8 * (2.0 ** 15 * 2 * 2.0 ** -11 * term * 2 + 512 ** 0.5 * 2.0 ** 10.5 * 2.0 ** -24 * 2.0 ** 10.5 * term * 2) + 2.0 ** -11 * want.abs() + 2.0 ** -25
        assert (torch.isinf(v.double()) & (want.abs() > 60000)).logical_or((v.double() - want).abs() <= limit).all(), (v, want, limit)
