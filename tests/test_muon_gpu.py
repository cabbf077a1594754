"""ngp_hip_muon_step on the GPU against 64-bit values (tests/muon_reference.py: the bounds and where they come from)."""
import numpy as np
import pytest
import torch

import capi
import muon_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": (torch.float16, 0), "bf16": (torch.bfloat16, 1), "f32": (torch.float32, 2)}
SENTINEL = 77.0


class Vector:
    """Parameter vectors that hold matrices of the given shapes with `gap` other parameters in front of each and behind the last"""

    def __init__(self, shapes, dtype, gap=3, seed=0, scale=1.0):
        self.shapes, self.t, self.code = shapes, *TYPES[dtype]
        self.desc = np.zeros(len(shapes), capi.MUON_MATRIX)
        at = gap
        for d, (r, c) in zip(self.desc, shapes):
            d["offset"], d["rows"], d["cols"] = at, r, c
            at += r * c + gap
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.size = at
        self.grads = (torch.randn(at, generator=gen, device="cuda") * scale).to(self.t)
        self.buf = torch.randn(at, generator=gen, device="cuda") * 0.5 * scale
        self.master = torch.randn(at, generator=gen, device="cuda") * 0.1
        self.params = torch.full((at,), SENTINEL, dtype=self.t, device="cuda") if dtype != "f32" else None

    def of(self, v, i):
        r, c = self.shapes[i]
        at = int(self.desc["offset"][i])
        return v[at:at + r * c].view(r, c)

    def inside(self):
        m = torch.zeros(self.size, dtype=torch.bool, device="cuda")
        for i in range(len(self.shapes)):
            self.of(m, i).fill_(True)
        return m

    def workspace(self, ngp):
        n = ngp.ngp_hip_muon_workspace_bytes(len(self.desc), self.desc.ctypes.data)
        return torch.full((n + 256,), 0xff, dtype=torch.uint8, device="cuda"), n

    def step(self, ngp, ws, n, lr=0.02, beta=0.95, decay=0.0, eps=1e-7, nesterov=1, iterations=5, loss_scale=1.0, params=True):
        capi.check(ngp.ngp_hip_muon_step(torch.cuda.current_stream().cuda_stream, len(self.desc), self.desc.ctypes.data, lr, beta, decay, eps, nesterov, iterations, loss_scale, self.code,
                                         self.grads.data_ptr(), self.master.data_ptr(), self.params.data_ptr() if params and self.params is not None else None, self.buf.data_ptr(),
                                         ws.data_ptr(), n))


def check_step(ngp, v, **kw):
    """One step, all of it against 64 bits.  lr 1, master 0 and no decay in `kw` leave the orthogonalised update itself in master."""
    a = dict(lr=0.02, beta=0.95, decay=0.01, eps=1e-7, nesterov=1, iterations=5, loss_scale=1.0)
    a.update(kw)
    before = [t.clone() for t in (v.grads, v.buf, v.master)]
    kept = None if v.params is None else v.params.clone()
    ws, n = v.workspace(ngp)
    v.step(ngp, ws, n, **a)
    torch.cuda.synchronize()
    assert (ws[n:] == 0xff).all() and torch.equal(v.grads, before[0])
    outside = ~v.inside()
    assert torch.equal(v.buf[outside], before[1][outside]) and torch.equal(v.master[outside], before[2][outside])
    assert kept is None or torch.equal(v.params[outside], kept[outside])
    for i, (rows, cols) in enumerate(v.shapes):
        g, b, w = (v.of(t, i) for t in before)
        m, master, x, u = R.step(g, w, b, a["lr"], a["beta"], a["decay"], a["eps"], a["nesterov"], a["iterations"], a["loss_scale"])
        # three roundings: the scaled gradient (1 / loss_scale and the product), the product, the sum
        limit = 4 * 2.0 ** -24 * (a["beta"] * b.double().abs() + g.double().abs() / a["loss_scale"]) + 1e-44
        assert ((v.of(v.buf, i).double() - m).abs() <= limit).all(), "momentum of matrix %d" % i
        rate = a["lr"] * max(1.0, rows / cols) ** 0.5
        far = R.bound(u, a["eps"], a["iterations"], x)
        off = v.of(v.master, i).double() - master
        spread = 3 * 2.0 ** -24 * master.norm().item() + 3 * 2.0 ** -24 * w.double().norm().item()
        assert off.norm().item() <= rate * far + spread, "matrix %d (%d x %d): off by %.3g, may be %.3g" % (i, rows, cols, off.norm().item(), rate * far + spread)
        # no entry carries more than all of it; and none more than 16 times its share beyond its own roundings
        share = 16 * (rate * far + spread) / (rows * cols) ** 0.5
        assert rows * cols < 64 or off.abs().max().item() <= share + 4 * 2.0 ** -24 * (master.abs().max().item() + w.abs().max().item())
        if v.params is not None:
            assert torch.equal(v.of(v.params, i), v.of(v.master, i).to(v.t))


SHAPES = [(1, 1), (1, 7), (5, 1), (3, 2), (16, 64), (64, 32), (64, 64), (33, 65), (63, 200), (64, 256), (256, 17), (257, 30), (65, 64), (128, 128), (100, 300), (300, 100), (129, 257), (130, 1000), (1000, 127), (768, 520), (520, 2050), (30, 5000), (1640, 24), (64, 8192), (8191, 64), (63, 8193), (65536, 70), (3, 65536), (513, 1), (2, 300)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_update_against_64_bits(ngp, cuda, shape):
    for dtype, nesterov in (("f16", 1), ("f32", 0)):
        v = Vector([shape], dtype, seed=shape[0])
        v.master.zero_()
        check_step(ngp, v, lr=1.0, decay=0.0, nesterov=nesterov)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_the_whole_step_on_matrices_of_many_shapes(ngp, cuda, dtype, nesterov):
    check_step(ngp, Vector([(64, 32), (16, 64), (64, 32), (64, 64), (16, 64), (200, 136), (1, 9), (129, 128)], dtype, seed=nesterov), nesterov=nesterov, loss_scale=128.0, decay=0.1)


@pytest.mark.parametrize("shapes", [[(500 - i, 530 + 3 * i) for i in range(22)], [(390 - i, 520 + i) for i in range(14)], [(640 - i, 650 + 3 * i) for i in range(20)], [(1130 + 5 * i, 1100 - i) for i in range(14)] + [(64, 2100), (700, 90)]], ids=["eight waves and 128x128", "64x64 and eight waves", "128x128 and 128x256", "eight waves twice"])
def test_larger_tiles(ngp, cuda, shapes):
    """enough matrices at once for each of the tiles of the symmetric products and of X B"""
    check_step(ngp, Vector(shapes, "bf16", gap=1), iterations=5)


@pytest.mark.parametrize("shapes", [[(65, 8200)], [(5000, 96)], [(100, 512), (66, 513), (300, 1111), (130, 131)], [(40, 3000), (64, 300), (5000, 17), (33, 257), (60, 60)] * 4, [(40, 2000), (64, 300), (150, 200)] * 15, [(40, 3000), (64, 300)] * 12], ids=["wide", "tall", "several", "slabs", "two batches of slabs", "too many slabs"])
def test_sums_over_a_long_side_in_parts(ngp, cuda, shapes):
    for dtype in ("f16", "f32"):
        v = Vector(shapes, dtype, seed=5)
        v.master.zero_()
        check_step(ngp, v, lr=1.0, decay=0.0)


def test_more_matrices_than_one_launch_takes(ngp, cuda):
    check_step(ngp, Vector([(8 + 3 * i, 90 - i) for i in range(60)], "bf16", gap=1), iterations=5)
    check_step(ngp, Vector([(70 + i, 150 - i) for i in range(30)], "f16", gap=0), iterations=3)
    check_step(ngp, Vector([(2 + i % 5, 3 + i % 7) if i % 3 else (66, 70) for i in range(160)], "f32", gap=2), iterations=2)


@pytest.mark.parametrize("iterations", [1, 2, 3, 6])
@pytest.mark.parametrize("shape", [(48, 64), (200, 72), (140, 300)], ids=lambda s: "%dx%d" % s)
def test_iterations(ngp, cuda, shape, iterations):
    v = Vector([shape], "f32", seed=iterations)
    v.master.zero_()
    check_step(ngp, v, lr=1.0, decay=0.0, iterations=iterations)


@pytest.mark.parametrize("shape", [(48, 64), (260, 140)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1.0, 1e30])
def test_magnitudes_of_single_precision(ngp, cuda, shape, scale):
    """squares beyond and below what fp32 holds; eps counts where the update is of its size"""
    v = Vector([shape], "f32", seed=2, scale=scale)
    v.master.zero_()
    check_step(ngp, v, lr=1.0, decay=0.0, eps=0.0 if scale == 1e-30 else 1e-7)


@pytest.mark.parametrize("shape", [(64, 64), (150, 200)], ids=lambda s: "%dx%d" % s)
def test_low_rank_and_spread_spectra(ngp, cuda, shape):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for power in (0.0, 1.0, 3.0):   # singular values i^-power; power 0: rank 3
        r, c = shape
        p, q = (torch.linalg.qr(torch.randn(s, s, generator=gen, device="cuda", dtype=torch.float64))[0] for s in shape)
        n = min(shape)
        s = torch.arange(1, n + 1, device="cuda", dtype=torch.float64) ** -power if power else (torch.arange(n, device="cuda") < 3).double()
        v = Vector([shape], "f32")
        v.buf.zero_()
        v.master.zero_()
        v.of(v.grads, 0).copy_((p[:, :n] * s) @ q[:, :n].T)
        check_step(ngp, v, lr=1.0, decay=0.0, nesterov=0)


def test_zero_update(ngp, cuda):
    for shape in ((40, 64), (140, 150)):
        v = Vector([shape], "f16")
        v.grads.zero_()
        v.buf.zero_()
        before = v.master.clone()
        ws, n = v.workspace(ngp)
        v.step(ngp, ws, n, decay=0.0)
        torch.cuda.synchronize()
        assert torch.equal(v.master, before) and (v.of(v.buf, 0) == 0).all()
        v.step(ngp, ws, n, decay=0.0, eps=0.0)   # 0 / 0 is that zero too
        torch.cuda.synchronize()
        assert torch.equal(v.master, before)


def test_a_gradient_that_is_not_finite_stays_in_its_matrix(ngp, cuda):
    shapes = [(40, 64), (64, 64), (150, 140), (64, 200)]
    for bad, value in ((1, float("nan")), (2, float("inf"))):
        v, w = Vector(shapes, "f16", seed=1), Vector(shapes, "f16", seed=1)
        v.of(v.grads, bad)[3, 4] = value
        for t in (v, w):
            ws, n = t.workspace(ngp)
            t.step(ngp, ws, n)
        torch.cuda.synchronize()
        assert not torch.isfinite(v.of(v.master, bad)).any()
        for i in range(len(shapes)):
            if i != bad:
                assert torch.equal(v.of(v.master, i), w.of(w.master, i))


def test_same_bits_on_another_stream_in_a_graph_and_beside_other_matrices(ngp, cuda):
    shapes = [(64, 32), (64, 64), (200, 136), (300, 513)]
    runs = [Vector(shapes, "bf16", seed=6) for _ in range(3)]
    ws, n = runs[0].workspace(ngp)
    runs[0].step(ngp, ws, n)
    with torch.cuda.stream(torch.cuda.Stream()):
        ws1, _ = runs[1].workspace(ngp)
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        runs[1].step(ngp, ws1, n)
    torch.cuda.synchronize()
    ws2, _ = runs[2].workspace(ngp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        runs[2].step(ngp, ws2, n)
    graph.replay()
    torch.cuda.synchronize()
    for other in runs[1:]:
        assert torch.equal(runs[0].master, other.master) and torch.equal(runs[0].buf, other.buf) and torch.equal(runs[0].params, other.params)
    for k in range(3):
        g = torch.randn(runs[0].size, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(torch.bfloat16)
        runs[0].grads.copy_(g)
        runs[2].grads.copy_(g)
        graph.replay()
        runs[0].step(ngp, ws, n)
        torch.cuda.synchronize()
        assert torch.equal(runs[0].master, runs[2].master) and torch.equal(runs[0].buf, runs[2].buf) and torch.equal(runs[0].params, runs[2].params)


def test_without_params(ngp, cuda):
    v, w = Vector([(48, 64), (130, 140)], "f16", seed=8), Vector([(48, 64), (130, 140)], "f16", seed=8)
    ws, n = v.workspace(ngp)
    v.step(ngp, ws, n)
    w.step(ngp, ws, n, params=False)
    torch.cuda.synchronize()
    assert torch.equal(v.master, w.master) and (w.params == SENTINEL).all()


def test_offsets_that_pass_32_bits(ngp, cuda):
    """two matrices whose elements lie behind 2^31 bytes and 2^32 elements of the vectors' start"""
    desc = np.zeros(2, capi.MUON_MATRIX)
    desc["offset"], desc["rows"], desc["cols"] = [(1 << 31) + 5, (1 << 32) + 7], [48, 140], [64, 136]
    size = (1 << 32) + 7 + 140 * 136
    small = Vector([(48, 64), (140, 136)], "f16", seed=3)
    far = [torch.empty(size, dtype=t.dtype, device="cuda") for t in (small.grads, small.master, small.params, small.buf)]
    for i in range(2):
        at, n = int(desc["offset"][i]), int(desc["rows"][i]) * int(desc["cols"][i])
        for big, t in zip(far, (small.grads, small.master, small.params, small.buf)):
            big[at:at + n].copy_(small.of(t, i).reshape(-1))
    ws, n = small.workspace(ngp)
    small.step(ngp, ws, n)
    capi.check(ngp.ngp_hip_muon_step(torch.cuda.current_stream().cuda_stream, 2, desc.ctypes.data, 0.02, 0.95, 0.0, 1e-7, 1, 5, 1.0, 0, far[0].data_ptr(), far[1].data_ptr(), far[2].data_ptr(),
                                     far[3].data_ptr(), ws.data_ptr(), n))
    torch.cuda.synchronize()
    for i in range(2):
        at, k = int(desc["offset"][i]), int(desc["rows"][i]) * int(desc["cols"][i])
        for big, t in zip(far[1:], (small.master, small.params, small.buf)):
            assert torch.equal(big[at:at + k], small.of(t, i).reshape(-1))


def test_two_streams_at_once_and_graphs_that_share_a_workspace(ngp, cuda):
    shapes = [(64, 32), (40, 900), (200, 136), (300, 513)]
    runs = [Vector(shapes, "f16", seed=s) for s in (1, 2)]
    want = [Vector(shapes, "f16", seed=s) for s in (1, 2)]
    for v in want:
        ws, n = v.workspace(ngp)
        for _ in range(4):
            v.step(ngp, ws, n)
    torch.cuda.synchronize()
    spaces, streams = [v.workspace(ngp) for v in runs], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(2):
        for v, (ws, n), s in zip(runs, spaces, streams):
            with torch.cuda.stream(s):
                v.step(ngp, ws, n)
    torch.cuda.synchronize()
    graphs = []
    for v in runs:   # one workspace for both
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            v.step(ngp, *spaces[0])
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for v, w in zip(runs, want):
        assert torch.equal(v.master, w.master) and torch.equal(v.buf, w.buf) and torch.equal(v.params, w.params)


@pytest.mark.parametrize("count", [24, 25, 36, 37, 75])
def test_lists_around_what_one_launch_takes(ngp, cuda, count):
    """one batch, two and three; large matrices among small ones"""
    check_step(ngp, Vector([(600, 420) if i % 9 == 4 else (70 + i, 130 - i % 50) for i in range(count)], "bf16", gap=1), iterations=3)
    check_step(ngp, Vector([(390, 410)] * count, "f16", gap=0), iterations=2)


@pytest.mark.parametrize("iterations", [5, 8, 10])
@pytest.mark.parametrize("rank", [1, 3])
@pytest.mark.parametrize("shape", [(64, 64), (150, 200), (40, 900), (768, 768)], ids=lambda s: "%dx%d" % s)
def test_rounding_noise_in_directions_that_the_update_lacks(ngp, cuda, shape, rank, iterations):
    """The stated bound, 2^-20 3.4445^n of the norm of X: what is stored of an X is off by 2^-22 of it, an iteration multiplies that by 3.4445 where the singular value is zero, every iteration
    adds as much again (a factor of 1 / (1 - 1 / 3.4445) = 1.41 in all), X is at most 1.21 times its last norm in between: 1.7 units of 2^-22.  The rest of the four is for the sums in fp32."""
    gen = torch.Generator(device="cuda").manual_seed(rank)
    p, q = (torch.linalg.qr(torch.randn(s, rank, generator=gen, device="cuda", dtype=torch.float64))[0] for s in shape)
    v = Vector([shape], "f32")
    v.buf.zero_()
    v.master.zero_()
    v.of(v.grads, 0).copy_(p @ q.T)
    _, want, x, _ = R.step(v.of(v.grads, 0), v.of(v.master, 0), v.of(v.buf, 0), 1.0, 0.0, 0.0, 0.0, 0, iterations, 1.0)
    ws, n = v.workspace(ngp)
    v.step(ngp, ws, n, lr=1.0, beta=0.0, eps=0.0, nesterov=0, iterations=iterations)
    torch.cuda.synchronize()
    assert (v.of(v.master, 0).double() - want).norm().item() <= 2.0 ** -20 * 3.4445 ** iterations * want.norm().item()


SLABS = [(40, 900), (3000, 24), (64, 8192)]   # a short side up to 64: a launch to an iteration, its own code for the norm


@pytest.mark.parametrize("shape", SLABS, ids=lambda s: "%dx%d" % s)
def test_zero_update_in_slabs(ngp, cuda, shape):
    v = Vector([shape], "f16")
    v.grads.zero_()
    v.buf.zero_()
    before = v.master.clone()
    for eps in (1e-7, 0.0):
        ws, n = v.workspace(ngp)
        v.step(ngp, ws, n, decay=0.0, eps=eps)
        torch.cuda.synchronize()
        assert torch.equal(v.master, before) and (v.of(v.buf, 0) == 0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
def test_a_gradient_that_is_not_finite_stays_in_its_matrix_of_slabs(ngp, cuda, value):
    shapes = SLABS + [(40, 64), (150, 140)]
    for bad in range(len(shapes)):
        v, w = Vector(shapes, "f16", seed=1), Vector(shapes, "f16", seed=1)
        v.of(v.grads, bad)[-1, -1] = value
        for t in (v, w):
            ws, n = t.workspace(ngp)
            t.step(ngp, ws, n)
        torch.cuda.synchronize()
        assert not torch.isfinite(v.of(v.master, bad)).any()
        for i in range(len(shapes)):
            if i != bad:
                assert torch.equal(v.of(v.master, i), w.of(w.master, i))


@pytest.mark.parametrize("shape", SLABS, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1.0, 1e30])
def test_magnitudes_of_single_precision_in_slabs(ngp, cuda, shape, scale):
    v = Vector([shape], "f32", seed=2, scale=scale)
    v.master.zero_()
    check_step(ngp, v, lr=1.0, decay=0.0, eps=0.0 if scale == 1e-30 else 1e-7)


@pytest.mark.parametrize("shape", SLABS, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("power", [0.0, 1.0, 3.0])
def test_low_rank_and_spread_spectra_in_slabs(ngp, cuda, shape, power):
    """singular values i^-power; power 0: rank 3"""
    gen = torch.Generator(device="cuda").manual_seed(4)
    n = min(shape)
    p, q = (torch.linalg.qr(torch.randn(s, n, generator=gen, device="cuda", dtype=torch.float64))[0] for s in shape)
    s = torch.arange(1, n + 1, device="cuda", dtype=torch.float64) ** -power if power else (torch.arange(n, device="cuda") < 3).double()
    v = Vector([shape], "f32")
    v.buf.zero_()
    v.master.zero_()
    v.of(v.grads, 0).copy_((p * s) @ q.T)
    check_step(ngp, v, lr=1.0, decay=0.0, nesterov=0)


@pytest.mark.parametrize("shape", SLABS, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("iterations", [1, 2, 6])
def test_iterations_in_slabs(ngp, cuda, shape, iterations):
    v = Vector([shape], "f32", seed=iterations)
    v.master.zero_()
    check_step(ngp, v, lr=1.0, decay=0.0, iterations=iterations)


@pytest.mark.parametrize("shape", [(48, 64), (40, 900), (260, 140), (768, 768)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("below", [1e-3, 1e-6, 1e-9])
def test_updates_far_below_epsilon(ngp, cuda, shape, below):
    """X is then as small, and its entries are held to 2^-40: half a step of the smallest fp16 over 2^15, which the iterations multiply by 3.4445 each and, new in every one, sum to 1.41 of that"""
    v = Vector([shape], "f32", seed=9)
    v.buf.zero_()
    v.master.zero_()
    u = v.of(v.grads, 0)
    u.mul_(below * 1e-3 / u.norm())
    _, want, _, _ = R.step(u, v.of(v.master, 0), v.of(v.buf, 0), 1.0, 0.0, 0.0, 1e-3, 0, 5, 1.0)
    ws, n = v.workspace(ngp)
    v.step(ngp, ws, n, lr=1.0, beta=0.0, eps=1e-3, nesterov=0)
    torch.cuda.synchronize()
    rate, grown = max(1.0, shape[0] / shape[1]) ** 0.5, 3.4445 ** 5
    assert (v.of(v.master, 0).double() - want).norm().item() <= 1.41 * 2.0 ** -40 * (shape[0] * shape[1]) ** 0.5 * grown * rate + 2.0 ** -20 * want.norm().item()
