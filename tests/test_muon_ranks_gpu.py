"""optimizer.otype "Muon" under data parallelism: several ranks on the one GPU, the gradients all-reduced, the whole step on every rank (an update needs its whole matrix)."""
import os
import sys
import time

import numpy as np
import pytest
import torch

import muon_reference as M
from test_dp_loopback_gpu import ROOT, run_ranks

pytestmark = pytest.mark.gpu
WORKER = os.path.join(ROOT, "tests", "loopback", "muon_worker.py")
SHAPES, RATE = [(64, 32), (16, 64), (64, 32), (64, 64), (16, 64)], 1e-2   # configs/nerf/muon.json


@pytest.mark.timeout(600)
@pytest.mark.parametrize("world", [2, 3])
def test_one_model_on_every_rank_and_the_update_of_the_summed_gradients(cuda, world, tmp_path):
    out = str(tmp_path)
    run_ranks([[sys.executable, WORKER, str(r), str(world), "mu_%d_%d" % (os.getpid(), int(time.time() * 1000) % 1000000), out] for r in range(world)], out, timeout=300)
    ranks = [np.load(os.path.join(out, "rank%d.npz" % r)) for r in range(world)]
    for r in ranks[1:]:
        for name in r.files:
            if name != "loss_after":   # each on its own again
                np.testing.assert_array_equal(r[name], ranks[0][name])
    r = ranks[0]
    assert r["stale"].tolist() == [False, False] and np.isfinite(r["loss"]) and all(np.isfinite(q["loss_after"]) for q in ranks)
    half = lambda name: torch.from_numpy(r[name].view(np.float16).astype(np.float64)).cuda()   # noqa: E731
    momentum = torch.zeros(sum(a * b for a, b in SHAPES), dtype=torch.float64, device="cuda")
    for step in (1, 2, 3):   # three steps by the formula, from the gradients that every rank holds behind the all-reduce
        before, after, g = half("params_%d" % (step - 1)), half("params_%d" % step), half("gradients_%d" % step) / 128
        assert g[:len(momentum)].abs().sum() > 0
        momentum = 0.95 * momentum + g[:len(momentum)]
        at = 0
        for rows, cols in SHAPES:
            p0, p1, u = (t[at:at + rows * cols].view(rows, cols) for t in (before, after, g[:len(momentum)] + 0.95 * momentum))
            at += rows * cols
            rate = RATE * max(1.0, rows / cols) ** 0.5
            off = (p0 - p1 - rate * M.orthogonalise(u, 1e-7, 5)).abs()
            # both weights are the master's rounded to fp16: half a step each; X is within 2^-20 3.4445^5 of its norm, at most 1.21 a direction, whatever the gradient's singular values
            limit = 2.0 ** -11 * (p0.abs() + p1.abs()) + 2.0 ** -24 + rate * 2.0 ** -20 * 3.4445 ** 5 * 1.21 * min(rows, cols) ** 0.5
            assert (off <= limit).all(), "step %d, %d x %d: off by up to %.3g of what it may" % (step, rows, cols, (off / limit).max().item())
    snaps = [open(os.path.join(out, "rank%d.msgpack" % k), "rb").read() for k in range(world)]
    assert all(s == snaps[0] for s in snaps[1:])
    import pyngp
    tb = pyngp.Testbed(pyngp.TestbedMode.Nerf)
    tb.load_snapshot(os.path.join(out, "rank%d.msgpack" % (world - 1)))
    np.testing.assert_array_equal(tb.debug_params("training"), r["params"])
    np.testing.assert_array_equal(tb.debug_params("inference"), r["inference"])
