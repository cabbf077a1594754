"""ngp_hip_muon_step: the refusals (arguments are checked before any GPU call) and the workspace size."""
import numpy as np
import pytest

import capi

P = 1 << 20


def matrices(*rows):
    d = np.zeros(len(rows), capi.MUON_MATRIX)
    for e, (o, r, c) in zip(d, rows):
        e["offset"], e["rows"], e["cols"] = o, r, c
    return d


GOOD = matrices((0, 64, 32), (2048, 160, 64), (12288, 80, 100))


def call(ngp, m=GOOD, count=None, **kw):
    a = dict(lr=0.02, beta=0.95, decay=0.0, eps=1e-7, nesterov=1, iterations=5, scale=128.0, dtype=0, g=P, w=P, p=P, b=P, ws=P, n=1 << 40)
    a.update(kw)
    return ngp.ngp_hip_muon_step(None, len(m) if count is None else count, m.ctypes.data if m is not None else None, a["lr"], a["beta"], a["decay"], a["eps"], a["nesterov"], a["iterations"], a["scale"],
                                 a["dtype"], a["g"], a["w"], a["p"], a["b"], a["ws"], a["n"])


@pytest.mark.parametrize("m,word", [(matrices((0, 0, 32)), b"rows and cols"), (matrices((0, 4, 0)), b"rows and cols"), (matrices((0, 65537, 2)), b"rows and cols"), (matrices((0, 2, 65537)), b"rows and cols"),
                                    (matrices((0, 64, 32), (2047, 16, 64)), b"overlap"), (matrices((0, 64, 32), (0, 64, 32)), b"overlap"), (matrices((4096, 64, 32), (0, 16, 64)), b"order"),
                                    (matrices(((1 << 48) + 1, 2, 2)), b"offset")])
def test_lists_that_are_refused(ngp, m, word):
    assert call(ngp, m) != 0 and word in ngp.ngp_hip_last_error(), ngp.ngp_hip_last_error()
    assert ngp.ngp_hip_muon_workspace_bytes(len(m), m.ctypes.data) == 0


@pytest.mark.parametrize("kw,word", [(dict(g=None), b"null"), (dict(w=None), b"null"), (dict(b=None), b"null"), (dict(ws=None), b"workspace"), (dict(ws=P + 4), b"workspace"), (dict(iterations=0), b"n_iterations"),
                                     (dict(iterations=33), b"n_iterations"), (dict(scale=0.0), b"loss_scale"), (dict(scale=-1.0), b"loss_scale"), (dict(scale=float("nan")), b"loss_scale"),
                                     (dict(eps=-1.0), b"epsilon"), (dict(eps=float("nan")), b"epsilon"), (dict(dtype=3), b"dtype"), (dict(dtype=2), b"params"), (dict(w=P + 2), b"aligned"), (dict(b=P + 1), b"aligned"),
                                     (dict(g=P + 1), b"aligned"), (dict(p=P + 1), b"aligned"), (dict(dtype=2, p=None, g=P + 2), b"aligned")])
def test_arguments_that_are_refused(ngp, kw, word):
    assert call(ngp, **kw) != 0 and word in ngp.ngp_hip_last_error(), ngp.ngp_hip_last_error()


def test_null_list_and_too_many(ngp):
    assert ngp.ngp_hip_muon_step(None, 1, None, 0.1, 0.9, 0.0, 1e-7, 1, 5, 1.0, 0, P, P, P, P, P, 1 << 40) != 0 and b"no matrices" in ngp.ngp_hip_last_error()
    assert call(ngp, count=65537) != 0 and b"65536" in ngp.ngp_hip_last_error()


def test_workspace(ngp):
    n = ngp.ngp_hip_muon_workspace_bytes(len(GOOD), GOOD.ctypes.data)
    assert n > 0 and call(ngp, n=n - 1) != 0 and b"workspace" in ngp.ngp_hip_last_error()


def test_small_matrices_need_no_workspace(ngp):
    m = matrices((0, 64, 32), (2048, 16, 64), (4096, 256, 64), (1 << 20, 1, 256))
    assert ngp.ngp_hip_muon_workspace_bytes(len(m), m.ctypes.data) == 0
    for big in ((1, 257), (257, 1), (65, 65)):
        m = matrices((0, *big))
        assert ngp.ngp_hip_muon_workspace_bytes(1, m.ctypes.data) > 0


def test_no_matrices_is_no_work(ngp):
    assert call(ngp, count=0, g=None, w=None, p=None, b=None, ws=None, n=0) == 0


def listed(*shapes):
    at, rows = 0, []
    for r, c in shapes:
        rows.append((at, r, c))
        at += r * c
    return matrices(*rows)


def test_the_choice_of_slabs_does_not_depend_on_the_order_of_the_list(ngp):
    """seventeen of 16 slabs and three of 32 are more than one round of the chip either way round"""
    short, long = [(16, 2048)] * 17, [(64, 8192)] * 3
    size = [ngp.ngp_hip_muon_workspace_bytes(len(m), m.ctypes.data) for m in (listed(*short, *long), listed(*long, *short), listed(*short[:9], *long, *short[9:]))]
    assert size[0] == size[1] == size[2] > 0


def test_a_batch_is_as_many_small_matrices_as_the_arguments_of_a_launch_hold(ngp):
    """the workspace is that of the largest batch: matrices of one size take the same each"""
    def size(*shapes):
        m = listed(*shapes)
        return ngp.ngp_hip_muon_workspace_bytes(len(m), m.ctypes.data)

    one = size((200, 300))
    for together in (2, 24, 25, 32, 36):
        assert size(*[(200, 300)] * together) == together * one
    for count in (37, 60, 200):
        assert one * 18 <= size(*[(200, 300)] * count) <= one * 36
