"""ngp_hip_gated_ffn_*: the refusals (no GPU call is made before the arguments are checked) and the workspace sizes."""
import numpy as np
import pytest

import capi

P = 1 << 20   # an address that nothing reads: every call below is refused on the host


def block(d=136, f=264, o=136, dtype=0, act=4):
    b = np.zeros(1, capi.GATED_FFN)
    b["n_in"], b["n_hidden"], b["n_out"], b["dtype"], b["activation"] = d, f, o, dtype, act
    return b


def fwd(ngp, b, **kw):
    a = dict(rows=500, x=P, xs=136, wg=P, wu=P, wd=P, y=P, ys=136, ws=P, n=1 << 40)
    a.update(kw)
    return ngp.ngp_hip_gated_ffn_forward(None, None if b is None else b.ctypes.data, a["rows"], a["x"], a["xs"], a["wg"], a["wu"], a["wd"], a["y"], a["ys"], a["ws"], a["n"])


def bwd(ngp, b, **kw):
    a = dict(rows=500, x=P, xs=136, wg=P, wu=P, wd=P, dy=P, dys=136, dx=P, dxs=136, g=P, u=P, d=P, ws=P, n=1 << 40)
    a.update(kw)
    return ngp.ngp_hip_gated_ffn_backward(None, None if b is None else b.ctypes.data, a["rows"], a["x"], a["xs"], a["wg"], a["wu"], a["wd"], a["dy"], a["dys"], a["dx"], a["dxs"], a["g"], a["u"],
                                          a["d"], a["ws"], a["n"])


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("bad,word", [(dict(d=0), b"widths"), (dict(f=0), b"widths"), (dict(o=0), b"widths"), (dict(f=(1 << 20) + 1), b"widths"), (dict(dtype=2), b"dtype"), (dict(dtype=-1), b"dtype"),
                                      (dict(act=3), b"activation"), (dict(act=6), b"activation")])
def test_blocks_that_are_refused(ngp, call, bad, word):
    assert call(ngp, block(**bad)) != 0 and word in ngp.ngp_hip_last_error()
    assert ngp.ngp_hip_gated_ffn_workspace_bytes(block(**bad).ctypes.data, 500, 0) == 0


@pytest.mark.parametrize("call,bad", [(c, k) for c, ks in ((fwd, ("x", "wg", "wu", "wd", "y", "ws")), (bwd, ("x", "wg", "wu", "wd", "dy", "ws"))) for k in ks])
def test_null_tensors(ngp, call, bad):
    assert call(ngp, block(), **{bad: None}) != 0 and b"null" in ngp.ngp_hip_last_error()


@pytest.mark.parametrize("call,kw,word", [
    (fwd, dict(xs=135), b"stride"), (fwd, dict(ys=135), b"stride"), (bwd, dict(xs=135), b"stride"), (bwd, dict(dys=135), b"stride"), (bwd, dict(dxs=135), b"stride"),
    (fwd, dict(x=P + 1), b"aligned"), (fwd, dict(y=P + 1), b"aligned"), (bwd, dict(dy=P + 1), b"aligned"), (bwd, dict(u=P + 1), b"aligned"), (fwd, dict(ws=P + 8), b"workspace"),
    (fwd, dict(rows=(1 << 30) + 1), b"rows"), (bwd, dict(rows=(1 << 30) + 1), b"rows"), (bwd, dict(g=None), b"together"), (bwd, dict(d=None), b"together"),
    (bwd, dict(dx=None, g=None, u=None, d=None), b"nothing")])
def test_arguments_that_are_refused(ngp, call, kw, word):
    assert call(ngp, block(), **kw) != 0 and word in ngp.ngp_hip_last_error(), ngp.ngp_hip_last_error()


@pytest.mark.parametrize("call,flags", [(fwd, 0), (bwd, 1)])
def test_workspace_one_byte_too_small(ngp, call, flags):
    b = block()
    n = ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, 500, flags)
    assert n > 0 and call(ngp, b, n=n - 1) != 0 and b"workspace" in ngp.ngp_hip_last_error()
    # a base that is no multiple of 16 bytes needs room for copies, and is told so
    assert ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, 500, flags | capi.FFN_ANY_LAYOUT) > n
    assert call(ngp, b, x=P + 2, n=n) != 0 and b"ANY_LAYOUT" in ngp.ngp_hip_last_error()


def test_workspace_of_a_narrow_block(ngp):
    """weights that fit into LDS: the forward pass needs none, the backward pass room for its sums whatever the rows' alignment"""
    b = block(32, 64, 16)
    assert ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, 5000, 0) == 0
    n = ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, 5000, 1)
    assert n > 0 and ngp.ngp_hip_gated_ffn_workspace_bytes(b.ctypes.data, 5000, 3) == n
    for bad in (dict(n=n - 1), dict(ws=None), dict(ws=P + 8)):
        assert bwd(ngp, b, rows=5000, xs=32, dxs=32, dys=16, **bad) != 0 and b"workspace" in ngp.ngp_hip_last_error()


def test_workspace_holds_fewer_rows(ngp):
    """the size never falls with the number of rows, across every change of kernel and tile"""
    for d, f, o in ((32, 64, 16), (64, 128, 64), (33, 65, 17), (1024, 2816, 1024), (4096, 10240, 4096), (8192, 1000, 64)):
        for flags in range(4):
            last = 0
            for rows in [*range(0, 300), *range(300, 20000, 371), 1 << 17, 1 << 18]:
                n = ngp.ngp_hip_gated_ffn_workspace_bytes(block(d, f, o).ctypes.data, rows, flags)
                assert n >= last, (d, f, o, flags, rows)
                last = n


def test_empty_batches_need_nothing(ngp):
    assert fwd(ngp, block(), rows=0, x=None, y=None, ws=None, n=0) == 0
    assert bwd(ngp, block(), rows=0, x=None, dy=None, g=None, u=None, d=None, ws=None, n=0) == 0
