"""The gated block in 64 bits, with a bound on how far an evaluation may be that accumulates in fp32 and rounds where include/ngp_hip.h says it does.

Every bound is the usual forward analysis: a sum of k products in fp32, in any order, is off by at most (k + 2) 2^-24 of the sum of their magnitudes; a rounding to the
tensors' type by half a step (u = eps / 2), or by half the smallest subnormal; act and act' by 64 x 2^-24 (the exponential's argument is below 45 in magnitude in these tests,
an argument rounded to 24 bits moves the exponential by 45 x 2^-24, and the division and the products add a handful)."""
import math

import torch

ACTS = {"none": 0, "relu": 1, "logistic": 2, "silu": 4, "gelu": 5}
E32 = 2.0 ** -24


def activation(kind, g):
    """act, act', sup |act'|, sup |act''|"""
    if kind == "none":
        return g, torch.ones_like(g), 1.0, 0.0
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double(), 1.0, 0.0
    s = torch.sigmoid(g)
    if kind == "logistic":
        return s, s * (1 - s), 0.25, 0.1
    if kind == "silu":
        return g * s, s * (1 + g * (1 - s)), 1.1, 0.5
    phi = torch.special.ndtr(g)
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 1.13, 0.8


class Block:
    def __init__(self, kind, x, wg, wu, wd, dy=None):
        t = x.dtype
        self.u, self.tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
        x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
        d, f = x.shape[1], wg.shape[0]
        gam = lambda k: (k + 2) * E32   # noqa: E731
        g, u = x @ wg.T, x @ wu.T
        eg, eu = gam(d) * (x.abs() @ wg.abs().T), gam(d) * (x.abs() @ wu.abs().T)
        a, s, a1, a2 = activation(kind, g)
        ea, es = a1 * eg + 64 * E32 * a.abs().clamp(max=1e30), a2 * eg + 64 * E32
        if kind == "relu":
            es = torch.where(g.abs() <= eg, 1.0, 0.0)   # which side of the kink
        if kind == "none":
            es = torch.zeros_like(g)
        h = a * u
        eh = self._rounded(h, ea * u.abs() + (a.abs() + ea) * eu + 2 * E32 * h.abs())
        self.y = h @ wd.T
        self.ey = self._rounded(self.y, (eh + gam(f) * (h.abs() + eh)) @ wd.abs().T)
        if dy is None:
            return
        dy = dy.double()
        rows, o = dy.shape
        dh = dy @ wd
        edh = gam(o) * (dy.abs() @ wd.abs())
        hi = dh.abs() + edh
        dg, du = dh * u * s, dh * a
        edg = self._rounded(dg, edh * (u * s).abs() + hi * (eu * (s.abs() + es) + u.abs() * es) + 4 * E32 * dg.abs())
        edu = self._rounded(du, edh * a.abs() + hi * ea + 2 * E32 * du.abs())
        self.dx = dg @ wg + du @ wu
        self.edx = self._rounded(self.dx, (edg + gam(2 * f) * (dg.abs() + edg)) @ wg.abs() + (edu + gam(2 * f) * (du.abs() + edu)) @ wu.abs())
        self.dwg, self.dwu, self.dwd = dg.T @ x, du.T @ x, dy.T @ h
        self.edwg = self._rounded(self.dwg, (edg + gam(rows) * (dg.abs() + edg)).T @ x.abs())
        self.edwu = self._rounded(self.dwu, (edu + gam(rows) * (du.abs() + edu)).T @ x.abs())
        self.edwd = self._rounded(self.dwd, dy.abs().T @ (eh + gam(rows) * (h.abs() + eh)))

    def _rounded(self, v, e):
        """bound of v, known to e, after a rounding to the tensors' type"""
        return e + self.u * (v.abs() + e) + self.tiny


def check(name, got, want, bound):
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert not (off > bound).any() and torch.isfinite(got).all(), "%s: off by up to %.3g of the bound" % (name, worst)
