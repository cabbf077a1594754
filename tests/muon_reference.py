"""The Muon step in 64 bits, and how far an evaluation may be that keeps its matrices to 22 bits and sums in fp32.

The bound is the error model run as numbers: the 64-bit iteration once more with every stored matrix (X, A, B) moved by what its representation and its sums may do to it, a few
times with other signs, and 4 times the largest deviation seen (the deviations of one size scatter by a few per cent: they are sums over all entries).  The model, per entry:
storage in two fp16 halves 2^-22 of the entry (half a step of the low half is 2^-12 of a low half that is at most 2^-11 of the value, and lo lo is dropped: 2^-22); a sum of k
products in fp32: the roundings of the partial sums have no common sign, sqrt(k) 2^-24 of the root mean square of the sums, and 2^-24 of the entry."""
import numpy as np
import torch

A, B, C = 3.4445, -4.7750, 2.0315


def moved(v, k, gen):
    if gen is None:
        return v
    z = torch.randn(v.shape, generator=gen, dtype=torch.float64, device=v.device)
    w = torch.randn(v.shape, generator=gen, dtype=torch.float64, device=v.device)
    return v + v * z * 2.0 ** -22 + w * v.square().mean().sqrt() * (k ** 0.5 + 1) * 2.0 ** -24


def orthogonalise(u, eps, iterations, gen=None):
    x = u / (u.norm() + eps)
    turn = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if turn else x
    n, k = x.shape
    x = moved(x, 0, gen)
    eye = torch.eye(n, dtype=torch.float64, device=x.device)
    for _ in range(iterations):
        a = moved(x @ x.T, k, gen)
        b = moved(A * eye + B * a + C * (a @ a), n, gen)
        x = moved(b @ x, n, gen)
    return x.T if turn else x


def bound(u, eps, iterations, exact):
    """the largest deviation of the model over four runs, in the Frobenius norm, times 4; at least two roundings to fp32"""
    far = 0.0
    for seed in range(4):
        gen = torch.Generator(device=u.device).manual_seed(seed)
        far = max(far, (orthogonalise(u, eps, iterations, gen) - exact).norm().item())
    return 4 * far + 2.0 ** -23 * exact.norm().item()


def step(g, master, buf, lr, beta, decay, eps, nesterov, iterations, loss_scale):
    """in 64 bits: momentum, master, X, u"""
    g, master, buf = g.double() / loss_scale, master.double(), buf.double()
    m = beta * buf + g
    u = g + beta * m if nesterov else m
    x = orthogonalise(u, eps, iterations)
    rows, cols = g.shape
    return m, (1 - lr * decay) * master - lr * max(1.0, rows / cols) ** 0.5 * x, x, u
