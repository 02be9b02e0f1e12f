"""The gated feed-forward block and its gradients in float64, from the definition."""

from __future__ import annotations

import math

import torch


def activation(a, act: str):
    """``(act(a), act'(a))``."""
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-a / math.sqrt(2.0))
        return a * phi, phi + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    sig = torch.special.expit(a)
    return (a * sig, sig + a * sig * (1 - sig)) if act == "silu" else (sig, sig * (1 - sig))


def feed(x, wg, wu, bg, bu, act: str, gy=None):
    """``y``, and with ``gy`` also the gradients ``[dx, dwg, dwu, dbg, dbu]`` and, for error bounds, what each is a sum of
    the magnitudes of. x ``[rows, D]``; biases may be None (their gradients are formed all the same)."""
    x, wg, wu = (t.detach().double() for t in (x, wg, wu))
    a, b = x @ wg.T, x @ wu.T
    if bg is not None:
        a = a + bg.detach().double()
    if bu is not None:
        b = b + bu.detach().double()
    f, df = activation(a, act)
    if gy is None:
        return f * b
    gy = gy.detach().double()
    da, db = gy * b * df, gy * f
    grads = [da @ wg + db @ wu, da.T @ x, db.T @ x, da.sum(0), db.sum(0)]
    sums = [da.abs() @ wg.abs() + db.abs() @ wu.abs(), da.abs().T @ x.abs(), db.abs().T @ x.abs(), da.abs().sum(0), db.abs().sum(0)]
    return f * b, grads, sums
