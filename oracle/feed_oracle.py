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


def reach(x, wg, wu, bg, bu, act: str, gy):
    """What a relative error of every sum's terms is relative to in the end, for ``y`` and ``[dx, dwg, dwu, dbg, dbu]``: a and b are off by that
    part of A = |x| |Wg| + |bg| and B = |x| |Wu| + |bu| (not of a and b, which may have cancelled), so act(a) b by that of B |f| + A |f'| |b|, da =
    gy b f' by that of |gy| (B |f'| + |b| A |f''|) and db = gy f by that of |gy| (|f| + A |f'|); |f''| <= 1 (0.8 at most, gelu's at 0)."""
    x, wg, wu, gy = (t.detach().double() for t in (x, wg, wu, gy))
    zero = x.new_zeros(())
    bg, bu = (zero if t is None else t.detach().double() for t in (bg, bu))
    a, b = x @ wg.T + bg, x @ wu.T + bu
    A, B = x.abs() @ wg.abs().T + bg.abs(), x.abs() @ wu.abs().T + bu.abs()
    f, df = (t.abs() for t in activation(a, act))
    ra, rb = gy.abs() * (B * df + b.abs() * A + b.abs() * df), gy.abs() * (f + A * df)
    return B * f + A * df * b.abs() + f * b.abs(), [ra @ wg.abs() + rb @ wu.abs(), ra.T @ x.abs(), rb.T @ x.abs(), ra.sum(0), rb.sum(0)]
