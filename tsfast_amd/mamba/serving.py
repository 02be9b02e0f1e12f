"""A Mamba layer in service: prompts of different lengths packed into one row of tokens, and single tokens.

A layer runs ``in_proj -> conv -> x_proj, dt_proj -> scan -> out_proj``. ``mamba_conv`` and ``mamba_ssm`` run the conv and the scan
of rows of equal length, in training. Here the conv and the scan take a packed row and give the states that its sequences
leave, and ``mamba_step`` goes on from them, all of the layer between ``in_proj`` and ``out_proj`` at once::

    u, conv_state = mamba_conv_packed(x, starts, conv_weight, conv_bias)
    dt, B_t, C_t = (u @ x_proj.T).split([R, N, N], -1)
    y, ssm_state = mamba_ssm_packed(dt @ dt_proj.T + dt_bias, A, B_t, C_t, u, z, Dp, starts)
    ...
    y = mamba_step(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp)

Sequence ``s`` of a packed row has the tokens ``starts[s] .. starts[s + 1)``. The reference has no packed rows and steps a layer by
running it on one token (``tsfast/models/architectures/mamba/core.py:175-213``). Dispatch is this package's: the
``"hip"`` family for GPU tensors, torch code for what it declines, sequence by sequence.
"""

from __future__ import annotations

__all__ = ["mamba_conv_packed", "mamba_ssm_packed", "mamba_step"]

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from ..dispatch import resolve
from ..ops import has_tangent
from . import core, packed_hip


class _ConvDispatch:
    """The convolution's part of ``packed_hip``, in the protocol ``resolve`` asks."""

    supports = staticmethod(packed_hip.supports_conv)
    run = staticmethod(packed_hip.conv)


class _SsmDispatch:
    supports = staticmethod(packed_hip.supports_ssm)
    run = staticmethod(packed_hip.ssm)


class _StepDispatch:
    supports = staticmethod(packed_hip.supports_step)
    run = staticmethod(packed_hip.step)


_CONV_BACKENDS, _SSM_BACKENDS, _STEP_BACKENDS = {"hip": _ConvDispatch}, {"hip": _SsmDispatch}, {"hip": _StepDispatch}
_AUTO_ORDER = {"cuda": ("hip",)}


def _no_gradient(what: str, instead: str, *tensors):
    if forward_ad._current_level >= 0 and has_tangent(tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it without tangents, or use {instead}")
    if not torch.is_grad_enabled():
        return
    wanted = False
    for t in tensors:
        wanted = wanted or (t is not None and t.requires_grad)
    if wanted:
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or use {instead}")


def _check_starts(starts):
    if starts.dim() != 1 or starts.shape[0] < 1 or starts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"starts must be [S + 1] of int32 or int64, got {tuple(starts.shape)} of {starts.dtype}")
    return starts.shape[0] - 1


def _check(t, name: str, shape: tuple, dtype=None, optional: bool = False):
    if t is None and optional:
        return
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _bounds(starts, T: int):
    """The sequences' bounds on the host, checked."""
    at = starts.tolist()
    if at[0] < 0 or at[-1] > T or any(a > b for a, b in zip(at[:-1], at[1:])):
        raise ValueError(f"starts must not decrease and lie in [0, {T}], got {at[:8]}..{at[-1]}")
    return list(zip(at[:-1], at[1:]))


def _check_conv_weight(weight, bias, D: int) -> int:
    if weight.dim() != 3 or weight.shape[0] != D or weight.shape[1] != 1 or weight.shape[2] < 2:
        raise ValueError(f"the conv's weight must be [{D}, 1, K] with K of 2 or more, got {tuple(weight.shape)}")
    _check(bias, "the conv's bias", (D,), optional=True)
    return weight.shape[-1]


def mamba_conv_packed(x, starts, weight, bias=None, tails=None):
    """``silu`` of a causal depthwise convolution over packed sequences.

    Args:
        x: ``[T, D]``, any distance between rows. starts: ``[S + 1]`` int32 or int64 on x's device, not decreasing, within ``[0, T]``;
            a sequence may be empty.
        weight: ``[D, 1, K]``; bias: ``[D]`` or None.
        tails: the inputs before each sequence, ``[S, D, K - 1]`` of x's type, or None (zero).

    Returns:
        ``(u [T, D], the sequences' last K - 1 inputs [S, D, K - 1])``, in x's type; zeros where a token belongs to no sequence.
        Without a gradient. On the GPU starts is not checked (that would wait for the device): where it decreases, results are undefined.
    """
    _no_gradient("mamba_conv_packed", "mamba_conv", x, weight, bias, tails)
    if x.dim() != 2:
        raise ValueError(f"x must be [T, D], got {tuple(x.shape)}")
    S, (T, D) = _check_starts(starts), x.shape
    K = _check_conv_weight(weight, bias, D)
    _check(tails, "tails", (S, D, K - 1), x.dtype, optional=True)
    mod = resolve("mamba.conv_packed", _CONV_BACKENDS, _AUTO_ORDER.get(x.device.type, ()), (x, starts, weight, bias, tails))
    if mod is not None:
        return mod.run(x, starts, weight, bias, tails)
    u, left = x.new_zeros(T, D), x.new_zeros(S, D, K - 1) if tails is None else tails.clone()
    wide = x.dtype if x.dtype == torch.float64 else torch.float32
    for s, (t0, t1) in enumerate(_bounds(starts, T)):
        if t1 > t0:
            row = torch.cat((left[s], x[t0:t1].T), 1)
            pre = F.conv1d(row[None].to(wide), weight.to(wide), None if bias is None else bias.to(wide), groups=D)[0].T
            u[t0:t1] = F.silu(pre).to(x.dtype)
            left[s] = row[:, row.shape[1] - (K - 1) :]
    return u, left


def mamba_ssm_packed(draw, A, B_t, C_t, u, z, Dp, starts, h0=None):
    """The scan section of a Mamba layer (:func:`mamba_ssm`) over packed sequences.

    Args:
        draw, u, z: ``[T, D]``; B_t, C_t: ``[T, N]``; all of one type, any distance between rows. A: ``[D, N]``, Dp: ``[D]``, float32.
        starts: ``[S + 1]`` int32 or int64, as in :func:`mamba_conv_packed`. h0: states before each sequence, ``[S, D, N]`` float32, or None (zero).

    Returns:
        ``(out [T, D], the states that the sequences leave [S, D, N] float32)``, without a gradient; zeros where a token belongs to no
        sequence. Rows may be cut into segments by T and D: a sequence's results agree with those it has alone to float32 rounding.
    """
    _no_gradient("mamba_ssm_packed", "mamba_ssm", draw, A, B_t, C_t, u, z, Dp, h0)
    if draw.dim() != 2 or A.dim() != 2 or A.shape[1] < 1:
        raise ValueError(f"draw must be [T, D] and A [D, N], got {tuple(draw.shape)} and {tuple(A.shape)}")
    S, (T, D), N = _check_starts(starts), draw.shape, A.shape[1]
    wide = torch.float64 if draw.dtype == torch.float64 else torch.float32
    for t, name, shape, dtype in ((A, "A", (D, N), wide), (Dp, "Dp", (D,), wide), (u, "u", (T, D), draw.dtype), (z, "z", (T, D), draw.dtype),
                                  (B_t, "B_t", (T, N), draw.dtype), (C_t, "C_t", (T, N), draw.dtype)):
        _check(t, name, shape, dtype)
    _check(h0, "h0", (S, D, N), wide, optional=True)
    mod = resolve("mamba.ssm_packed", _SSM_BACKENDS, _AUTO_ORDER.get(draw.device.type, ()), (draw, A, B_t, C_t, u, z, Dp, starts, h0))
    if mod is not None:
        return mod.run(draw, A, B_t, C_t, u, z, Dp, starts, h0)
    out = draw.new_zeros(T, D)
    last = draw.new_zeros(S, D, N, dtype=wide) if h0 is None else h0.clone()
    for s, (t0, t1) in enumerate(_bounds(starts, T)):
        if t1 > t0:
            row = [t[None, t0:t1].to(wide) for t in (draw, B_t, C_t, u, z)]
            y, h = core._sliced_ssm(row[0], A, row[1], row[2], row[3], row[4], Dp, last[s : s + 1], per_step=False)
            out[t0:t1], last[s] = y[0].to(draw.dtype), h.view(D, N)
    return out, last


def mamba_step(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp):
    """One token of each sequence through a Mamba layer between its input and output projections, the states updated in place.

    ``u = silu(conv(conv_state, x))``, ``(dt, B, C) = x_proj u``, ``delta = softplus(dt_proj dt + dt_bias)``,
    ``h = exp(delta A) h + delta u B``, ``out = (h C + Dp u) silu(z)``; all of it in float32, rounded once.

    Args:
        x, z: ``[B, D]`` of one type (the halves of in_proj's output, any distance between rows).
        conv_state: the last K - 1 inputs ``[B, D, K - 1]`` of x's type, and ssm_state: ``[B, D, N]`` float32; overwritten.
        conv_weight: ``[D, 1, K]``; conv_bias: ``[D]`` or None; x_proj: ``[R + 2 N, D]``; dt_proj: ``[D, R]``; dt_bias: ``[D]`` or None; float32
            or bfloat16 each, or x's type. A: ``[D, N]``, Dp: ``[D]``, float32.

    Returns:
        ``out [B, D]`` in x's type. For prediction: the step has no gradient, and asking for one is an error. The channels whose products with
        x_proj are summed together depend on B and D: a sequence alone and in a batch agree to float32 rounding.
    """
    _no_gradient("mamba_step", "mamba_conv and mamba_ssm", x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp)
    if x.dim() != 2 or A.dim() != 2 or A.shape[1] < 1:
        raise ValueError(f"x must be [B, D] and A [D, N], got {tuple(x.shape)} and {tuple(A.shape)}")
    (B, D), N = x.shape, A.shape[1]
    K = _check_conv_weight(conv_weight, conv_bias, D)
    if dt_proj.dim() != 2 or dt_proj.shape[0] != D or dt_proj.shape[1] < 1:
        raise ValueError(f"dt_proj must be [{D}, R], got {tuple(dt_proj.shape)}")
    R, wide = dt_proj.shape[1], torch.float64 if x.dtype == torch.float64 else torch.float32
    rows, channels, state = (B, D), (D,), (B, D, N)
    if (
        z.shape != rows or conv_state.shape != (B, D, K - 1) or ssm_state.shape != state or x_proj.shape != (R + 2 * N, D) or Dp.shape != channels
        or A.shape[0] != D or z.dtype != x.dtype or conv_state.dtype != x.dtype or ssm_state.dtype != wide or A.dtype != wide or Dp.dtype != wide
    ):  # all of it at once; by name what it is
        for t, name, shape, dtype in ((z, "z", rows, x.dtype), (conv_state, "conv_state", (B, D, K - 1), x.dtype), (A, "A", (D, N), wide),
                                      (ssm_state, "ssm_state", state, wide), (x_proj, "x_proj", (R + 2 * N, D), None), (Dp, "Dp", channels, wide)):
            _check(t, name, shape, dtype)
    _check(dt_bias, "dt_bias", channels, optional=True)
    args = (x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp)
    for t in (conv_weight, conv_bias, x_proj, dt_proj, dt_bias):
        if t is not None and t.dtype not in (x.dtype, torch.float32, torch.bfloat16):
            raise ValueError(f"parameters must be float32, bfloat16 or {x.dtype}, got {t.dtype}")
    mod = resolve("mamba.step", _STEP_BACKENDS, _AUTO_ORDER.get(x.device.type, ()), args)
    if mod is not None:
        return mod.run(*args)
    window = torch.cat((conv_state, x[..., None]), -1)
    u = (window.to(wide) * conv_weight[:, 0].to(wide)).sum(-1)
    u = F.silu(u if conv_bias is None else u + conv_bias.to(wide))
    dt, B_t, C_t = (u @ x_proj.to(wide).T).split([R, N, N], -1)
    draw = dt @ dt_proj.to(wide).T
    delta = F.softplus(draw if dt_bias is None else draw + dt_bias.to(wide))
    h = torch.exp(delta[..., None] * A) * ssm_state + (delta * u)[..., None] * B_t[:, None]
    conv_state.copy_(window[..., 1:])
    ssm_state.copy_(h)
    return (((h * C_t[:, None]).sum(-1) + Dp * u) * F.silu(z.to(wide))).to(x.dtype)
