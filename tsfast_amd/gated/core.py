"""The operators of a gated recurrent block, with fused-kernel dispatch.

Such a block runs ``norm -> projections -> gated_recurrence -> gated_norm -> projection`` beside a
residual stream that ``residual_norm`` continues into the next block::

    o, state = gated_recurrence(q, k, v, g, state)        # or gated_recurrence_step, token by token
    y = gated_norm(o.flatten(-2), gate, weight, groups=H) @ W_out
    stream, x = residual_norm(y, stream, next_weight, post_weight=.., scale=..)

The recurrence is linear with a matrix state per head and one decay per head and step,

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,    o_t = S_t^T q_t,

so one state holds K x V numbers for K + V projected ones. Nothing in the reference corresponds to these
operators (its selective scan keeps a vector per channel); they follow this package's other
dispatch points: ``dispatch.resolve`` picks the ``"hip"`` family for GPU tensors, and torch code
serves what it declines (CPU tensors, float64, wider heads), in float32 at least.
"""

from __future__ import annotations

__all__ = ["gated_recurrence", "gated_recurrence_step", "gated_norm", "residual_norm"]

import torch
import torch.nn.functional as F

from ..dispatch import resolve
from . import norm_hip, recurrence_hip

# Module objects, not import paths: this dispatch may run inside a compiled forward.
_RECURRENCE_BACKENDS = {"hip": recurrence_hip}
_NORM_BACKENDS = {"hip": norm_hip}
_AUTO_ORDER = {"cuda": ("hip",)}

_CHUNK = 64  # steps whose products the torch path forms at once


def _check_shapes(q, k, v, g, state, lead: str):
    """Shapes of a call whose leading dimensions (one or two) are ``lead``."""
    qs, vs = q.shape, v.shape
    n = 2 if lead == "B, L" else 1
    if len(vs) != n + 2:
        raise ValueError(f"v must be [{lead}, H, V], got {tuple(vs)}")
    if len(qs) != n + 2 or qs[:n] != vs[:n] or qs != k.shape:
        raise ValueError(f"q and k must be alike, [{lead}, Hk, K] for v {tuple(vs)}; got {tuple(qs)} and {tuple(k.shape)}")
    H, Hk = vs[n], qs[n]
    if Hk < 1 or H < 1 or H % Hk != 0:
        raise ValueError(f"{H} heads of v do not share {Hk} heads of q and k evenly")
    if g.shape != vs[:-1]:
        raise ValueError(f"g must be [{lead}, H] = {tuple(vs[:-1])}, got {tuple(g.shape)}")
    if state is not None and state.shape != (vs[0], H, qs[-1], vs[-1]):
        raise ValueError(f"state must be [B, H, K, V] = {(vs[0], H, qs[-1], vs[-1])}, got {tuple(state.shape)}")


def _wide(t):
    """``t`` in the torch path's arithmetic: float32, or float64 where it is given."""
    return t if t.dtype == torch.float64 else t.float()


def _share(t, heads: int):
    return t if t.shape[-2] == heads else t.repeat_interleave(heads // t.shape[-2], dim=-2)


def _chunked_recurrence(q, k, v, g, state):
    B, L, H, V = v.shape
    dtype = v.dtype
    q, k, v, g = (_wide(t) for t in (_share(q, H), _share(k, H), v, g))
    S = v.new_zeros(B, H, q.shape[-1], V) if state is None else state.to(v.dtype)
    outs = []
    for t0 in range(0, L, _CHUNK):
        qc, kc, vc = (t[:, t0 : t0 + _CHUNK].transpose(1, 2) for t in (q, k, v))  # [B, H, C, width]
        gc = g[:, t0 : t0 + _CHUNK].transpose(1, 2)
        at = torch.arange(gc.shape[-1], device=g.device)
        # sums over the steps after j up to i: sums and no differences, so that -inf stays -inf
        spans = torch.where(at[:, None] > at, gc[..., :, None], 0.0).cumsum(-2)
        decay = spans.masked_fill(at[:, None] < at, float("-inf")).exp()
        o = (qc @ kc.transpose(-1, -2) * decay) @ vc + (qc * gc.cumsum(-1).exp()[..., None]) @ S
        S = gc.sum(-1).exp()[..., None, None] * S + (kc * decay[..., -1, :, None]).transpose(-1, -2) @ vc
        outs.append(o.transpose(1, 2))
    o = torch.cat(outs, 1) if outs else v.new_zeros(B, 0, H, V)
    return o.to(dtype), S


def gated_recurrence(q, k, v, g, state=None):
    """A linear recurrence with a matrix state per head: ``S_t = exp(g_t) S_{t-1} + k_t v_t^T``,
    ``o_t = S_t^T q_t``.

    Args:
        q, k: ``[B, L, Hk, K]``; v: ``[B, L, H, V]`` with ``H`` a multiple of ``Hk``: head ``h`` reads head
            ``h // (H // Hk)`` of q and k. A scale of the scores belongs into q.
        g: log decays ``[B, L, H]``, usually at most 0. ``-inf`` (any value whose exp is zero) forgets the
            state, as where another sequence begins in a packed row; a padded step has ``g = 0``, ``k = 0``.
        state: ``[B, H, K, V]`` before the first step, or None (zero).

    Returns:
        ``(o [B, L, H, V], last state [B, H, K, V])``, differentiable in all inputs. The state is float32
        (float64 for float64 inputs) whatever the others' type.

    All of q, k, v must be finite: the fused kernel works in chunks of 64 steps, and a value that is not may
    reach every step of its chunk and, with the state, the chunks after it (in gradients before it), whatever g is.
    """
    _check_shapes(q, k, v, g, state, "B, L")
    mod = resolve("gated.recurrence", _RECURRENCE_BACKENDS, _AUTO_ORDER.get(v.device.type, ()), (q, k, v, g, state))
    if mod is not None:
        return mod.run(q, k, v, g, state)
    return _chunked_recurrence(q, k, v, g, state)


class _StepDispatch:
    """The step's half of ``recurrence_hip``, in the protocol ``resolve`` asks."""

    supports = staticmethod(recurrence_hip.supports_step)
    run = staticmethod(recurrence_hip.step)


_STEP_BACKENDS = {"hip": _StepDispatch}


def gated_recurrence_step(q, k, v, g, state):
    """One step of :func:`gated_recurrence` with the state updated in place.

    Args:
        q, k: ``[B, Hk, K]``; v: ``[B, H, V]``; g: ``[B, H]``; state: ``[B, H, K, V]`` float32, overwritten.

    Returns:
        ``o [B, H, V]``. For prediction: the step has no gradient, and asking for one is an error.
    """
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or state.requires_grad):
        raise RuntimeError("gated_recurrence_step has no gradient: call it under torch.no_grad(), or use gated_recurrence")
    _check_shapes(q, k, v, g, state, "B")
    mod = resolve("gated.recurrence_step", _STEP_BACKENDS, _AUTO_ORDER.get(v.device.type, ()), (q, k, v, g, state))
    if mod is not None:
        return mod.run(q, k, v, g, state)
    H = v.shape[-2]
    qw, kw, vw, gw = (t.to(state.dtype) for t in (_share(q, H), _share(k, H), v, g))
    state.copy_(gw.exp()[..., None, None] * state + kw[..., None] * vw[..., None, :])
    return (qw[..., None, :] @ state)[..., 0, :].to(v.dtype)


def _rms(x, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def _check_param(t, name, D):
    if t is not None and tuple(t.shape) != (D,):
        raise ValueError(f"{name} must be [{D}], got {tuple(t.shape)}")


def gated_norm(x, gate, weight, groups: int = 1, eps: float = 1e-5, gate_first: bool = False):
    """RMS norm of ``x`` with a SiLU gate: ``rms(x) * weight * silu(gate)``, or with ``gate_first``
    ``rms(x * silu(gate)) * weight``; ``rms(x) = x / sqrt(mean(x^2) + eps)``.

    Args:
        x: ``[..., D]``; gate: like x, or None (no gate); weight: ``[D]`` or None (ones).
        groups: parts of ``D`` that are normalised apart (one per head, say).

    Returns:
        ``[..., D]`` in x's type, differentiable in x, gate and weight.
    """
    D = x.shape[-1] if x.dim() else 0
    if D < 1 or groups < 1 or D % groups != 0:
        raise ValueError(f"x must be [..., D] with D a multiple of groups={groups}, got {tuple(x.shape)}")
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError(f"gate must be like x, {tuple(x.shape)} of {x.dtype}; got {tuple(gate.shape)} of {gate.dtype}")
    _check_param(weight, "weight", D)
    mod = resolve("gated.norm", _NORM_BACKENDS, _AUTO_ORDER.get(x.device.type, ()), (x, gate, (weight,), D // groups))
    if mod is not None:
        return mod.gated_norm(x, gate, weight, groups, eps, gate_first)
    y = _wide(x)
    act = None if gate is None else F.silu(_wide(gate))
    if act is not None and gate_first:
        y = y * act
    y = _rms(y.unflatten(-1, (groups, D // groups)), eps).flatten(-2)
    if weight is not None:
        y = y * weight
    if act is not None and not gate_first:
        y = y * act
    return y.to(x.dtype)


def residual_norm(x, residual, weight, post_weight=None, scale=None, eps: float = 1e-5):
    """What stands between two blocks: the post-norm of a block's output, its residual scale, the residual
    sum and the next block's pre-norm. ``new = residual + scale * rms(x) * post_weight``,
    ``y = rms(new) * weight``.

    Args:
        x: the block's output ``[..., D]``; residual: the stream, ``[..., D]`` of x's type or float32.
        weight: the pre-norm's ``[D]``, or None (ones).
        post_weight: the post-norm's ``[D]``, or None: no post-norm, ``x`` is added as it is.
        scale: ``[D]`` or None (ones).

    Returns:
        ``(new stream in residual's type, y in x's type)``, differentiable in all inputs. ``y`` is the norm of
        the sum before its rounding to residual's type.
    """
    D = x.shape[-1] if x.dim() else 0
    if D < 1:
        raise ValueError(f"x must be [..., D], got {tuple(x.shape)}")
    if residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(
            f"residual must be {tuple(x.shape)} of {x.dtype} or float32; got {tuple(residual.shape)} of {residual.dtype}"
        )
    for t, name in ((weight, "weight"), (post_weight, "post_weight"), (scale, "scale")):
        _check_param(t, name, D)
    mod = resolve("gated.norm", _NORM_BACKENDS, _AUTO_ORDER.get(x.device.type, ()), (x, residual, (weight, post_weight, scale), D))
    if mod is not None:
        return mod.residual_norm(x, residual, weight, post_weight, scale, eps)
    b = _wide(x)
    if post_weight is not None:
        b = _rms(b, eps) * post_weight
    if scale is not None:
        b = b * scale
    new = _wide(residual) + b
    y = _rms(new, eps)
    if weight is not None:
        y = y * weight
    return new.to(residual.dtype), y.to(x.dtype)
