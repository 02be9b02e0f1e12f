"""HIP backend of the norms before and after a block (``csrc/norm.hip``).

``supports(x, other, params, width)`` answers for both operators (``other`` is the gate or the residual,
``width`` the columns normalised together); ``gated_norm`` and ``residual_norm`` run them, differentiable in
all tensors through the ``tsfast_hip::gated_norm`` / ``residual_norm`` custom ops and their ``_bwd``. Only the
inputs are saved for the backward.

x, gate and y are float32 or bfloat16 alike, the residual stream of that type or float32, rows at any stride
and alignment (a last dimension that is not dense is copied); parameters are float32 (bfloat16 ones are upcast
before the op, so autograd casts their gradients back). All arithmetic is float32, each output rounded once;
parameter gradients are sums in a fixed order.
"""

from __future__ import annotations

__all__ = ["supports", "gated_norm", "residual_norm"]

import torch

from .. import _lib
from ..ops import custom_op

_IO_DTYPES = {torch.float32: _lib.TSF_DTYPE_F32, torch.bfloat16: _lib.TSF_DTYPE_BF16}
_MAX_WIDTH = 8192  # columns normalised together (norm.hip kMaxWidth; tests pin it against the library)


def supports(x, other, params, width: int) -> str | None:
    """Reason the fused norms cannot handle these tensors, or None if they can."""
    if x.device.type != "cuda":
        return f"x on {x.device.type}, hip backend is GPU-only"
    if x.dtype not in _IO_DTYPES:
        return f"x dtype {x.dtype} not float32/bfloat16"
    for t in (other, *params):
        if t is not None and t.device != x.device:
            return f"a tensor on {t.device}, x on {x.device}"
    for t in params:
        if t is not None and t.dtype not in _IO_DTYPES:
            return f"parameters must be float32 or bfloat16, got {t.dtype}"
    if width > _MAX_WIDTH:
        return f"{width} columns normalised together, at most {_MAX_WIDTH}"
    if x.shape[-1] // width > 65535 or x.shape[-1] >= 1 << 31:
        return f"rows of {x.shape[-1]} columns"
    return None


def _rows(t, D: int):
    """``t`` as ``[rows, D]`` with dense columns, and its row stride."""
    if t is None:
        return None, 0
    t = t.reshape(-1, D)
    if t.stride(1) != 1 and D > 1:
        t = t.contiguous()
    return t, t.stride(0)


def _param(t):
    return None if t is None else t.float().contiguous()


def _screen(x, *others):
    if x.device.type != "cuda" or x.dtype not in _IO_DTYPES:
        raise TypeError(f"x: {x.dtype} on {x.device}, expected float32 or bfloat16 on a GPU")
    for name, t, dtypes in others:
        if t is not None and (t.dtype not in dtypes or t.device != x.device):
            raise TypeError(f"{name}: {t.dtype} on {t.device}, expected {dtypes} on {x.device}")


def _empty(t):
    return torch.empty(t.shape, device=t.device, dtype=t.dtype)


@custom_op("tsfast_hip::gated_norm")
def _gated_op(
    x: torch.Tensor, gate: torch.Tensor | None, weight: torch.Tensor | None, groups: int, eps: float, gate_first: bool
) -> torch.Tensor:
    lib = _lib.load()
    _screen(x, ("gate", gate, (x.dtype,)))
    _lib.require(weight, "weight", (torch.float32,), x.device)
    D = x.shape[-1]
    y = _empty(x)
    (x2, sx), (g2, sg) = _rows(x, D), _rows(gate, D)
    _lib.check(
        lib.tsfast_hip_gated_norm_fwd(
            x2.shape[0], groups, D // groups, _IO_DTYPES[x.dtype], gate_first, eps, _lib.ptr(x2), sx, _lib.ptr(g2), sg,
            _lib.ptr(weight), _lib.ptr(y), _lib.stream_of(x),
        ),
        "tsfast_hip_gated_norm_fwd",
    )
    return y


@_gated_op.register_fake
def _(x, gate, weight, groups, eps, gate_first):
    return _empty(x)


@custom_op("tsfast_hip::gated_norm_bwd")
def _gated_bwd_op(
    gy: torch.Tensor, x: torch.Tensor, gate: torch.Tensor | None, weight: torch.Tensor | None, groups: int, eps: float, gate_first: bool
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(x, ("gate", gate, (x.dtype,)), ("gy", gy, (x.dtype,)))
    _lib.require(weight, "weight", (torch.float32,), x.device)
    D = x.shape[-1]
    gx = _empty(x)
    ggate = None if gate is None else _empty(gate)
    gw = None if weight is None else _empty(weight)
    (x2, sx), (g2, sg), (d2, sd) = _rows(x, D), _rows(gate, D), _rows(gy, D)
    nbytes = lib.tsfast_hip_gated_norm_workspace_bytes(x2.shape[0], groups, D // groups) if weight is not None else 0
    ws = _lib.workspace(nbytes, x.device) if nbytes > 0 else None
    _lib.check(
        lib.tsfast_hip_gated_norm_bwd(
            x2.shape[0], groups, D // groups, _IO_DTYPES[x.dtype], gate_first, eps, _lib.ptr(x2), sx, _lib.ptr(g2), sg,
            _lib.ptr(weight), _lib.ptr(d2), sd, *map(_lib.ptr, (gx, ggate, gw, ws)), nbytes, _lib.stream_of(x),
        ),
        "tsfast_hip_gated_norm_bwd",
    )
    return gx, (x.new_empty(0) if ggate is None else ggate), (x.new_empty(0, dtype=torch.float32) if gw is None else gw)


@_gated_bwd_op.register_fake
def _(gy, x, gate, weight, groups, eps, gate_first):
    return (
        _empty(x),
        x.new_empty(0) if gate is None else _empty(gate),
        x.new_empty(0, dtype=torch.float32) if weight is None else _empty(weight),
    )


def _gated_setup(ctx, inputs, output):
    x, gate, weight, *ctx.how = inputs
    ctx.save_for_backward(x, gate, weight)


def _gated_backward(ctx, gy):
    x, gate, weight = ctx.saved_tensors
    gx, ggate, gw = _gated_bwd_op(gy, x, gate, weight, *ctx.how)
    return gx, (None if gate is None else ggate), (None if weight is None else gw), None, None, None


_gated_op.register_autograd(_gated_backward, setup_context=_gated_setup)


def gated_norm(x, gate, weight, groups: int, eps: float, gate_first: bool):
    """The fused gated norm; see :func:`tsfast_amd.gated.gated_norm`."""
    return _gated_op(x, gate, _param(weight), int(groups), float(eps), bool(gate_first))


@custom_op("tsfast_hip::residual_norm")
def _residual_op(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor | None,
    post_weight: torch.Tensor | None,
    scale: torch.Tensor | None,
    eps: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(x, ("residual", residual, (x.dtype, torch.float32)))
    for name, t in (("weight", weight), ("post_weight", post_weight), ("scale", scale)):
        _lib.require(t, name, (torch.float32,), x.device)
    D = x.shape[-1]
    new, y = _empty(residual), _empty(x)
    (x2, sx), (r2, sr) = _rows(x, D), _rows(residual, D)
    _lib.check(
        lib.tsfast_hip_residual_norm_fwd(
            x2.shape[0], D, _IO_DTYPES[x.dtype], _IO_DTYPES[residual.dtype], eps, _lib.ptr(x2), sx, _lib.ptr(r2), sr,
            *map(_lib.ptr, (post_weight, scale, weight, new, y)), _lib.stream_of(x),
        ),
        "tsfast_hip_residual_norm_fwd",
    )
    return new, y


@_residual_op.register_fake
def _(x, residual, weight, post_weight, scale, eps):
    return _empty(residual), _empty(x)


@custom_op("tsfast_hip::residual_norm_bwd")
def _residual_bwd_op(
    gnew: torch.Tensor | None,
    gy: torch.Tensor | None,
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor | None,
    post_weight: torch.Tensor | None,
    scale: torch.Tensor | None,
    eps: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(x, ("residual", residual, (x.dtype, torch.float32)), ("gnew", gnew, (residual.dtype,)), ("gy", gy, (x.dtype,)))
    for name, t in (("weight", weight), ("post_weight", post_weight), ("scale", scale)):
        _lib.require(t, name, (torch.float32,), x.device)
    D = x.shape[-1]
    gx, gres = _empty(x), _empty(residual)
    params = (post_weight, scale, weight)
    gparams = [None if t is None else _empty(t) for t in params]
    (x2, sx), (r2, sr), (n2, sn), (d2, sd) = _rows(x, D), _rows(residual, D), _rows(gnew, D), _rows(gy, D)
    nbytes = lib.tsfast_hip_residual_norm_workspace_bytes(x2.shape[0], D)
    ws = _lib.workspace(nbytes, x.device)
    _lib.check(
        lib.tsfast_hip_residual_norm_bwd(
            x2.shape[0], D, _IO_DTYPES[x.dtype], _IO_DTYPES[residual.dtype], eps, _lib.ptr(x2), sx, _lib.ptr(r2), sr,
            *map(_lib.ptr, params), _lib.ptr(n2), sn, _lib.ptr(d2), sd, *map(_lib.ptr, (gx, gres, *gparams, ws)), nbytes,
            _lib.stream_of(x),
        ),
        "tsfast_hip_residual_norm_bwd",
    )
    gpost, gscale, gw = (x.new_empty(0, dtype=torch.float32) if t is None else t for t in gparams)
    return gx, gres, gw, gpost, gscale


@_residual_bwd_op.register_fake
def _(gnew, gy, x, residual, weight, post_weight, scale, eps):
    params = (x.new_empty(0, dtype=torch.float32) if t is None else _empty(t) for t in (weight, post_weight, scale))
    return (_empty(x), _empty(residual), *params)


def _residual_setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    *tensors, ctx.eps = inputs
    ctx.save_for_backward(*tensors)


def _residual_backward(ctx, gnew, gy):
    x, residual, *params = ctx.saved_tensors
    gx, gres, *gparams = _residual_bwd_op(gnew, gy, x, residual, *params, ctx.eps)
    return (gx, gres, *(None if p is None else t for p, t in zip(params, gparams)), None)


_residual_op.register_autograd(_residual_backward, setup_context=_residual_setup)


def residual_norm(x, residual, weight, post_weight, scale, eps: float):
    """The fused residual norm; see :func:`tsfast_amd.gated.residual_norm`."""
    return _residual_op(x, residual, _param(weight), _param(post_weight), _param(scale), float(eps))
