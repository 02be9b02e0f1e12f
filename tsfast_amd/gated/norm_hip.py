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
    """``t`` as rows of ``D`` dense columns: a tensor that keeps them alive, their address and row stride."""
    if t is None:
        return None, None, 0
    if t.is_contiguous():
        return t, t.data_ptr(), D
    t = t.reshape(-1, D)
    if t.stride(1) != 1 and D > 1:
        t = t.contiguous()
    return t, t.data_ptr(), t.stride(0)


def _param(t):
    return None if t is None else t.float().contiguous()


def _screen(x, likes, params, residual=None):
    """What a raw-pointer kernel relies on: x's type and device, ``likes`` of both, float32 dense ``params``."""
    dtype, dev = x.dtype, x.get_device()
    if dev < 0 or dtype not in _IO_DTYPES:
        raise TypeError(f"x: {dtype} on {x.device}, expected float32 or bfloat16 on a GPU")
    for t in likes:
        if t is not None and (t.dtype != dtype or t.get_device() != dev):
            raise TypeError(f"{t.dtype} on {t.device}, expected {dtype} on {x.device}")
    if residual is not None and (residual.dtype not in (dtype, torch.float32) or residual.get_device() != dev):
        raise TypeError(f"residual: {residual.dtype} on {residual.device}, expected {dtype} or float32 on {x.device}")
    for t in params:
        if t is not None and (t.dtype != torch.float32 or t.get_device() != dev or not t.is_contiguous()):
            raise TypeError(f"a parameter is {t.dtype} on {t.device}, expected dense float32 on {x.device}")


def _empty(t):
    if t.is_contiguous():
        return torch.empty_like(t)  # the cheaper call
    return torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _ptr(t):
    return None if t is None else t.data_ptr()


@custom_op("tsfast_hip::gated_norm")
def _gated_op(
    x: torch.Tensor, gate: torch.Tensor | None, weight: torch.Tensor | None, groups: int, eps: float, gate_first: bool
) -> torch.Tensor:
    lib = _lib.load()
    _screen(x, (gate,), (weight,))
    D = x.shape[-1]
    y = _empty(x)
    (_x, px, sx), (_g, pg, sg) = _rows(x, D), _rows(gate, D)
    _lib.check(
        lib.tsfast_hip_gated_norm_fwd(
            x.numel() // D, groups, D // groups, _IO_DTYPES[x.dtype], gate_first, eps, px, sx, pg, sg, _ptr(weight), y.data_ptr(),
            _lib.stream_of(x),
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
    _screen(x, (gate, gy), (weight,))
    D = x.shape[-1]
    rows = x.numel() // D
    gx = _empty(x)
    ggate = None if gate is None else _empty(gate)
    gw = None if weight is None else torch.empty_like(weight)
    (_x, px, sx), (_g, pg, sg), (_d, pd, sd) = _rows(x, D), _rows(gate, D), _rows(gy, D)
    nbytes = lib.tsfast_hip_gated_norm_workspace_bytes(rows, groups, D // groups) if weight is not None else 0
    ws = _lib.workspace(nbytes, x.device) if nbytes > 0 else None
    _lib.check(
        lib.tsfast_hip_gated_norm_bwd(
            rows, groups, D // groups, _IO_DTYPES[x.dtype], gate_first, eps, px, sx, pg, sg, _ptr(weight), pd, sd, gx.data_ptr(),
            _ptr(ggate), _ptr(gw), _ptr(ws), nbytes, _lib.stream_of(x),
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
    _screen(x, (), (weight, post_weight, scale), residual)
    D = x.shape[-1]
    new, y = _empty(residual), _empty(x)
    (_x, px, sx), (_r, pr, sr) = _rows(x, D), _rows(residual, D)
    _lib.check(
        lib.tsfast_hip_residual_norm_fwd(
            x.numel() // D, D, _IO_DTYPES[x.dtype], _IO_DTYPES[residual.dtype], eps, px, sx, pr, sr, _ptr(post_weight), _ptr(scale),
            _ptr(weight), new.data_ptr(), y.data_ptr(), _lib.stream_of(x),
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
    _screen(x, (gy,), (weight, post_weight, scale), residual)
    if gnew is not None and (gnew.dtype != residual.dtype or gnew.device != x.device):
        raise TypeError(f"gnew: {gnew.dtype} on {gnew.device}, expected {residual.dtype} on {x.device}")
    D = x.shape[-1]
    rows = x.numel() // D
    gx, gres = _empty(x), _empty(residual)
    params = (post_weight, scale, weight)
    gparams = [None if t is None else torch.empty_like(t) for t in params]
    (_x, px, sx), (_r, pr, sr), (_n, pn, sn), (_d, pd, sd) = _rows(x, D), _rows(residual, D), _rows(gnew, D), _rows(gy, D)
    nbytes = lib.tsfast_hip_residual_norm_workspace_bytes(rows, D)
    ws = _lib.workspace(nbytes, x.device)
    _lib.check(
        lib.tsfast_hip_residual_norm_bwd(
            rows, D, _IO_DTYPES[x.dtype], _IO_DTYPES[residual.dtype], eps, px, sx, pr, sr, *map(_ptr, params), pn, sn, pd, sd,
            gx.data_ptr(), gres.data_ptr(), *map(_ptr, gparams), _ptr(ws), nbytes, _lib.stream_of(x),
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
