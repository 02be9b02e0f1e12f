"""HIP backend of the gated feed-forward block (``csrc/feed.hip``).

``supports(x, weight_gate, weight_up, bias_gate, bias_up)`` / ``run(..., activation) -> y``, differentiable in
all tensors through the ``tsfast_hip::feed_forward`` / ``feed_forward_train`` / ``feed_forward_bwd`` custom ops.
A call that will be differentiated keeps both projections for the backward (``kept``: 32 bits of each value with
float32, 24 with bfloat16).

All tensors are float32 or bfloat16 alike, rows at any stride and alignment (a last dimension that is not dense
is copied). Products are formed on the bfloat16 matrix cores and summed in float32; float32 operands go in as three
bfloat16 parts each, six products, which keeps float32's accuracy and takes infinities and NaN where float32 products would.
"""

from __future__ import annotations

__all__ = ["supports", "run", "ACTIVATIONS"]

import torch

from .. import _lib
from ..ops import custom_op

_IO_DTYPES = {torch.float32: _lib.TSF_DTYPE_F32, torch.bfloat16: _lib.TSF_DTYPE_BF16}
ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}  # feed.hip Act
_MAX_WIDTH = 1 << 20  # D and F (feed.hip feed_status)
_MAX_LD = 1 << 22  # elements between rows (feed.hip kMaxLd)
_MAX_TILES = (1 << 24) - 1  # workgroups of 256 threads in a launch
_FEW_ROWS = {torch.float32: 64, torch.bfloat16: 32}  # read as they lie, without a workspace (feed.hip few_rows; tests pin it)


def supports(x, weight_gate, weight_up, bias_gate, bias_up) -> str | None:
    """Reason the fused block cannot handle these tensors, or None if it can."""
    dtype, dev = x.dtype, x.get_device()
    if dev < 0:
        return f"x on {x.device.type}, hip backend is GPU-only"
    if dtype not in _IO_DTYPES:
        return f"x dtype {dtype} not float32/bfloat16"
    for t in (weight_gate, weight_up, bias_gate, bias_up):
        if t is not None and (t.dtype != dtype or t.get_device() != dev):
            return f"a parameter is {t.dtype} on {t.device}, x {x.dtype} on {x.device}"
    F, D = weight_gate.shape
    if D > _MAX_WIDTH or F > _MAX_WIDTH:
        return f"widths D={D}, F={F} above {_MAX_WIDTH}"
    rows = x.numel() // D
    tiles = max(-(-rows // 64) * max(-(-F // 32), -(-D // 64)), 2 * -(-(-(-F // 8) * 16) // 256) * -(-D // 256))  # feed.hip feed_status
    if rows > (1 << 31) - 64 or tiles > _MAX_TILES:
        return f"{rows} rows of D={D}, F={F} need more workgroups than one launch has"
    return None


def _rows(t, width: int):
    """``t`` as rows of ``width`` dense columns that the kernels can step through: a tensor that keeps them alive, and the rows' distance."""
    if t.is_contiguous():
        return t, width
    t = t.reshape(-1, width)
    if t.shape[0] <= 1:
        return t.contiguous(), width
    if (width > 1 and t.stride(1) != 1) or not width <= t.stride(0) <= _MAX_LD:
        return t.contiguous(), width
    return t, t.stride(0)


def _screen(x, *others):
    dtype, dev = x.dtype, x.get_device()
    if dev < 0 or dtype not in _IO_DTYPES:
        raise TypeError(f"x: {dtype} on {x.device}, expected float32 or bfloat16 on a GPU")
    for t in others:
        if t is not None and (t.dtype != dtype or t.get_device() != dev):
            raise TypeError(f"{t.dtype} on {t.device}, expected {dtype} on {x.device}")


def _empty(t):
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _dense(t):
    return None if t is None else t.contiguous()


def kept_bytes(rows: int, F: int, dtype: torch.dtype) -> int:
    """Bytes that a training step's forward keeps (tests pin it against ``tsfast_hip_feed_kept_bytes``). Computed here,
    so that the fake implementation makes no library call while torch.compile traces it."""
    return -(-rows // 16) * -(-F // 16) * 64 * (24 if dtype == torch.bfloat16 else 32)


def _forward(x, weight_gate, weight_up, bias_gate, bias_up, activation: int, train: bool):
    lib = _lib.load()
    _screen(x, weight_gate, weight_up, bias_gate, bias_up)
    F, D = weight_gate.shape
    rows, io = x.numel() // D, _IO_DTYPES[x.dtype]
    (xr, sx), (wg, sg), (wu, su) = _rows(x, D), _rows(weight_gate, D), _rows(weight_up, D)
    bg, bu = _dense(bias_gate), _dense(bias_up)
    with _lib.device_of(x):
        y = torch.empty((*x.shape[:-1], F), device=x.device, dtype=x.dtype)
        kept = torch.empty(kept_bytes(rows, F, x.dtype), device=x.device, dtype=torch.uint8) if train else None
        where = (xr.data_ptr(), sx, wg.data_ptr(), sg, wu.data_ptr(), su)
        nbytes = lib.tsfast_hip_feed_fwd_workspace_bytes(rows, D, F, io, *where, train) if train or rows > _FEW_ROWS[x.dtype] else 0
        ws = _lib.workspace(nbytes, x.device) if nbytes > 0 else None
        _lib.check(
            lib.tsfast_hip_feed_fwd(
                rows, D, F, io, activation, *where, _lib.ptr(bg), _lib.ptr(bu), y.data_ptr(), _lib.ptr(kept), _lib.ptr(ws), nbytes,
                _lib.stream_of(x),
            ),
            "tsfast_hip_feed_fwd",
        )
    return y, kept


@custom_op("tsfast_hip::feed_forward")
def _feed_op(
    x: torch.Tensor,
    weight_gate: torch.Tensor,
    weight_up: torch.Tensor,
    bias_gate: torch.Tensor | None,
    bias_up: torch.Tensor | None,
    activation: int,
) -> torch.Tensor:
    return _forward(x, weight_gate, weight_up, bias_gate, bias_up, activation, train=False)[0]


@custom_op("tsfast_hip::feed_forward_train")
def _feed_train_op(
    x: torch.Tensor,
    weight_gate: torch.Tensor,
    weight_up: torch.Tensor,
    bias_gate: torch.Tensor | None,
    bias_up: torch.Tensor | None,
    activation: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    return _forward(x, weight_gate, weight_up, bias_gate, bias_up, activation, train=True)


def _out(x, weight_gate):
    return x.new_empty((*x.shape[:-1], weight_gate.shape[0]))


@_feed_op.register_fake
def _(x, weight_gate, weight_up, bias_gate, bias_up, activation):
    return _out(x, weight_gate)


@_feed_train_op.register_fake
def _(x, weight_gate, weight_up, bias_gate, bias_up, activation):
    F, D = weight_gate.shape
    return _out(x, weight_gate), x.new_empty(kept_bytes(x.numel() // D, F, x.dtype), dtype=torch.uint8)


@custom_op("tsfast_hip::feed_forward_bwd")
def _feed_bwd_op(
    gy: torch.Tensor,
    kept: torch.Tensor,
    x: torch.Tensor,
    weight_gate: torch.Tensor,
    weight_up: torch.Tensor,
    has_bias_gate: bool,
    has_bias_up: bool,
    activation: int,
    want_x: bool,
    want_weights: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(x, weight_gate, weight_up, gy)
    F, D = weight_gate.shape
    rows, io = x.numel() // D, _IO_DTYPES[x.dtype]
    if kept.dtype != torch.uint8 or kept.numel() != kept_bytes(rows, F, x.dtype) or kept.get_device() != x.get_device() or not kept.is_contiguous():
        raise TypeError(f"kept: {kept.numel()} of {kept.dtype} on {kept.device}, expected the forward's on {x.device}")
    (xr, sx), (wg, sg), (wu, su), (gr, sgy) = _rows(x, D), _rows(weight_gate, D), _rows(weight_up, D), _rows(gy, F)
    with _lib.device_of(x):
        gx = _empty(x) if want_x else x.new_empty(0)
        gwg, gwu = (_empty(w) if want_weights else x.new_empty(0) for w in (weight_gate, weight_up))
        gbg, gbu = (x.new_empty(F if want else 0) for want in (has_bias_gate, has_bias_up))
        where = (xr.data_ptr(), sx, wg.data_ptr(), sg, wu.data_ptr(), su)
        nbytes = lib.tsfast_hip_feed_bwd_workspace_bytes(rows, D, F, io, *where)
        ws = _lib.workspace(nbytes, x.device)
        _lib.check(
            lib.tsfast_hip_feed_bwd(
                rows, D, F, io, activation, *where, gr.data_ptr(), sgy, kept.data_ptr(),
                *(t.data_ptr() if t.numel() else None for t in (gx, gwg, gwu, gbg, gbu)), ws.data_ptr(), nbytes, _lib.stream_of(x),
            ),
            "tsfast_hip_feed_bwd",
        )
    return gx, gwg, gwu, gbg, gbu


@_feed_bwd_op.register_fake
def _(gy, kept, x, weight_gate, weight_up, has_bias_gate, has_bias_up, activation, want_x, want_weights):
    F, D = weight_gate.shape
    empty = lambda want, *shape: x.new_empty(shape if want else (0,))  # noqa: E731
    return empty(want_x, *x.shape), empty(want_weights, F, D), empty(want_weights, F, D), empty(has_bias_gate, F), empty(has_bias_up, F)


def _setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    x, weight_gate, weight_up, bias_gate, bias_up, ctx.activation = inputs
    ctx.bias = (bias_gate is not None, bias_up is not None)
    ctx.save_for_backward(x, weight_gate, weight_up, output[1])


def _backward(ctx, gy, gkept=None):
    need = ctx.needs_input_grad
    if gy is None or not any(need[:5]):
        return (None,) * 6
    x, weight_gate, weight_up, kept = ctx.saved_tensors
    want_bias = [has and n for has, n in zip(ctx.bias, need[3:5])]
    grads = _feed_bwd_op(gy, kept, x, weight_gate, weight_up, *want_bias, ctx.activation, need[0], need[1] or need[2])
    want = (need[0], need[1], need[2], *want_bias)
    return (*(g if w else None for g, w in zip(grads, want)), None)


_feed_train_op.register_autograd(_backward, setup_context=_setup)


def run(x, weight_gate, weight_up, bias_gate, bias_up, activation: str):
    """The fused block; see :func:`tsfast_amd.gated.gated_feed_forward`."""
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (
        x.requires_grad
        or weight_gate.requires_grad
        or weight_up.requires_grad
        or (bias_gate is not None and bias_gate.requires_grad)
        or (bias_up is not None and bias_up.requires_grad)
    ):
        return _feed_train_op(x, weight_gate, weight_up, bias_gate, bias_up, act)[0]
    return _feed_op(x, weight_gate, weight_up, bias_gate, bias_up, act)
