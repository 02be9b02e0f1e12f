"""HIP backend of the gated linear recurrence (``csrc/gated.hip``).

``supports(q, k, v, g, state)`` / ``run(...) -> (o, last)``, differentiable in all inputs through the
``tsfast_hip::gated_recurrence`` / ``gated_recurrence_bwd`` custom ops, and ``supports_step`` / ``step`` for
one token with the state updated in place (``tsfast_hip::gated_recurrence_step``). The inputs are saved for the
backward, and the states between the segments of cut rows (``gated_recurrence_train``).

q, k, v, g and their gradients are float32 or bfloat16, all alike, at any strides with a dense last
dimension (others are copied); states are float32. The kernels sum in float32 and keep the state in it. With
bfloat16 they multiply on the bfloat16 matrix cores: what is not bfloat16 already (the decayed scores, the state,
the decayed keys) goes in as a sum of two or three bfloat16 numbers, so outputs are rounded once.
"""

from __future__ import annotations

__all__ = ["supports", "run", "supports_step", "step"]

import ctypes

import torch

from .. import _lib
from ..ops import custom_op

_IO_DTYPES = {torch.float32: _lib.TSF_DTYPE_F32, torch.bfloat16: _lib.TSF_DTYPE_BF16}
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_MAX_WIDTH = 128
_STEP_MAX_K = 1024
_MAX_GRID = (1 << 24) - 1
_MAX_STEP = 1 << 23  # elements between the steps of a row


def _tensor_reason(q, k, v, g, state) -> str | None:
    dtype, dev = v.dtype, v.device
    if dev.type != "cuda":
        return f"v on {dev.type}, hip backend is GPU-only"
    if dtype not in _IO_DTYPES:
        return f"v dtype {dtype} not float32/bfloat16"
    if q.dtype != dtype or k.dtype != dtype or g.dtype != dtype:
        return f"q dtype {q.dtype}, k dtype {k.dtype} or g dtype {g.dtype} != v dtype {dtype}"
    if q.device != dev or k.device != dev or g.device != dev:
        return f"q on {q.device}, k on {k.device} or g on {g.device}, v on {dev}"
    if state is not None:
        if state.dtype != torch.float32:
            return f"needs float32 state, got {state.dtype}"
        if state.device != dev:
            return f"state on {state.device}, v on {dev}"
    return None


def _size_reason(B: int, L: int, H: int, K: int, V: int) -> str | None:
    """The kernels' limits (gated.hip args_status), repeated here so that supports() makes no library call."""
    if not (1 <= K <= _MAX_WIDTH and 1 <= V <= _MAX_WIDTH):
        return f"head widths K={K}, V={V} outside [1, {_MAX_WIDTH}]"
    rows = max(B, 1)
    too_many = H > 1 << 16 or L > 1 << 30 or rows > _MAX_GRID // H or rows * H > _MAX_GRID // 64
    if too_many or rows * H * (-(-L // 64) + 8) > _MAX_GRID:
        return f"B={B}, L={L}, H={H} needs more workgroups than one launch has"
    return None


def supports(q, k, v, g, state) -> str | None:
    """Reason the fused recurrence cannot handle these tensors, or None if it can."""
    reason = _tensor_reason(q, k, v, g, state)
    if reason is not None:
        return reason
    B, L, H, V = v.shape
    return _size_reason(B, L, H, q.shape[-1], V)


def supports_step(q, k, v, g, state) -> str | None:
    """Reason the fused step cannot handle these tensors, or None if it can."""
    reason = _tensor_reason(q, k, v, g, state)
    if reason is not None:
        return reason
    if not state.is_contiguous():
        return "the state, updated in place, must be contiguous"
    B, H, V = v.shape
    K = q.shape[-1]
    if not (1 <= K <= _STEP_MAX_K and V >= 1):
        return f"head widths K={K}, V={V}: K must be in [1, {_STEP_MAX_K}]"
    if V > 1 << 20 or H > 1 << 20 or B * H > _MAX_GRID // -(-V // 64):
        return f"B={B}, H={H}, V={V} needs more workgroups than one launch has"
    return None


def _dense(t):
    """``t`` with a dense last dimension, the only one the kernels read without a stride, and steps (if there is more than one) that
    64-step chunks reach with 32-bit offsets."""
    if (t.stride(-1) == 1 or t.shape[-1] == 1) and (t.dim() == 3 or t.stride(1) <= _MAX_STEP or t.shape[1] <= 1):
        return t
    return t.contiguous()


# the leading strides of q, k, v, g (and go): batch row, step and head; batch row and head in a step
_Strides8, _Strides12, _Strides15 = (ctypes.c_int64 * n for n in (8, 12, 15))


def _workspace(nbytes: int, t):
    return None if nbytes == 0 else _lib.workspace(nbytes, t.device)


def _screen(v, *others):
    dtype, dev = v.dtype, v.get_device()
    if dev < 0 or dtype not in _IO_DTYPES:
        raise TypeError(f"v: {dtype} on {v.device}, expected float32 or bfloat16 on a GPU")
    for t in others:
        if t.dtype != dtype or t.get_device() != dev:
            raise TypeError(f"{t.dtype} on {t.device}, expected {dtype} on {v.device}")


def _forward(q, k, v, g, state, train: bool):
    lib = _lib.load()
    _screen(v, q, k, g)
    q, k, v = _dense(q), _dense(k), _dense(v)
    state = None if state is None else state.contiguous()
    _lib.require(state, "state", (torch.float32,), v.device)
    B, L, H, V = v.shape
    Hk, K = q.shape[2:]
    o = torch.empty(B, L, H, V, device=v.device, dtype=v.dtype)
    last = torch.empty(B, H, K, V, device=v.device, dtype=torch.float32)
    io = _IO_DTYPES[v.dtype]
    kept = torch.empty(lib.tsfast_hip_gated_kept_bytes(B, L, H, Hk, K, V, io), device=v.device, dtype=torch.uint8) if train else None
    nbytes = lib.tsfast_hip_gated_fwd_workspace_bytes(B, L, H, Hk, K, V, io)
    ws = _workspace(nbytes, v)
    _lib.check(
        lib.tsfast_hip_gated_fwd_train(
            B, L, H, Hk, K, V, io, *map(_lib.ptr, (q, k, v, g)), _Strides12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride()),
            *map(_lib.ptr, (state, o, last)), _kept_ptr(kept), _lib.ptr(ws), nbytes, _lib.stream_of(v),
        ),
        "tsfast_hip_gated_fwd_train",
    )
    return o, last, kept


def _kept_ptr(kept):
    return None if kept is None or not kept.numel() else kept.data_ptr()


@custom_op("tsfast_hip::gated_recurrence")
def _recurrence_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor | None
) -> tuple[torch.Tensor, torch.Tensor]:
    return _forward(q, k, v, g, state, train=False)[:2]


@custom_op("tsfast_hip::gated_recurrence_train")
def _recurrence_train_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor | None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _forward(q, k, v, g, state, train=True)


@_recurrence_op.register_fake
def _(q, k, v, g, state):
    B, L, H, V = v.shape
    return v.new_empty(B, L, H, V), v.new_empty(B, H, q.shape[-1], V, dtype=torch.float32)


@_recurrence_train_op.register_fake
def _(q, k, v, g, state):
    B, L, H, V = v.shape
    kept = v.new_empty(torch.library.get_ctx().new_dynamic_size(), dtype=torch.uint8)  # the library's rule, by the chip's size
    return v.new_empty(B, L, H, V), v.new_empty(B, H, q.shape[-1], V, dtype=torch.float32), kept


@custom_op("tsfast_hip::gated_recurrence_bwd")
def _recurrence_bwd_op(
    go: torch.Tensor,
    glast: torch.Tensor | None,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    state: torch.Tensor | None,
    kept: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(v, q, k, g, go)
    q, k, v, go = _dense(q), _dense(k), _dense(v), _dense(go)
    state, glast = (None if t is None else t.contiguous() for t in (state, glast))
    _lib.require(state, "state", (torch.float32,), v.device)
    _lib.require(glast, "glast", (torch.float32,), v.device)
    B, L, H, V = v.shape
    Hk, K = q.shape[2:]
    gq, gk, gv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
    gg = torch.empty(B, L, H, device=v.device, dtype=v.dtype)
    gstate = None if state is None else torch.empty_like(state)
    io = _IO_DTYPES[v.dtype]
    if kept is not None:
        need = lib.tsfast_hip_gated_kept_bytes(B, L, H, Hk, K, V, io)
        if kept.dtype != torch.uint8 or kept.numel() != need or kept.get_device() != v.get_device() or not kept.is_contiguous():
            raise TypeError(f"kept: {kept.numel()} of {kept.dtype} on {kept.device}, expected {need} dense bytes on {v.device}")
    nbytes = lib.tsfast_hip_gated_bwd_workspace_bytes(B, L, H, Hk, K, V, io)
    ws = _workspace(nbytes, v)
    _lib.check(
        lib.tsfast_hip_gated_bwd_train(
            B, L, H, Hk, K, V, io, *map(_lib.ptr, (q, k, v, g, go)),
            _Strides15(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *go.stride()[:3]),
            *map(_lib.ptr, (state, glast, gq, gk, gv, gg, gstate)), _kept_ptr(kept), _lib.ptr(ws), nbytes, _lib.stream_of(v),
        ),
        "tsfast_hip_gated_bwd_train",
    )
    return gq, gk, gv, gg, (gstate if gstate is not None else v.new_empty(0, dtype=torch.float32))


@_recurrence_bwd_op.register_fake
def _(go, glast, q, k, v, g, state, kept=None):
    outs = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v, g))
    return (*outs, torch.empty(0 if state is None else state.shape, device=v.device, dtype=torch.float32))


def _setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*inputs, *output[2:])


def _backward(ctx, go, glast, gkept=None):
    q, k, v, g, state, *kept = ctx.saved_tensors
    if go is None:
        go = torch.zeros_like(v)
    gq, gk, gv, gg, gstate = _recurrence_bwd_op(go, glast, q, k, v, g, state, *kept)
    return gq, gk, gv, gg, (gstate if state is not None else None)


_recurrence_op.register_autograd(_backward, setup_context=_setup)
_recurrence_train_op.register_autograd(_backward, setup_context=_setup)


def run(q, k, v, g, state):
    """The fused recurrence: ``(o [B, L, H, V], last state [B, H, K, V] float32)``. A call that will be differentiated
    keeps the states between a row's segments (67 MB at most) for the backward, which would walk the rows for them again."""
    # a trace keeps the inputs alone: how many bytes more is not known to it
    if torch.is_grad_enabled() and not torch.compiler.is_compiling() and type(v) in _PLAIN:
        if q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or (state is not None and state.requires_grad):
            return _recurrence_train_op(q, k, v, g, state)[:2]
    return _recurrence_op(q, k, v, g, state)


@custom_op("tsfast_hip::gated_recurrence_step", mutates_args=("state",))
def _step_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    lib = _lib.load()
    _screen(v, q, k, g)
    if state.dtype != torch.float32 or state.get_device() != v.get_device() or not state.is_contiguous():
        raise TypeError(f"state: {state.dtype} on {state.device}, expected dense float32 on {v.device}")
    q, k, v = _dense(q), _dense(k), _dense(v)
    B, H, V = v.shape
    _, Hk, K = q.shape
    o = torch.empty(B, H, V, device=v.device, dtype=v.dtype)
    _lib.check(
        lib.tsfast_hip_gated_step(
            B, H, Hk, K, V, _IO_DTYPES[v.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
            _Strides8(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *g.stride()), state.data_ptr(), o.data_ptr(), _lib.stream_of(v),
        ),
        "tsfast_hip_gated_step",
    )
    return o


@_step_op.register_fake
def _(q, k, v, g, state):
    return v.new_empty(v.shape)


def step(q, k, v, g, state):
    """One fused step; ``state`` is updated in place. Returns ``o [B, H, V]``."""
    return _step_op(q, k, v, g, state)
