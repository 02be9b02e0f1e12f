"""HIP backend of a Mamba layer in service: packed prompts and single tokens (``csrc/packed.hip``, ``csrc/step.hip``).

``supports_conv`` / ``conv``, ``supports_ssm`` / ``ssm`` run the convolution and the scan over sequences of different lengths
packed into one row of tokens; ``supports_step`` / ``step`` everything between a layer's projections for one token of each
sequence, with both states in place. The ops ``tsfast_hip::mamba_conv_packed``, ``mamba_ssm_packed`` and ``mamba_step`` have no
gradient: training runs ``mamba_conv`` and ``mamba_ssm``.

Sequence tensors are float32 or bfloat16 at any distance between rows (a last dimension that is not dense is copied); the state
of the scan is float32, the sums too.
"""

from __future__ import annotations

__all__ = ["supports_conv", "conv", "supports_ssm", "ssm", "supports_step", "step"]

import torch

from .. import _lib
from ..ops import custom_op

_IO_DTYPES = {torch.float32: _lib.TSF_DTYPE_F32, torch.bfloat16: _lib.TSF_DTYPE_BF16}
_MAX_GRID = (1 << 24) - 1
_MAX_D, _MAX_T, _MAX_S = 1 << 24, 1 << 30, 1 << 30
_MAX_N, _MAX_P = 64, 1024  # states; columns of x_proj (step.hip kMaxP)


def _tensor_reason(x, alike, params, wide, starts=None) -> str | None:
    """``alike``: of x's type; ``params``: float32 or bfloat16; ``wide``: float32 (each a tuple, None where an optional tensor is absent)."""
    dtype, dev = x.dtype, x.get_device()
    if dev < 0:
        return f"x on {x.device}, hip backend is GPU-only"
    if dtype not in _IO_DTYPES:
        return f"sequence dtype {dtype} not float32/bfloat16"
    bad = starts if starts is not None and starts.get_device() != dev else None
    for t in alike:
        if t is not None and (t.dtype != dtype or t.get_device() != dev):
            bad = t
    for t in params:
        if t is not None and (t.dtype not in _IO_DTYPES or t.get_device() != dev):
            bad = t
    for t in wide:
        if t is not None and (t.dtype != torch.float32 or t.get_device() != dev):
            bad = t
    return None if bad is None else f"a tensor is {bad.dtype} on {bad.device}, x {dtype} on {x.device}"


def _packed_reason(T: int, S: int, D: int) -> str | None:
    if D > _MAX_D or T > _MAX_T or S > _MAX_S:
        return f"T={T}, S={S}, D={D} beyond the kernels' sizes"
    return None


def supports_conv(x, starts, weight, bias, tails) -> str | None:
    """Reason the packed convolution cannot handle these tensors, or None if it can."""
    reason = _tensor_reason(x, (tails,), (weight, bias), (), starts) or _packed_reason(x.shape[0], starts.shape[0] - 1, x.shape[1])
    if reason is not None:
        return reason
    K = weight.shape[-1]
    if not 2 <= K <= 8:
        return f"kernel width {K} outside the supported range [2, 8]"
    T, D = x.shape
    if -(-(-(-T // 4) + starts.shape[0] - 1) * -(-D // (8 if x.dtype == torch.bfloat16 else 4)) // 256) > _MAX_GRID:
        return f"T={T}, S={starts.shape[0] - 1}, D={D} needs more workgroups than one launch has"
    return None


def supports_ssm(draw, A, B_t, C_t, u, z, Dp, starts, h0) -> str | None:
    """Reason the packed scan cannot handle these tensors, or None if it can."""
    reason = _tensor_reason(draw, (B_t, C_t, u, z), (), (A, Dp, h0), starts) or _packed_reason(draw.shape[0], starts.shape[0] - 1, draw.shape[1])
    if reason is not None:
        return reason
    if A.shape[-1] > _MAX_N:
        return f"state size N={A.shape[-1]} above {_MAX_N}"
    return None  # rows are cut into 256 segments at most, few where D is large: any T and D is one launch


def supports_step(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp) -> str | None:
    """Reason the fused step cannot handle these tensors, or None if it can."""
    reason = _tensor_reason(x, (z, conv_state), (conv_weight, conv_bias, x_proj, dt_proj, dt_bias), (ssm_state, A, Dp))
    if reason is not None:
        return reason
    if not (conv_state.is_contiguous() and ssm_state.is_contiguous()):
        return "the states, updated in place, must be contiguous"
    (B, D), N, P, K = x.shape, A.shape[-1], x_proj.shape[0], conv_weight.shape[-1]
    if not 2 <= K <= 8 or N > _MAX_N or P > _MAX_P:
        return f"kernel width {K}, N={N} states or {P} columns of x_proj: at most 2..8, {_MAX_N} and {_MAX_P}"
    if D > _MAX_D or B > 1 << 31 or -(-B // 8) * -(-D // 64) > _MAX_GRID:
        return f"B={B}, D={D} needs more workgroups than one launch has"
    return None


def _screen(x, alike, params, wide, starts=None):
    reason = _tensor_reason(x, alike, params, wide, starts)
    if reason is not None:
        raise TypeError(reason)


def _rows(t):
    """``t [rows, width]`` with a dense last dimension."""
    return t if t.is_contiguous() or t.stride(1) == 1 else t.contiguous()


def _dense(t):
    return None if t is None else t.contiguous()


@custom_op("tsfast_hip::mamba_conv_packed")
def _conv_op(
    x: torch.Tensor, starts: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, tails: torch.Tensor | None
) -> tuple[torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(x, (tails,), (weight, bias), (), starts)
    (T, D), S, K = x.shape, starts.shape[0] - 1, weight.shape[-1]
    x, starts, weight, bias, tails = _rows(x), starts.contiguous(), weight.contiguous(), _dense(bias), _dense(tails)
    with _lib.device_of(x):
        out = torch.empty(T, D, device=x.device, dtype=x.dtype)
        tails_out = torch.empty(S, D, K - 1, device=x.device, dtype=x.dtype)
        _lib.check(
            lib.tsfast_hip_conv_packed(
                T, S, D, K, _IO_DTYPES[x.dtype], starts.dtype == torch.int64, _IO_DTYPES[weight.dtype],
                _IO_DTYPES[weight.dtype if bias is None else bias.dtype], x.data_ptr(), x.stride(0),
                *map(_lib.ptr, (starts, tails, weight, bias, out, tails_out)), _lib.stream_of(x),
            ),
            "tsfast_hip_conv_packed",
        )
    return out, tails_out


@_conv_op.register_fake
def _(x, starts, weight, bias, tails):
    return x.new_empty(x.shape), x.new_empty(starts.shape[0] - 1, x.shape[1], weight.shape[-1] - 1)


def conv(x, starts, weight, bias, tails):
    """The fused packed convolution; see :func:`tsfast_amd.mamba.mamba_conv_packed`."""
    return _conv_op(x, starts, weight, bias, tails)


@custom_op("tsfast_hip::mamba_ssm_packed")
def _ssm_op(
    draw: torch.Tensor,
    A: torch.Tensor,
    B_t: torch.Tensor,
    C_t: torch.Tensor,
    u: torch.Tensor,
    z: torch.Tensor,
    Dp: torch.Tensor,
    starts: torch.Tensor,
    h0: torch.Tensor | None,
) -> tuple[torch.Tensor, torch.Tensor]:
    lib = _lib.load()
    _screen(draw, (B_t, C_t, u, z), (), (A, Dp, h0), starts)
    (T, D), S, N = draw.shape, starts.shape[0] - 1, A.shape[-1]
    draw, B_t, C_t, u, z = map(_rows, (draw, B_t, C_t, u, z))
    A, Dp, starts, h0 = A.contiguous(), Dp.contiguous(), starts.contiguous(), _dense(h0)
    with _lib.device_of(draw):
        out = torch.empty(T, D, device=draw.device, dtype=draw.dtype)
        h_last = torch.empty(S, D, N, device=draw.device, dtype=torch.float32)
        nbytes = lib.tsfast_hip_mamba_packed_workspace_bytes(T, S, D, N)
        ws = _lib.workspace(nbytes, draw.device) if nbytes > 0 else None
        _lib.check(
            lib.tsfast_hip_mamba_packed(
                T, S, D, N, _IO_DTYPES[draw.dtype], starts.dtype == torch.int64, draw.data_ptr(), draw.stride(0), A.data_ptr(),
                B_t.data_ptr(), B_t.stride(0), C_t.data_ptr(), C_t.stride(0), u.data_ptr(), u.stride(0), z.data_ptr(), z.stride(0),
                *map(_lib.ptr, (Dp, starts, h0, out, h_last, ws)), nbytes, _lib.stream_of(draw),
            ),
            "tsfast_hip_mamba_packed",
        )
    return out, h_last


@_ssm_op.register_fake
def _(draw, A, B_t, C_t, u, z, Dp, starts, h0):
    return draw.new_empty(draw.shape), draw.new_empty(starts.shape[0] - 1, *A.shape, dtype=torch.float32)


def ssm(draw, A, B_t, C_t, u, z, Dp, starts, h0):
    """The fused packed scan; see :func:`tsfast_amd.mamba.mamba_ssm_packed`."""
    return _ssm_op(draw, A, B_t, C_t, u, z, Dp, starts, h0)


@custom_op("tsfast_hip::mamba_step", mutates_args=("conv_state", "ssm_state"))
def _step_op(
    x: torch.Tensor,
    z: torch.Tensor,
    conv_state: torch.Tensor,
    ssm_state: torch.Tensor,
    conv_weight: torch.Tensor,
    conv_bias: torch.Tensor | None,
    x_proj: torch.Tensor,
    dt_proj: torch.Tensor,
    dt_bias: torch.Tensor | None,
    A: torch.Tensor,
    Dp: torch.Tensor,
) -> torch.Tensor:
    lib = _lib.load()
    params = (conv_weight, conv_bias, x_proj, dt_proj, dt_bias)
    _screen(x, (z, conv_state), params, (ssm_state, A, Dp))
    if not (conv_state.is_contiguous() and ssm_state.is_contiguous()):
        raise TypeError("the states must be contiguous")
    x, z = _rows(x), _rows(z)
    A, Dp = (t if t.is_contiguous() else t.contiguous() for t in (A, Dp))
    one = conv_weight.dtype
    if x_proj.dtype != one or dt_proj.dtype != one or (conv_bias is not None and conv_bias.dtype != one):  # the kernels take these four in one type
        params = (*(None if t is None else t.float() for t in params[:4]), dt_bias)
    conv_weight, conv_bias, x_proj, dt_proj, dt_bias = (t if t is None or t.is_contiguous() else t.contiguous() for t in params)
    (B, D), N, R, K = x.shape, A.shape[-1], dt_proj.shape[-1], conv_weight.shape[-1]
    with _lib.device_of(x):
        out = torch.empty(B, D, device=x.device, dtype=x.dtype)
        nbytes = lib.tsfast_hip_mamba_step_workspace_bytes(B, D, N, R, K)
        ws = _lib.workspace(nbytes, x.device)
        _lib.check(
            lib.tsfast_hip_mamba_step(
                B, D, N, R, K, _IO_DTYPES[x.dtype], _IO_DTYPES[conv_weight.dtype], 0 if dt_bias is None else _IO_DTYPES[dt_bias.dtype],
                x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0), conv_state.data_ptr(), ssm_state.data_ptr(), conv_weight.data_ptr(),
                None if conv_bias is None else conv_bias.data_ptr(), x_proj.data_ptr(), dt_proj.data_ptr(),
                None if dt_bias is None else dt_bias.data_ptr(), A.data_ptr(), Dp.data_ptr(), out.data_ptr(), ws.data_ptr(), nbytes,
                _lib.stream_of(x),
            ),
            "tsfast_hip_mamba_step",
        )
    return out


@_step_op.register_fake
def _(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp):
    return x.new_empty(x.shape)


def step(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp):
    """The fused step; see :func:`tsfast_amd.mamba.mamba_step`."""
    return _step_op(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp)
