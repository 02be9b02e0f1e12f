"""A Mamba layer in service in float64, token by token, from the definition: packed convolution and scan, and one step."""

from __future__ import annotations

import torch


def _d(t):
    return None if t is None else t.detach().double()


def _silu(x):
    return x * torch.special.expit(x)


def conv_packed(x, starts, weight, bias, tails=None):
    x, w, bias, tails = _d(x), _d(weight)[:, 0], _d(bias), _d(tails)
    (T, D), S, K = x.shape, len(starts) - 1, weight.shape[-1]
    u, left = torch.zeros_like(x), x.new_zeros(S, D, K - 1) if tails is None else tails.clone()
    at = starts.tolist()
    for s in range(S):
        past = left[s]
        for t in range(at[s], at[s + 1]):
            window = torch.cat((past, x[t][:, None]), 1)
            pre = (window * w).sum(1)
            u[t] = _silu(pre if bias is None else pre + bias)
            past = window[:, 1:]
        left[s] = past
    return u, left


def ssm_packed(draw, A, B_t, C_t, u, z, Dp, starts, h0=None):
    draw, A, B_t, C_t, u, z, Dp, h0 = map(_d, (draw, A, B_t, C_t, u, z, Dp, h0))
    S, D, N = len(starts) - 1, *A.shape
    out, last = torch.zeros_like(draw), draw.new_zeros(S, D, N) if h0 is None else h0.clone()
    delta = torch.nn.functional.softplus(draw)
    at = starts.tolist()
    for s in range(S):
        h = last[s]
        for t in range(at[s], at[s + 1]):
            h = torch.exp(delta[t][:, None] * A) * h + (delta[t] * u[t])[:, None] * B_t[t]
            out[t] = (h @ C_t[t] + Dp * u[t]) * _silu(z[t])
        last[s] = h
    return out, last


def step(x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp):
    """``(out, new conv_state, new ssm_state)``."""
    x, z, tail, h, wc, bc, xp, dp, db, A, Dp = map(_d, (x, z, conv_state, ssm_state, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, Dp))
    N, R = A.shape[1], dp.shape[1]
    window = torch.cat((tail, x[..., None]), -1)
    pre = (window * wc[:, 0]).sum(-1)
    u = _silu(pre if bc is None else pre + bc)
    p = u @ xp.T
    draw = p[:, :R] @ dp.T
    delta = torch.nn.functional.softplus(draw if db is None else draw + db)
    h = torch.exp(delta[..., None] * A) * h + (delta * u)[..., None] * p[:, None, R : R + N]
    return ((h * p[:, None, R + N :]).sum(-1) + Dp * u) * _silu(z), window[..., 1:], h
