"""The operators of ``tsfast_amd.gated`` from their definitions, in float64 on the CPU.

Step by step, with the adjoints written out; shares no code with the package. Arguments are
torch tensors of any type, results float64 tensors.
"""

from __future__ import annotations

import torch


def _d(t):
    return None if t is None else t.detach().cpu().double()


def recurrence(q, k, v, g, state=None):
    """``S_t = exp(g_t) S_{t-1} + k_t v_t^T``, ``o_t = S_t^T q_t``: (o, S_L, every S_t with S_0 first)."""
    q, k, v, g, state = map(_d, (q, k, v, g, state))
    B, L, H, V = v.shape
    Hk, K = q.shape[2:]
    head = torch.arange(H) // (H // Hk)
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if state is None else state
    o, states = torch.zeros(B, L, H, V, dtype=torch.float64), [S]
    for t in range(L):
        S = torch.exp(g[:, t])[..., None, None] * S + k[:, t, head][..., :, None] * v[:, t][..., None, :]
        o[:, t] = (q[:, t, head][..., :, None] * S).sum(-2)
        states.append(S)
    return o, S, states


def recurrence_grads(go, glast, q, k, v, g, state=None):
    """Gradients of ``<go, o> + <glast, S_L>``: (q, k, v, g, state)."""
    *_, states = recurrence(q, k, v, g, state)
    q, k, v, g, go, glast = map(_d, (q, k, v, g, go, glast))
    B, L, H, V = v.shape
    Hk, K = q.shape[2:]
    share = H // Hk
    head = torch.arange(H) // share
    T = torch.zeros(B, H, K, V, dtype=torch.float64) if glast is None else glast
    gq, gk = torch.zeros(B, L, H, K, dtype=torch.float64), torch.zeros(B, L, H, K, dtype=torch.float64)
    gv, gg = torch.zeros_like(v), torch.zeros_like(g)
    for t in range(L - 1, -1, -1):
        T = T + q[:, t, head][..., :, None] * go[:, t][..., None, :]
        gq[:, t] = (states[t + 1] * go[:, t][..., None, :]).sum(-1)
        gk[:, t] = (T * v[:, t][..., None, :]).sum(-1)
        gv[:, t] = (T * k[:, t, head][..., :, None]).sum(-2)
        a = torch.exp(g[:, t])
        gg[:, t] = a * (states[t] * T).sum((-1, -2))
        T = a[..., None, None] * T
    gq, gk = (t.view(B, L, Hk, share, K).sum(3) for t in (gq, gk))
    return gq, gk, gv, gg, T


def _rms(x, eps):
    inv = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    n = x * inv
    return n, lambda dn: inv * (dn - n * (dn * n).mean(-1, keepdim=True))


def _silu(z):
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def gated_norm(x, gate, weight, groups, eps, gate_first, gy=None):
    """The output, or with ``gy`` (output, gradients of x, gate, weight)."""
    x, gate, weight, gy = map(_d, (x, gate, weight, gy))
    shape, D = x.shape, x.shape[-1]
    split = lambda t: t.reshape(-1, groups, D // groups)  # noqa: E731
    x = split(x)
    w = torch.ones(groups, D // groups, dtype=torch.float64) if weight is None else weight.view(groups, -1)
    act, slope = (torch.ones_like(x), torch.zeros_like(x)) if gate is None else _silu(split(gate))
    n, back = _rms(x * act if gate_first else x, eps)
    y = n * w if gate_first else n * w * act
    if gy is None:
        return y.reshape(shape)
    gy = split(gy)
    if gate_first:
        du = back(gy * w)
        gx, ggate, gw = du * act, du * x * slope, (gy * n).sum(0)
    else:
        gx, ggate, gw = back(gy * w * act), gy * n * w * slope, (gy * n * act).sum(0)
    return y.reshape(shape), gx.reshape(shape), ggate.reshape(shape), gw.reshape(D)


def residual_norm(x, residual, weight, post_weight, scale, eps, gnew=None, gy=None):
    """(new, y), or with ``gnew`` and ``gy`` also the gradients of x, residual, weight, post_weight, scale."""
    x, r, w, p, s, gnew, gy = map(_d, (x, residual, weight, post_weight, scale, gnew, gy))
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    w, s = (one if t is None else t for t in (w, s))
    n1, back1 = (x, lambda d: d) if p is None else _rms(x, eps)
    b = n1 if p is None else n1 * p
    new = r + b * s
    n, back = _rms(new, eps)
    if gnew is None:
        return new, n * w
    rows = tuple(range(x.dim() - 1))
    dnew = gnew + back(gy * w)
    gx = back1(dnew * s * (one if p is None else p))
    gp = (dnew * s * n1).sum(rows)
    return new, n * w, gx, dnew, (gy * n).sum(rows), gp, (dnew * b).sum(rows)
