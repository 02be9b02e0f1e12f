"""The gradient of the gated recurrence's log decays where decays are strong, where rows are packed and where
parts of a row have no loss (HIP), each head, sequence and step group against its own size.

Every term of dg_t = exp(g_t) <S_{t-1}, T_t> carries the decay over step t, so the result is as accurate
relative to its own size as any other. Bars, derived before the first run, relative to the largest value of the head (the
sequence, the steps) compared and not of the tensor: float32 1e-5, the package's bar (sums of up to 64 x 64 pairs over 128
columns in float32, about 1e-6; an exponent of 2^-100 rounded to float32 adds 100 x 2^-24 x ln 2 = 4e-6). bfloat16 rounds dg
once, 2^-9 of its own size, and what is split into bfloat16 parts before it carries 2^-16: 2^-8. What the definition makes
zero, whatever surrounds it, is zero.
"""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import dispatch, gated

_DTYPES = [torch.float32, torch.bfloat16]
_BAR = {torch.float32: 1e-5, torch.bfloat16: 2**-8}


def _inputs(B, L, H, Hk, K, V, dtype, seed=0, device="cuda"):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    g = -torch.rand(B, L, H, generator=r) * 0.05
    seq = (n(B, L, Hk, K), n(B, L, Hk, K) / K**0.5, n(B, L, H, V), g)
    rest = (n(B, H, K, V), n(B, L, H, V).to(dtype), n(B, H, K, V))
    return *(t.to(device, dtype) for t in seq), *(t.to(device) for t in rest)


def _grads(q, k, v, g, state, go, gl, backend="hip"):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state) if t is not None]
    with dispatch.use_backend(backend):
        o, last = gated.gated_recurrence(*leaves[:4], leaves[4] if state is not None else None)
    return torch.autograd.grad([o, last] if gl is not None else [o], leaves, [go, gl] if gl is not None else [go])


def _assert_close(got, want, bar, what):
    """``got`` within ``bar`` of ``want``'s own largest value, and zero where all of it is."""
    got, want = got.detach().cpu().double(), want.double()
    assert torch.isfinite(got).all(), what
    size = float(want.abs().max()) if want.numel() else 0.0
    if size == 0.0:
        assert (got == 0).all(), (what, float(got.abs().max()))
    else:
        assert float((got - want).abs().max()) < bar * size, (what, float((got - want).abs().max()) / size)


_STRONG = (-0.02, -1.0, -3.0, -5.0, -8.0, -12.0, -16.0, -30.0)


def _check_constant(B, L, Hk, K, V, dtype, device="cuda", backend="hip"):
    H = len(_STRONG)
    q, k, v, g, s, go, gl = _inputs(B, L, H, Hk, K, V, dtype, seed=L + K, device=device)
    g = torch.tensor(_STRONG, device=device).to(dtype).expand(B, L, H).contiguous()
    got = _grads(q, k, v, g, s, go, gl, backend)
    want = G.recurrence_grads(go, gl, q, k, v, g, s)
    for b in range(B):
        for h in range(H):
            _assert_close(got[3][b, :, h], want[3][b, :, h], _BAR[dtype], (b, _STRONG[h]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("B,L,Hk,K,V", [(1, 1, 8, 16, 16), (2, 64, 8, 20, 100), (1, 65, 2, 128, 128), (1, 200, 8, 5, 7), (1, 1100, 8, 64, 64),
                                        (1, 1100, 4, 100, 33), (1, 1100, 8, 128, 128)])
def test_strong_constant_decays(gpu, B, L, Hk, K, V, dtype):
    """Slow heads and ones that forget within a step in one call."""
    _check_constant(B, L, Hk, K, V, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("K,V", [(24, 40), (128, 128)])
def test_single_strong_steps_among_mild_ones(gpu, K, V, dtype):
    """Gates that forget now and then: the gradients of those steps, 1e-4 to 1e-9 of their neighbours', by themselves."""
    q, k, v, g, s, go, gl = _inputs(2, 700, 3, 3, K, V, dtype, seed=5)
    where = torch.zeros(700, dtype=torch.bool)
    where[[0, 17, 63, 64, 100, 127, 128, 191, 300, 301, 555, 699]] = True
    for h, strong in enumerate((-9.0, -14.0, -20.0)):
        g[:, where, h] = strong
    got, want = _grads(q, k, v, g, s, go, gl)[3].cpu(), G.recurrence_grads(go, gl, q, k, v, g, s)[3]
    for b in range(2):
        for h in range(3):
            _assert_close(got[b, where, h], want[b, where, h], _BAR[dtype], (b, h, "strong"))
            _assert_close(got[b, ~where, h], want[b, ~where, h], _BAR[dtype], (b, h, "mild"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("K,V,Hk", [(16, 24, 2), (64, 64, 1), (100, 128, 2)])
def test_packed_sequences_do_not_leak(gpu, K, V, Hk, dtype):
    """Sequences parted by -inf, one without a loss and one with a small weight: each by itself."""
    L = 900
    starts = [0, 40, 64, 65, 128, 300, 448, 640, 700, L]
    weights = [1.0, 0.0, 1.0, 1e-3, 0.0, 1e-3, 30.0, 0.0, 1.0]
    q, k, v, g, s, go, gl = _inputs(1, L, 2, Hk, K, V, dtype, seed=9)
    for t0, t1, w in zip(starts, starts[1:], weights):
        go[:, t0:t1] *= w
        if t0:
            g[:, t0] = float("-inf")
    got, want = _grads(q, k, v, g, s, go, gl), G.recurrence_grads(go, gl, q, k, v, g, s)
    for t0, t1, w in zip(starts, starts[1:], weights):
        for h in range(2):
            _assert_close(got[3][0, t0:t1, h], want[3][0, t0:t1, h], _BAR[dtype], (t0, w, h))
        for n in (1, 2):  # dk and dv, which part sequences in the same way
            _assert_close(got[n][0, t0:t1], want[n][0, t0:t1], _BAR[dtype], (t0, w, "kv"[n - 1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("L,K,V", [(300, 32, 48), (1200, 64, 128)])
def test_steps_without_loss_or_state_have_no_gradient(gpu, L, K, V, dtype):
    """After the last step with a loss, and before the first key, dg is zero by definition."""
    first, end = 80, L - 110
    q, k, v, g, _, go, _ = _inputs(1, L, 2, 2, K, V, dtype, seed=3)
    go[:, end:] = 0
    k[:, :first] = 0
    got, want = _grads(q, k, v, g, None, go, None)[3], G.recurrence_grads(go, None, q, k, v, g)[3]
    assert (want[:, : first + 1] == 0).all() and (want[:, end:] == 0).all()
    assert (got[:, : first + 1] == 0).all() and (got[:, end:] == 0).all()
    for h in range(2):
        _assert_close(got[0, first + 1 : end, h], want[0, first + 1 : end, h], _BAR[dtype], h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _DTYPES)
def test_a_compiled_pass_has_the_same_gate_gradient(gpu, dtype):
    """Without the forward's segment states kept."""
    q, k, v, g, s, go, gl = _inputs(1, 1100, len(_STRONG), 1, 48, 80, dtype, seed=4)
    g = torch.tensor(_STRONG, device="cuda").to(dtype).expand(1, 1100, len(_STRONG)).contiguous()
    from tsfast_amd.gated import recurrence_hip

    with torch.no_grad():
        got = recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, s)[3]
    want = G.recurrence_grads(go, gl, q, k, v, g, s)[3]
    for h, c in enumerate(_STRONG):
        _assert_close(got[0, :, h], want[0, :, h], _BAR[dtype], c)


def test_torch_path_keeps_the_same_bars():
    _check_constant(1, 200, 2, 12, 20, torch.float32, device="cpu", backend="reference")


def test_oracle_gate_gradients_agree_with_autograd_at_strong_decays():
    """The written-out adjoint against torch's of the recurrence step by step, both in float64 (1e-12 of each head's size: products
    of 20 steps)."""
    q, k, v, g, s, go, gl = (t.double() for t in _inputs(1, 20, len(_STRONG), 2, 5, 6, torch.float32, seed=6, device="cpu"))
    g = torch.tensor(_STRONG, dtype=torch.float64).expand(1, 20, len(_STRONG)).clone().requires_grad_()
    head = torch.arange(len(_STRONG)) // (len(_STRONG) // 2)
    S, loss = s, 0.0
    for t in range(20):
        S = torch.exp(g[:, t])[..., None, None] * S + k[:, t, head][..., None] * v[:, t][..., None, :]
        loss = loss + (go[:, t] * (q[:, t, head][..., None] * S).sum(-2)).sum()
    (want,) = torch.autograd.grad(loss + (gl * S).sum(), g)
    got = G.recurrence_grads(go, gl, q, k, v, g, s)[3]
    for h, c in enumerate(_STRONG):
        _assert_close(got[0, :, h], want[0, :, h], 1e-12, c)
