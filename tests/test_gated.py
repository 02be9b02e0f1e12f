"""The gated block's operators without a GPU: the torch path against the float64 oracle, the oracle against
differences, the refusals, and the size limits the Python side repeats.

Bars: the torch path in float64 to 1e-11 and in float32 to 1e-5 of the largest value (the reduction lengths here
are below 300, so float32 sums stay within 300 x 2^-24 = 2e-5 in the worst and about 1e-6 in the usual case; the
package's float32 bar is 1e-5)."""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import _lib, gated
from tsfast_amd.gated import norm_hip, recurrence_hip


def _rel(a, b):
    return float((a.detach().double() - b.detach()).abs().max() / b.abs().max().clamp_min(1e-30)) if b.numel() else 0.0


def _inputs(B, L, H, Hk, K, V, dtype=torch.float64, seed=0):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, dtype=torch.float64).to(dtype)  # noqa: E731
    g = (-torch.rand(B, L, H, generator=r, dtype=torch.float64) * 0.3).to(dtype)
    return n(B, L, Hk, K), n(B, L, Hk, K) / K**0.5, n(B, L, H, V), g, n(B, H, K, V), n(B, L, H, V), n(B, H, K, V)


@pytest.mark.parametrize("dtype,tol", [(torch.float64, 1e-11), (torch.float32, 1e-5)])
@pytest.mark.parametrize("B,L,H,Hk,K,V", [(2, 1, 2, 2, 3, 5), (1, 64, 1, 1, 8, 8), (2, 130, 6, 2, 7, 9), (1, 65, 4, 1, 200, 3)])
def test_torch_path_matches_the_oracle(B, L, H, Hk, K, V, dtype, tol):
    q, k, v, g, state, go, gl = _inputs(B, L, H, Hk, K, V, dtype)
    g[:, ::29] = float("-inf")
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    o, last = gated.gated_recurrence(*leaves)
    grads = torch.autograd.grad([o, last], leaves, [go, gl])
    want_o, want_last, _ = G.recurrence(q, k, v, g, state)
    assert o.dtype == dtype and _rel(o, want_o) < tol and _rel(last, want_last) < tol
    for got, want in zip(grads, G.recurrence_grads(go, gl, q, k, v, g, state)):
        assert torch.isfinite(got).all() and _rel(got, want) < tol


def test_oracle_gradients_agree_with_differences():
    args = _inputs(1, 9, 2, 1, 3, 4, seed=3)
    q, k, v, g, state, go, gl = args

    def loss(*a):
        o, last, _ = G.recurrence(*a)
        return float((o * go).sum() + (last * gl).sum())

    grads = G.recurrence_grads(go, gl, q, k, v, g, state)
    d = 1e-6
    for n, t in enumerate((q, k, v, g, state)):
        for at in (0, t.numel() // 2, t.numel() - 1):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[at] = d
            up, down = ([a if i != n else a + s * step.view(t.shape) for i, a in enumerate((q, k, v, g, state))] for s in (1, -1))
            want = (loss(*up) - loss(*down)) / (2 * d)
            assert abs(want - float(grads[n].flatten()[at])) < 1e-6 * max(1.0, abs(want))


@pytest.mark.parametrize("L", [0, 1, 70])
def test_torch_path_state_and_step(L):
    q, k, v, g, state, *_ = _inputs(2, L, 4, 2, 5, 6)
    o, last = gated.gated_recurrence(q, k, v, g, state)
    S, outs = state.clone(), []
    for t in range(L):
        outs.append(gated.gated_recurrence_step(q[:, t], k[:, t], v[:, t], g[:, t], S))
    assert o.shape == v.shape and torch.allclose(last, S, atol=1e-12)
    if L:
        assert torch.allclose(o, torch.stack(outs, 1), atol=1e-12)
    empty, zero = gated.gated_recurrence(q[:0], k[:0], v[:0], g[:0])
    assert empty.shape == (0, L, 4, 6) and zero.shape == (0, 4, 5, 6)


@pytest.mark.parametrize("groups,first,gate", [(1, False, True), (3, False, True), (3, True, True), (2, False, False)])
def test_gated_norm_torch_path(groups, first, gate):
    r = torch.Generator().manual_seed(5)
    x, z, gy = (torch.randn(2, 7, 12, generator=r, dtype=torch.float64) for _ in range(3))
    w = torch.rand(12, generator=r, dtype=torch.float64) + 0.5
    z = z if gate else None
    leaves = [t.requires_grad_() for t in (x, z, w) if t is not None]
    y = gated.gated_norm(x, z, w, groups=groups, eps=1e-3, gate_first=first)
    want = G.gated_norm(x, z, w, groups, 1e-3, first and gate, gy)
    assert _rel(y, want[0]) < 1e-12
    wants = [t for t, there in zip(want[1:], (True, gate, True)) if there]
    for got, ref in zip(torch.autograd.grad(y, leaves, gy), wants):
        assert _rel(got, ref) < 1e-11


@pytest.mark.parametrize("post,scale", [(True, True), (False, True), (True, False), (False, False)])
def test_residual_norm_torch_path(post, scale):
    r = torch.Generator().manual_seed(6)
    x, res, gn, gy = (torch.randn(3, 5, 10, generator=r, dtype=torch.float64) for _ in range(4))
    w, p, s = (torch.rand(10, generator=r, dtype=torch.float64) + 0.5 for _ in range(3))
    p, s = p if post else None, s if scale else None
    leaves = [t.requires_grad_() for t in (x, res, w, p, s) if t is not None]
    new, y = gated.residual_norm(x, res, w, post_weight=p, scale=s, eps=1e-3)
    want = G.residual_norm(x, res, w, p, s, 1e-3, gn, gy)
    assert _rel(new, want[0]) < 1e-12 and _rel(y, want[1]) < 1e-12
    wants = [t for t, there in zip(want[2:], (True, True, True, post, scale)) if there]
    for got, ref in zip(torch.autograd.grad([new, y], leaves, [gn, gy]), wants):
        assert _rel(got, ref) < 1e-11


@pytest.mark.parametrize("first", [False, True])
def test_norm_gradients_agree_with_differences(first):
    r = torch.Generator().manual_seed(7)
    x, z = (torch.randn(3, 8, generator=r, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w, p, s = (torch.rand(8, generator=r, dtype=torch.float64).add(0.5).requires_grad_() for _ in range(3))
    assert torch.autograd.gradcheck(lambda x, z, w: gated.gated_norm(x, z, w, groups=2, gate_first=first), (x, z, w))
    assert torch.autograd.gradcheck(lambda x, z, w, p, s: gated.residual_norm(x, z, w, post_weight=p, scale=s), (x, z, w, p, s))


def test_refusals():
    q, k, v, g, state, *_ = _inputs(2, 5, 4, 2, 3, 6)
    ok = gated.gated_recurrence
    for bad in (
        lambda: ok(q, k[:, :4], v, g),
        lambda: ok(q[:, :, :1].expand(-1, -1, 3, -1), k[:, :, :1].expand(-1, -1, 3, -1), v, g),  # 3 heads for 4
        lambda: ok(q, k, v[0], g),
        lambda: ok(q, k, v, g[..., :2]),
        lambda: ok(q, k, v, g, state[:, :, :2]),
        lambda: gated.gated_recurrence_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state[:1]),
        lambda: gated.gated_norm(v, None, None, groups=4),
        lambda: gated.gated_norm(v, v[:1], None),
        lambda: gated.gated_norm(v, v.float(), None),
        lambda: gated.gated_norm(v, v, torch.ones(5)),
        lambda: gated.residual_norm(v, v[:1], None),
        lambda: gated.residual_norm(v.float(), v, None),
        lambda: gated.residual_norm(v, v, None, scale=torch.ones(1)),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        gated.gated_recurrence_step(q[:, 0].requires_grad_(), k[:, 0], v[:, 0], g[:, 0], state)


@pytest.fixture(scope="module")
def lib():
    if not _lib.available():
        pytest.skip("libtsfast_hip.so not built (run __graft_entry__.build())")
    return _lib.load()


@pytest.mark.parametrize(
    "B,L,H,K,V",
    [(1, 1, 1, 1, 1), (16, 4096, 12, 128, 128), (1, 65536, 6, 64, 64), (1, 8, 1, 129, 8), (1, 8, 1, 8, 129), (0, 5, 2, 4, 4),
     (1, 1 << 30, 1, 8, 8), (1, (1 << 30) - 600, 1, 8, 8), (1, 1 << 31, 1, 8, 8), (262143, 1, 1, 8, 8), (262144, 1, 1, 8, 8),
     (100000, 9000, 1, 8, 8), (1 << 24, 1, 2, 8, 8), (1, 4, 65537, 8, 8)],
)
def test_recurrence_supports_mirrors_the_library(lib, B, L, H, K, V):
    ok = lib.tsfast_hip_gated_bwd_workspace_bytes(B, L, H, H, K, V, 0) >= 0
    assert (recurrence_hip._size_reason(B, L, H, K, V) is None) == ok
    assert (lib.tsfast_hip_gated_fwd_workspace_bytes(B, L, H, H, K, V, 1) >= 0) == ok


def test_entry_points_refuse_before_any_launch(lib):
    assert lib.tsfast_hip_norm_max_width() == norm_hip._MAX_WIDTH
    fwd = lib.tsfast_hip_gated_fwd
    assert fwd(1, 4, 3, 2, 8, 8, 0, *([None] * 9), 0, None) == -1  # 2 heads for 3
    assert fwd(1, 4, 2, 2, 8, 8, 7, *([None] * 9), 0, None) == -1  # no such type
    assert fwd(1, 4, 2, 2, 200, 8, 0, *([None] * 9), 0, None) == -3
    assert fwd(1, 4, 2, 2, 8, 8, 0, *([None] * 9), 0, None) == -1  # NULL tensors
    assert fwd(0, 4, 2, 2, 8, 8, 0, *([None] * 9), 0, None) == 0
    assert lib.tsfast_hip_gated_bwd(1, 4, 2, 2, 8, 8, 0, *([None] * 14), 0, None) == -1
    assert lib.tsfast_hip_gated_step(1, 2, 2, 1025, 8, 0, *([None] * 8)) == -3
    assert lib.tsfast_hip_gated_step(1, 2, 2, 8, 8, 0, *([None] * 8)) == -1
    nf = lib.tsfast_hip_gated_norm_fwd
    assert nf(4, 1, 8193, 0, 0, 1e-5, None, 0, None, 0, None, None, None) == -3
    assert nf(4, 1, 8, 0, 0, 1e-5, None, 0, None, 0, None, None, None) == -1
    assert nf(0, 1, 8, 0, 0, 1e-5, None, 0, None, 0, None, None, None) == 0
    rf = lib.tsfast_hip_residual_norm_fwd
    assert rf(4, 8, 0, 1, 1e-5, None, 0, None, 0, *([None] * 6)) == -1  # a bfloat16 stream beside float32
    assert lib.tsfast_hip_residual_norm_workspace_bytes(4, 8193) == -1
    assert lib.tsfast_hip_gated_norm_workspace_bytes(4, 0, 8) == -1
