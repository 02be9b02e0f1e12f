"""The gated feed-forward block without a GPU: the torch path against the float64 oracle, the oracle against differences,
the refusals, and what the Python side repeats of the library.

Bars: the torch path in float64 to 1e-11 of the largest value; in float32 and bfloat16 sums of at most 60 float32 products,
60 x 2^-24 = 4e-6 in the worst case, under the package's bar of 1e-5, and half a step of bfloat16 (2^-8) for the result."""

import pytest
import torch

from oracle import feed_oracle
from tsfast_amd import _lib, gated
from tsfast_amd.gated import feed_hip

F64, F32, BF = torch.float64, torch.float32, torch.bfloat16


def _inputs(shape, D, F, dtype=F64, bias=True, seed=0):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, dtype=F64)  # noqa: E731
    out = n(*shape, D), n(F, D) / D**0.5, n(F, D) / D**0.5, *((n(F), n(F)) if bias else (None, None)), n(*shape, F)
    return [None if t is None else t.to(dtype) for t in out]


def _rel(a, b):
    return float((a.detach().double() - b).abs().max() / b.abs().max().clamp_min(1e-30)) if b.numel() else 0.0


@pytest.mark.parametrize("dtype,tol", [(F64, 1e-11), (F32, 1e-5), (BF, 2.0**-8 + 1e-5)])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("shape,D,F,bias", [((1,), 1, 1, True), ((2, 3), 7, 5, False), ((4,), 33, 60, True), ((0,), 4, 6, True)])
def test_torch_path_matches_the_oracle(shape, D, F, bias, act, dtype, tol):
    x, wg, wu, bg, bu, gy = _inputs(shape, D, F, dtype, bias)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    y = gated.gated_feed_forward(x, wg, wu, bg, bu, activation=act)
    want, grads, _ = feed_oracle.feed(x.reshape(-1, D), wg, wu, bg, bu, act, gy.reshape(-1, F))
    assert y.dtype == dtype and y.shape == (*shape, F) and _rel(y.reshape(-1, F), want) < tol
    if dtype == F64:
        for got, g in zip(torch.autograd.grad(y, leaves, gy), grads if bias else grads[:3]):
            assert _rel(got, g.reshape(got.shape)) < tol


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_oracle_gradients_agree_with_differences(act):
    *args, gy = _inputs((3,), 4, 5)
    grads = feed_oracle.feed(*args, act, gy)[1]
    d = 1e-6
    for n, t in enumerate(args):
        for at in (0, t.numel() // 2, t.numel() - 1):
            step = torch.zeros(t.numel(), dtype=F64)
            step[at] = d
            up, down = ([a if i != n else a + s * step.view(t.shape) for i, a in enumerate(args)] for s in (1, -1))
            want = float(((feed_oracle.feed(*up, act) - feed_oracle.feed(*down, act)) * gy).sum()) / (2 * d)
            assert abs(want - float(grads[n].flatten()[at])) < 1e-6 * max(1.0, abs(want))


def test_refusals():
    x, wg, wu, bg, bu, _ = _inputs((2,), 4, 6, F32)
    f = gated.gated_feed_forward
    with pytest.raises(ValueError, match="activation"):
        f(x, wg, wu, activation="tanh")
    for bad in (dict(x=x[:, :3]), dict(weight_up=wu[:5]), dict(weight_gate=wg[0]), dict(weight_gate=wg[:0], weight_up=wu[:0]), dict(bias_gate=bg[:5]),
                dict(bias_up=bu[None]), dict(x=x.double()), dict(weight_up=wu.bfloat16()), dict(bias_up=bu.double()), dict(x=x[0, 0])):
        with pytest.raises(ValueError):
            f(**{**dict(x=x, weight_gate=wg, weight_up=wu, bias_gate=bg, bias_up=bu), **bad})


def test_backend_declines_what_it_cannot_serve():
    x, wg, wu, bg, bu, _ = _inputs((2,), 4, 6, F32)
    assert "GPU-only" in feed_hip.supports(x, wg, wu, bg, bu)
    with pytest.raises(TypeError):
        feed_hip._screen(x, wg)


def test_sizes_that_python_repeats():
    lib = _lib.load()
    for dtype, io in feed_hip._IO_DTYPES.items():
        for rows, F in ((0, 5), (1, 1), (17, 33), (4096, 1000)):
            assert lib.tsfast_hip_feed_kept_bytes(rows, 64, F, io) == feed_hip.kept_bytes(rows, F, dtype)
    assert lib.tsfast_hip_feed_kept_bytes(1, feed_hip._MAX_WIDTH, 1, 0) > 0
    assert lib.tsfast_hip_feed_kept_bytes(1, feed_hip._MAX_WIDTH + 1, 1, 0) == -1
    assert lib.tsfast_hip_feed_kept_bytes((1 << 31) - 63, 1, 1, 0) == -1


def test_abi_refuses_before_any_launch():
    """Sizes, strides and missing tensors are refused on the host; an aligned bfloat16 call needs no workspace forward."""
    lib = _lib.load()
    p = 1 << 20  # an address that is never read
    size = lib.tsfast_hip_feed_fwd_workspace_bytes
    assert size(100, 64, 32, 1, p, 64, p, 64, p, 64, 0) == 0
    assert size(100, 64, 32, 1, p + 2, 64, p, 64, p, 64, 0) >= 100 * 64 * 2  # x is packed
    assert size(100, 64, 32, 1, p, 64, p, 64, p, 72, 0) >= 2 * 32 * 64 * 2  # the weights' rows are not equally far apart
    assert size(100, 63, 32, 0, p, 63, p, 63, p, 63, 0) >= 3 * 2 * 64 * (100 + 2 * 32)
    for few, io in zip(feed_hip._FEW_ROWS.values(), (0, 1)):  # few rows are read as they lie
        where = (p, 63, p, 63, p, 63)
        assert size(few, 63, 32, io, *where, 0) == 0 < min(size(few, 63, 32, io, *where, 1), size(few + 1, 63, 32, io, *where, 0))
    fwd = lambda rows=4, D=8, F=8, io=1, act=0, x=p, sx=8: lib.tsfast_hip_feed_fwd(  # noqa: E731
        rows, D, F, io, act, x, sx, p, 8, p, 8, None, None, p, None, None, 0, None)
    assert fwd(rows=-1) == fwd(D=0) == fwd(io=2) == fwd(act=3) == fwd(x=None) == fwd(sx=7) == fwd(sx=(1 << 22) + 1) == -1
    assert fwd(D=(1 << 20) + 1) == -3 and fwd(rows=0) == 0
    back = lib.tsfast_hip_feed_bwd_workspace_bytes
    assert back(0, 8, 8, 0, None, 8, None, 8, None, 8) == 0 < back(1, 8, 8, 0, p, 8, p, 8, p, 8)
    for rows, D, F in ((1, 1, 1), (1, 1 << 20, 1), (1, 1, 1 << 20), (33, 1 << 16, 1 << 16), (1 << 24, 1, 1), (1000, 768, 2048), (100_000, 64, 256)):
        for io in (0, 1):
            assert back(rows, D, F, io, p, D, p, D, p, D) > 0
    assert lib.tsfast_hip_feed_fwd(100, 8, 8, 0, 0, p, 8, p, 8, p, 8, None, None, p, None, None, 0, None) == -2
    bwd = lambda kept=p, gw=p, ws=p, n=0: lib.tsfast_hip_feed_bwd(  # noqa: E731
        4, 8, 8, 1, 0, p, 8, p, 8, p, 8, p, 8, kept, p, gw, p, None, None, ws, n, None)
    assert bwd(kept=None) == bwd(gw=None) == -1 and bwd() == bwd(ws=None) == -2
