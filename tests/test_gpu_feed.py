"""The fused gated feed-forward block on the GPU against float64.

Bars. Forward, bfloat16: sums are float32 and the result is rounded once, so an element is off by half a step (2^-8 of it)
and float32's part. Gradients, bfloat16: da and db are rounded once more, each by up to 2^-8 of itself, so an element is off by up to
2^-8 of the sum of its terms' magnitudes (and half a step of itself); as the roundings are independent, the whole gradient is off by
less than 2^-8 of its norm. Biases' gradients are sums of unrounded values. float32: a sum of n products is off by up to
n 2^-24 of the sum of their magnitudes in the worst order and about sqrt(n) 2^-24 in the usual case; the pairs of bfloat16 parts
that are left out are below 2^-23 of a product; the activation adds about 3e-7 of its value: 1e-5 of the sum of the magnitudes covers n up to 65536."""

import pytest
import torch

from oracle import feed_oracle
from tsfast_amd import _lib, gated
from tsfast_amd.gated import feed_hip

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _inputs(shape, D, F, dtype, bias, seed=0, dev="cuda"):
    r = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, device=dev)  # noqa: E731
    x, wg, wu, gy = n(*shape, D).to(dtype), (n(F, D) / D**0.5).to(dtype), (n(F, D) / D**0.5).to(dtype), n(*shape, F).to(dtype)
    return x, wg, wu, *((n(F).to(dtype), n(F).to(dtype)) if bias else (None, None)), gy


def _near(got, want, sums, dtype, roundings, what):
    got, want = got.detach().double(), want.reshape(got.shape)
    sums = sums.reshape(got.shape)
    err = (got - want).abs()
    half = 2.0**-8 if dtype == BF else 2.0**-24
    bound = 1e-5 * sums + half * want.abs() + (half * sums if roundings > 1 else 0)
    assert torch.isfinite(got).all(), what
    assert (err <= bound + 1e-30).all(), f"{what}: {float((err / (bound + 1e-30)).max()):.2f} times the bound"
    if dtype == BF and roundings > 1 and want.numel() > 64:
        assert err.norm() <= half * want.norm(), f"{what}: {float(err.norm() / want.norm()):.2e}"


def _check(x, wg, wu, bg, bu, gy, act, dtype):
    D = x.shape[-1]
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    it = iter(leaves)
    lx, lg, lu, lbg, lbu = (None if t is None else next(it) for t in (x, wg, wu, bg, bu))
    with torch.no_grad():
        served = gated.gated_feed_forward(x, wg, wu, bg, bu, activation=act)
    y = gated.gated_feed_forward(lx, lg, lu, lbg, lbu, activation=act)
    grads = torch.autograd.grad(y, leaves, gy)
    want, wgrads, sums = feed_oracle.feed(x.reshape(-1, D), wg, wu, bg, bu, act, gy.reshape(-1, gy.shape[-1]))
    xa = x.reshape(-1, D).double().abs()
    # |b| (1 + |a|): what y's float32 part is relative to
    mag = (1 + xa @ wg.double().abs().T + (0 if bg is None else bg.double().abs())) * (xa @ wu.double().abs().T + (0 if bu is None else bu.double().abs()))
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], wg.shape[0])
    _near(served, want, mag, dtype, 1, "y")
    _near(y, want, mag, dtype, 1, "y of a training step")
    names = [n for n, t in zip(("dx", "dwg", "dwu", "dbg", "dbu"), (x, wg, wu, bg, bu)) if t is not None]
    by_name = dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), zip(wgrads, sums)))
    for n, g in zip(names, grads):
        assert g.dtype == dtype
        _near(g, *by_name[n], dtype, 1 if n in ("dbg", "dbu") else 2, n)
    return y, grads


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize(
    "rows,D,F,bias",
    [(1, 1, 1, True), (1, 8, 16, False), (5, 33, 47, True), (16, 64, 64, False), (17, 40, 130, True), (33, 195, 517, True), (64, 64, 32, False), (257, 96, 264, True)],
)
def test_small_sizes(gpu, rows, D, F, bias, act, dtype):
    _check(*_inputs((rows,), D, F, dtype, bias), act, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,D,F,bias", [(2050, 130, 700, True), (4096, 512, 1024, False), (20000, 64, 256, True), (1000, 1032, 2056, False), (700, 2048, 40, True)])
def test_larger_sizes(gpu, rows, D, F, bias, dtype):
    _check(*_inputs((rows,), D, F, dtype, bias, seed=1), "silu", dtype)
