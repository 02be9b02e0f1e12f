"""The fused feed-forward block on the GPU: values that are not finite go where the definition in float64 takes them."""

import pytest
import torch

from oracle import feed_oracle
from tests.test_gpu_feed import BF, F32, _inputs
from tsfast_amd import gated

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _all(x, wg, wu, bg, bu, gy, act):
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    y = gated.gated_feed_forward(*leaves, activation=act)
    with torch.no_grad():
        served = gated.gated_feed_forward(x, wg, wu, bg, bu, activation=act)
    return dict(served=served, y=y.detach(), **dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), torch.autograd.grad(y, leaves, gy))))


def _want(x, wg, wu, bg, bu, gy, act):
    y, grads, _ = feed_oracle.feed(x, wg, wu, bg, bu, act, gy)
    return dict(served=y, y=y, **dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), grads)))


def _alike(got, want, what):
    """Infinities with their signs and NaN at the same places."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    at = want.isinf() | got.isinf()
    assert torch.equal(got[at], want[at]), what
    assert (got.isfinite() == want.isfinite()).all(), what


@pytest.mark.parametrize("dtype", [BF])
@pytest.mark.parametrize("rows", [20, 70, 1000])
def test_rows_that_do_not_exist_are_in_no_sum(gpu, rows, dtype):
    """A gate that is open or closed for good by an infinite weight has no gradient (d sigmoid = 0): the last 16 rows' missing ones, 0 times
    that weight, are no NaN in the bias's."""
    t = _inputs((rows,), 24, 40, dtype, True, seed=3)
    t[1][0, 0], t[1][39, 23] = INF, -INF
    got, want = _all(*t, "sigmoid"), _want(*t, "sigmoid")
    for n in ("served", "y", "dwu", "dbg", "dbu"):
        _alike(got[n], want[n], n)
    assert want["dbg"][0] == 0 and want["dbg"][39] == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_a_large_gradient_at_a_closed_gate(gpu, act, dtype):
    """dy b is beyond float32 where the gate's derivative is zero: no NaN, and float32's part of the magnitudes in the biases' gradients. An act(a)
    or act'(a) below 2^-126, float32's least, may be zero there (silu(-150) is -1e-63): off by up to |dy| 2^-126 in db, and |b| times it in da."""
    x, wg, wu, bg, bu, gy = _inputs((70,), 16, 24, dtype, True, seed=6)
    wg.zero_(), wu.zero_(), gy.zero_()
    bg[2], bu[2], gy[3, 2] = 30.0 if act == "sigmoid" else -150.0, 64.0, 2.0**127
    got = _all(x, wg, wu, bg, bu, gy, act)
    _, wants, _ = feed_oracle.feed(x, wg, wu, bg, bu, act, gy)
    reaches = feed_oracle.reach(x, wg, wu, bg, bu, act, gy)[1]
    for n, i in (("dbg", 3), ("dbu", 4)):
        assert torch.isfinite(got[n]).all(), n
        assert ((got[n].double() - wants[i]).abs() <= 1e-5 * reaches[i] + 2.0**-8 * wants[i].abs() + 2.0**127 * 2.0**-126 * 64).all(), n
    assert torch.isfinite(got["dx"]).all()
