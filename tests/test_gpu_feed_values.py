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
