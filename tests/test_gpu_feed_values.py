"""The fused feed-forward block on the GPU: infinities, NaN and the largest values go where the definition in float64 takes them, whatever
kernel the number of rows selects."""

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


@pytest.mark.parametrize("dtype", [F32, BF])
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
@pytest.mark.parametrize("rows,D,F", [(20, 24, 40), (70, 24, 40), (70, 21, 39), (130, 2048, 33), (3000, 130, 260), (9000, 64, 520)])
@pytest.mark.parametrize("where", ["x", "wg", "wu", "bg", "gy", "x and wu"])
def test_infinities_and_nan(gpu, where, rows, D, F, act, dtype):
    t = dict(zip(("x", "wg", "wu", "bg", "bu", "gy"), _inputs((rows,), D, F, dtype, True, seed=3)))
    last = {n: tuple(s - 1 for s in v.shape) for n, v in t.items()}
    for n in where.split(" and "):
        t[n][(0,) * t[n].dim()] = INF
        t[n][last[n]] = -INF
        if where != "x and wu":
            t[n][tuple(s // 2 for s in t[n].shape)] = NAN
    got, want = _all(**t, act=act), _want(**t, act=act)
    for n in got:
        _alike(got[n], want[n], n)
    # what no such value reaches keeps its accuracy
    for n in ("served", "y", "dx", "dwg", "dwu", "dbg", "dbu"):
        ok = want[n].isfinite()
        if ok.any():
            err, size = (got[n].double() - want[n])[ok].norm(), want[n][ok].norm()
            assert err <= (1e-5 if dtype == F32 else 2.0**-7) * size, (n, float(err / size))


BIG = 3.402e38  # a float32 that rounds to no finite bfloat16


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows", [20, 70])
def test_values_above_bfloat16s_largest(gpu, rows, act):
    """What float32 holds of products with such a value it gives, to the package's 1e-5 of the magnitudes that are summed."""
    x, wg, wu, bg, bu, gy = _inputs((rows,), 16, 24, F32, True, seed=4)
    own = [3, 7, 9]
    x[own], x[:, 8] = 0.0, 0.0
    x[3, 5], x[7, 6], x[9, 8] = BIG, -BIG, 0.125
    wg.mul_(2.0**-100)
    wg[:, 5:7] = 2.0**-126
    wu[:, 5:7] = 0.0625 * wu[:, 5:7].sign()
    wu[5, 8] = -BIG
    t = (x, wg, wu, bg.clamp(-2, 2), bu)
    got, want = _all(*t, gy, act), feed_oracle.feed(*t, act)
    reach = feed_oracle.reach(*t, act, gy)[0]
    assert want[own].abs().max() > 1e37
    for n in ("served", "y"):
        assert torch.isfinite(got[n]).all(), n
        assert ((got[n].double() - want).abs()[own] <= 1e-5 * reach[own]).all(), n


def test_gradients_above_bfloat16s_largest(gpu):
    x, wg, wu, bg, bu, gy = _inputs((70,), 16, 24, F32, True, seed=5)
    wg.mul_(2.0**-100), wu.mul_(2.0**-100), x[3].mul_(0.1), gy.zero_()
    bg[2], gy[3, 2] = 20.0, BIG  # the gate is open: db = BIG
    got, want = _all(x, wg, wu, bg, bu, gy, "sigmoid"), _want(x, wg, wu, bg, bu, gy, "sigmoid")
    for n, at in (("dx", 3), ("dwu", 2), ("dbu", 2)):
        g, w = got[n][at].double(), want[n][at]
        assert w.abs().max() < 3.4028e38 and torch.isfinite(got[n]).all(), n
        assert ((g - w).abs() <= 1e-5 * w.abs().max()).all(), n


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


@pytest.mark.parametrize("rows", [50, 4000])
def test_gelus_tail(gpu, rows):
    """gelu keeps its accuracy where it is small. With D = F = 1, unit weights and b = 1 a is x exactly and y is act(a): its factors are off by 7e-8
    (the fit), 2^-22 (rcp and exp, one unit each, and the argument of t), 12 x 2^-24 at most (P's nine steps and three products): under 1.1e-6
    of the value. act' adds a phi'(a), which is off by as much of itself."""
    a = torch.linspace(-12.5, 6, rows, device="cuda")[:, None]
    one, none = torch.ones(1, 1, device="cuda"), torch.zeros(1, 1, device="cuda")
    t = (a, one, none, torch.zeros(1, device="cuda"), torch.ones(1, device="cuda"), torch.ones(rows, 1, device="cuda"))
    got, want = _all(*t, "gelu"), _want(*t, "gelu")
    for n in ("served", "y"):
        assert ((got[n].double() - want[n]).abs() <= 1.1e-6 * want[n].abs()).all(), n
    w = a.double()
    sizes = 0.5 * torch.special.erfc(-w / 2**0.5) + w.abs() * torch.exp(-w * w / 2) / (2 * torch.pi) ** 0.5
    assert ((got["dx"].double() - want["dx"]).abs() <= 1.1e-6 * sizes).all()
