"""A Mamba layer in service on the GPU: values that are not finite go where the definition takes them, and no further."""

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_serving import BF, F32, make
from tsfast_amd import mamba

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def scan(m, at, h0=None, **other):
    s = {**m["seq"], **other}
    return mamba.mamba_ssm_packed(s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, h0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N", [3, 16, 40])
@pytest.mark.parametrize("starts,t", [([0, 60], 0), ([0, 60], 59), ([3, 30, 900, 1100], 35), ([3, 30, 900, 1100], 899), ([0, 2000], 700)])
def test_a_nan_step_size_stays_in_its_sequence_and_channel(gpu, starts, t, N, dtype):
    """softplus of NaN is NaN, so from that token on the channel's outputs and last state are, in short rows and in rows cut into segments; all
    others keep their bits."""
    m = make(starts[-1] + 7, 70, N, 4, 2, 1, dtype, dev="cuda", seed=1)
    at, d = torch.tensor(starts, device="cuda"), 65
    h0 = m["state"](len(starts) - 1)[1]
    want, want_last = scan(m, at, h0)
    draw = m["seq"]["draw"].clone()
    draw[t, d] = NAN
    y, last = scan(m, at, h0, draw=draw)
    s = next(i for i, e in enumerate(starts[1:]) if t < e)
    assert y[t : starts[s + 1], d].isnan().all() and last[s, d].isnan().all()
    y[t : starts[s + 1], d] = want[t : starts[s + 1], d]
    last[s, d] = want_last[s, d]
    assert torch.equal(y, want) and torch.equal(last, want_last)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_nan_step_bias_shows_in_its_channel(gpu, dtype):
    m = make(1, 70, 16, 4, 5, 9, dtype, dev="cuda", seed=2)
    weights = dict(conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"], **m["proj"], A=m["A"], Dp=m["Dp"])

    def step(**other):
        token = {k: t.clone() for k, t in m["token"].items()}
        return mamba.mamba_step(**token, **{**weights, **other}), token["ssm_state"]

    want, want_h = step()
    bias = weights["dt_bias"].clone()
    bias[33] = NAN
    y, h = step(dt_bias=bias)
    assert y[:, 33].isnan().all() and h[:, 33].isnan().all()
    y[:, 33], h[:, 33] = want[:, 33], want_h[:, 33]
    assert torch.equal(y, want) and torch.equal(h, want_h)


def _alike(got, want):
    """Infinities with their signs and NaN at the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    at = want.isinf()
    assert torch.equal(got.isinf(), at) and torch.equal(got[at], want[at])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N", [1, 2, 3, 5, 16, 17])
@pytest.mark.parametrize("starts,t", [([0, 20], 7), ([2, 30, 900, 1100], 40)])
def test_an_infinite_step_size_makes_states_infinite(gpu, starts, t, N, dtype):
    """The states that a wave has beyond N take no part: with an infinite delta 0 times it, NaN, would be among the sums."""
    m = make(starts[-1] + 7, 70, N, 4, 2, 1, dtype, dev="cuda", seed=3)
    at = torch.tensor(starts, device="cuda")
    m["seq"]["draw"][t, 3] = INF
    s = m["seq"]
    got, want = scan(m, at), O.ssm_packed(s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at)
    assert want[1].isinf().any()
    for g, w in zip(got, want):
        _alike(g, w)


def _step_both(m):
    weights = dict(conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"], **m["proj"], A=m["A"], Dp=m["Dp"])
    y, tail, h = O.step(**m["token"], **weights)
    got = mamba.mamba_step(**m["token"], **weights)
    return (got, m["token"]["ssm_state"]), (y, h)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("B,D,N,R", [(1, 5, 1, 1), (20, 70, 1, 1), (9, 130, 4, 1), (5, 300, 16, 3)])
def test_a_step_from_values_that_are_not_finite(gpu, B, D, N, R, value, dtype):
    """Infinities with their signs and NaN where float64 has them, in the row with such an input; other rows keep their bits."""
    m, plain = (make(1, D, N, 4, R, B, dtype, dev="cuda", seed=3) for _ in range(2))
    b, d = B // 2, D - 1
    for t in (m, plain):  # u of this channel is +inf, not silu(-inf), which is NaN
        t["conv"]["weight"][d, 0].abs_()
    m["token"]["x"][b, d] = value
    (want_y, want_h), _ = _step_both(plain)
    got, want = _step_both(m)
    for g, w, other in zip(got, want, (want_y, want_h)):
        _alike(g[b], w[b])
        rest = torch.arange(B, device="cuda") != b
        assert torch.equal(g[rest], other[rest])


@pytest.mark.parametrize("sign", [1, -1])
def test_a_step_from_u_above_bfloat16s_largest(gpu, sign):
    """u = 3.4e38 between float32's and bfloat16's largest: what x_proj makes of it, and with it the other channels, to the package's 1e-5 of the
    largest value."""
    m = make(1, 70, 16, 2, 3, 9, BF, dev="cuda", seed=4)
    m["proj"]["x_proj"].mul_(2.0**-60)
    m["proj"]["x_proj"][:, 5] = (m["proj"]["x_proj"][:, 5] * 2.0**60).sign() * 2.0**-126 * torch.linspace(0.5, 1.0, 35, device="cuda").to(BF)
    m["conv"]["weight"][5, 0] = torch.tensor([1.0, 1.9921875])
    m["conv"]["bias"][5] = 0.0
    m["token"]["x"][:, 5], m["token"]["conv_state"][:, 5, 0] = 2.0**127, 1e36
    m["proj"]["x_proj"][:, 5] *= sign
    (y, h), (want_y, want_h) = _step_both(m)
    keep = torch.arange(70, device="cuda") != 5
    assert want_h[:, keep].abs().max() > 1
    assert (h[:, keep].double() - want_h.to("cuda")[:, keep]).abs().max() <= 1e-5 * want_h[:, keep.to(want_h.device)].abs().max()
    assert torch.isfinite(y[:, keep]).all()
