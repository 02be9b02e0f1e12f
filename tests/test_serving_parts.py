"""The three bfloat16 parts of a token's float32 factors beside bfloat16 parameters, emulated in float64: the GPU's bar on a new state's norm
(1.2e-6, ``test_gpu_serving_paths``) shows the loss of any part of u, and of dt's first two (softplus lets through too little of the third)."""

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_feed_parts import parts
from tests.test_serving import BF, F32, make


def _state(m, kept_u, kept_dt):
    """The new state from a zero one, with those parts of u and of dt in the products with the parameters."""
    N, R = m["A"].shape[1], m["proj"]["dt_proj"].shape[1]
    xp, dp, db = (m["proj"][k].to(BF).double() for k in ("x_proj", "dt_proj", "dt_bias"))
    window = torch.cat((m["token"]["conv_state"], m["token"]["x"][..., None]), -1).double()
    u = O._silu((window * m["conv"]["weight"].to(BF).double()[:, 0]).sum(-1) + m["conv"]["bias"].to(BF).double())
    p = sum(parts(u.float())[i] for i in kept_u) @ xp.T
    delta = torch.nn.functional.softplus(sum(parts(p[:, :R].float())[i] for i in kept_dt) @ dp.T + db)
    return (delta * u)[..., None] * p[:, None, R : R + N]


@pytest.mark.parametrize("B,D,N,R", [(1, 128, 16, 8), (40, 200, 16, 40), (7, 1100, 24, 69), (64, 1536, 16, 96)])
def test_the_bar_shows_every_part(B, D, N, R):
    m = make(1, D, N, 4, R, B, F32, seed=3)
    m["proj"]["dt_bias"].add_(4.0)
    every = (0, 1, 2)
    want = _state(m, every, every)
    off = lambda *kept: float((_state(m, *kept) - want).norm() / want.norm())  # noqa: E731
    for dropped in every:
        rest = [i for i in every if i != dropped]
        assert off(rest, every) > 1.2e-6, ("u", dropped)
        if dropped < 2:
            assert off(every, rest) > 1.2e-6, ("dt", dropped)
