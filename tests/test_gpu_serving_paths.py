"""A Mamba layer in service on the GPU against float64 where the sizes select the paths for much work: sixteen tokens of a thread in the
convolution, segments with more than 16 states in the scan; and the accuracy of a token's products, part by part.

Bars: ``test_gpu_serving``'s (1e-5 of the largest value, bfloat16 half a step more)."""

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_gpu_serving import near, tag
from tests.test_serving import BF, F32, make
from tsfast_amd import _lib, mamba

pytestmark = pytest.mark.gpu


def _starts(T, S, seed):
    """S sequences in T tokens: of random lengths, among them empty ones and ones of 1 to 5 tokens; some tokens before and behind."""
    r = torch.Generator().manual_seed(seed)
    cuts = torch.randint(3, T - 9, (S + 1,), generator=r).sort().values
    for i, n in enumerate((0, 1, 2, 3, 5, 0, 0, 16)):
        if 3 * i + 2 <= S:
            cuts[3 * i + 2] = torch.minimum(cuts[3 * i + 1] + n, cuts[3 * i + 3] if 3 * i + 3 <= S else cuts[3 * i + 1] + n)
    return cuts.to(torch.int32).cuda()


@pytest.mark.parametrize("K", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("T,D,S", [(16401, 1536, 30), (16411, 1283, 100), (40009, 541, 26)])
def test_sixteen_tokens_of_a_thread(gpu, T, D, S, K):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-T // 16) * -(-D // 8) >= 640 * cus  # packed.hip launch_conv
    m = make(T, D, 1, K, 1, 1, BF, dev="cuda", seed=1)
    at = _starts(T, S, seed=K)
    for tails in (None, m["state"](S)[0]):
        u, left = mamba.mamba_conv_packed(m["seq"]["x"], at, **m["conv"], tails=tails)
        want, wleft = O.conv_packed(m["seq"]["x"], at, **m["conv"], tails=tails)
        near(u, want, tag("u", BF))
        assert torch.equal(left.double(), wleft)
        assert not u[: at[0]].any() and not u[at[-1] :].any()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N", [17, 31, 32, 33, 48, 64])
@pytest.mark.parametrize("starts", [[0, 1400], [2, 100, 355, 357, 700, 700, 769, 1300]])
def test_segments_with_many_states(gpu, starts, N, dtype):
    assert _lib.load().tsfast_hip_mamba_packed_workspace_bytes(1409, len(starts) - 1, 130, N) > 0  # in segments
    m = make(1409, 130, N, 4, 2, 1, dtype, dev="cuda", seed=2)
    at, s = torch.tensor(starts, device="cuda"), m["seq"]
    for h0 in (None, m["state"](len(starts) - 1)[1]):
        args = (s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, h0)
        (y, last), (want, wlast) = mamba.mamba_ssm_packed(*args), O.ssm_packed(*args)
        near(y, want, tag("y", dtype))
        near(last, wlast, "last")


@pytest.mark.parametrize("other", [F32, BF])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,D,N,R", [(1, 128, 16, 8), (40, 200, 16, 40), (7, 1100, 24, 69), (64, 1536, 16, 96)])
def test_a_tokens_products_in_every_part(gpu, B, D, N, R, dtype, other):
    """From a zero state and with steps of about 1, the new one is delta u B: as exact as B, delta and u are. Each is off by what float32 leaves, 2e-7 and
    2^-25 sqrt(n / 16) for a sum of n products (``test_gpu_feed_plans.sums``): 1.2e-6 of its norm together for n up to 1536. Without the third of
    the parts that a float32 factor has beside bfloat16 parameters, B and delta's argument are each off by 1.66e-3 squared, 2.7e-6."""
    m = make(1, D, N, 4, R, B, dtype, dev="cuda", seed=3)
    m["token"]["ssm_state"].zero_()
    m["proj"]["dt_bias"].add_(4.0)
    kw = dict(conv_weight=m["conv"]["weight"].to(other), conv_bias=m["conv"]["bias"].to(other), A=m["A"], Dp=m["Dp"])
    kw |= {k: v.to(other) for k, v in m["proj"].items()} | m["token"]
    want = O.step(**kw)[2]
    mamba.mamba_step(**kw)
    assert float((kw["ssm_state"].double() - want).norm() / want.norm()) <= 1.2e-6
