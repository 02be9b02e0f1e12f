"""Packed prompts and single tokens of a Mamba layer on the GPU against float64.

Bars, against the largest value: float32 to the package's 1e-5 (the steps' rounding decays with the state; sums of up to 64 states and, in the
step, of up to 2048 products in float32 matrix sums), states likewise; bfloat16 outputs half a step of each value (2^-8) and that."""

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_serving import BF, F32, make
from tsfast_amd import mamba
from tsfast_amd.mamba import packed_hip

pytestmark = pytest.mark.gpu


def near(got, want, what):
    got, want = got.detach().double().cpu(), want.cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    if want.numel():
        half = 2.0**-8 if what.endswith("bf16") else 2.0**-24
        err = (got - want).abs() - half * want.abs() - 1e-5 * want.abs().max()
        assert (err <= 0).all(), f"{what}: {float((got - want).abs().max() / want.abs().max()):.2e}"


def tag(what, dtype):
    return what + (" bf16" if dtype == BF else "")


def check_packed(m, starts, carried, dtype, wide=torch.int32):
    at = torch.tensor(starts, dtype=wide, device="cuda")
    tails, h0 = m["state"](len(starts) - 1) if carried else (None, None)
    s = m["seq"]
    u, left = mamba.mamba_conv_packed(s["x"], at, **m["conv"], tails=tails)
    wu, wleft = O.conv_packed(s["x"], at, **m["conv"], tails=tails)
    near(u, wu, tag("u", dtype))
    assert torch.equal(left.double(), wleft)
    args = (s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, h0)
    y, last = mamba.mamba_ssm_packed(*args)
    wy, wlast = O.ssm_packed(*args)
    near(y, wy, tag("y", dtype))
    near(last, wlast, "last")
    for t in (u, y):
        assert not t[starts[-1] :].any() and not t[: starts[0]].any()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("carried", [False, True])
@pytest.mark.parametrize(
    "T,starts", [(0, [0]), (0, [0, 0, 0]), (5, [0]), (1, [0, 1]), (5, [0, 0, 5]), (43, [0, 7, 7, 8, 30, 30]), (43, [3, 9, 20]), (64, [0, 16, 32, 48, 64]), (70, [0, 1, 2, 3, 35, 70])]
)
@pytest.mark.parametrize("D,N,K", [(5, 3, 4), (64, 16, 4), (130, 20, 2)])
def test_packed_small(gpu, T, starts, D, N, K, carried, dtype):
    check_packed(make(T, D, N, K, 2, 1, dtype, dev="cuda"), starts, carried, dtype, torch.int64 if carried else torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N", [1, 4, 8, 32, 33, 64])
@pytest.mark.parametrize("K", [3, 8])
def test_packed_states_and_taps(gpu, N, K, dtype):
    check_packed(make(50, 24, N, K, 2, 1, dtype, dev="cuda"), [0, 2, 30, 50], True, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("starts", [[0, 1400], [0, 256, 512, 1400], [0, 100, 255, 257, 700, 700, 769, 1300], [600, 601, 1399], [0, 0, 512, 1024, 1024, 1280]])
def test_packed_segments(gpu, starts, dtype):
    """Rows that are cut into segments: sequences that begin and end at, before and behind the cuts, and lie across several."""
    check_packed(make(1400, 72, 16, 4, 2, 1, dtype, dev="cuda", seed=2), starts, True, dtype)
    assert packed_hip._lib.load().tsfast_hip_mamba_packed_workspace_bytes(1400, len(starts) - 1, 72, 16) > 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize(
    "B,D,N,K,R,bias", [(1, 1, 1, 2, 1, False), (1, 128, 16, 4, 8, True), (3, 7, 5, 4, 2, True), (4, 64, 16, 4, 4, False), (17, 130, 33, 3, 9, True), (33, 200, 64, 8, 40, True), (5, 1100, 16, 4, 69, True)]
)
def test_step(gpu, B, D, N, K, R, bias, dtype):
    m = make(1, D, N, K, R, B, dtype, dev="cuda")
    t, p = m["token"], m["proj"]
    conv = dict(conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"] if bias else None)
    if not bias:
        p["dt_bias"] = None
    for _ in range(2):  # the second one from the states of the first
        want = O.step(**t, **conv, **p, A=m["A"], Dp=m["Dp"])
        out = mamba.mamba_step(**t, **conv, **p, A=m["A"], Dp=m["Dp"])
        near(out, want[0], tag("out", dtype))
        assert torch.equal(t["conv_state"].double(), want[1])
        near(t["ssm_state"], want[2], "h")
