"""A Mamba layer in service without a GPU: the torch path against the float64 oracle and against the equal-length operators,
refusals, and the limits that Python repeats.

Bars: float64 to 1e-11 of the largest value; float32 to the package's 1e-5 (sums of at most 60 products and states of at most 40 steps, 100 x 2^-24 =
6e-6 in the worst case); bfloat16 half a step more (2^-8)."""

import pytest
import torch

from oracle import serving_oracle as O
from tsfast_amd import _lib, mamba
from tsfast_amd.mamba import core, packed_hip

F64, F32, BF = torch.float64, torch.float32, torch.bfloat16
TOLS = [(F64, 1e-11), (F32, 1e-5), (BF, 2.0**-8 + 1e-5)]
STARTS = [[0, 0], [0, 1], [0, 7, 7, 8, 30, 30], [3, 9, 20], [0, 40], [0], [0, 0, 0, 5]]


def make(T, D, N, K, R, B, dtype, seed=0, dev="cpu"):
    """Inputs of all three operators, in the values that a layer meets."""
    r = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, device=dev, dtype=F64)  # noqa: E731
    wide = F64 if dtype == F64 else F32
    rates = -torch.arange(1, N + 1, device=dev, dtype=F64) * (0.5 + torch.rand(D, 1, generator=r, device=dev, dtype=F64))
    return dict(
        seq={k: v.to(dtype) for k, v in dict(x=n(T, D), draw=n(T, D) - 3, B_t=n(T, N), C_t=n(T, N), u=n(T, D), z=n(T, D)).items()},
        conv=dict(weight=(n(D, 1, K) / K**0.5).to(dtype), bias=n(D).to(dtype)),
        A=rates.to(wide), Dp=n(D).to(wide),
        token=dict(x=n(B, D).to(dtype), z=n(B, D).to(dtype), conv_state=n(B, D, K - 1).to(dtype), ssm_state=n(B, D, N).to(wide)),
        proj=dict(x_proj=(n(R + 2 * N, D) / D**0.5).to(dtype), dt_proj=(n(D, R) / R**0.5).to(dtype), dt_bias=(n(D) - 3).to(wide)),
        state=lambda S: (n(S, D, K - 1).to(dtype), n(S, D, N).to(wide)),
    )


def rel(a, b):
    return float((a.detach().double() - b).abs().max() / b.abs().max().clamp_min(1e-30)) if b.numel() else 0.0


@pytest.mark.parametrize("dtype,tol", TOLS)
@pytest.mark.parametrize("starts", STARTS)
@pytest.mark.parametrize("carried", [False, True])
def test_packed_matches_the_oracle(starts, carried, dtype, tol):
    T, D, N, K = 43, 5, 3, 4
    m = make(T, D, N, K, 2, 1, dtype)
    at = torch.tensor(starts, dtype=torch.int32 if carried else torch.int64)
    tails, h0 = m["state"](len(starts) - 1) if carried else (None, None)
    s = m["seq"]
    got = mamba.mamba_conv_packed(s["x"], at, **m["conv"], tails=tails)
    for g, w in zip(got, O.conv_packed(s["x"], at, **m["conv"], tails=tails)):
        assert g.dtype == dtype and g.shape == w.shape and rel(g, w) <= tol
    args = (s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, h0)
    (y, last), (wy, wlast) = mamba.mamba_ssm_packed(*args), O.ssm_packed(*args)
    assert y.dtype == dtype and last.dtype == m["A"].dtype and rel(y, wy) <= tol and rel(last, wlast) <= min(tol, 1e-5)
    assert not y[starts[-1] :].any() and not y[: starts[0]].any()


@pytest.mark.parametrize("dtype,tol", TOLS)
@pytest.mark.parametrize("B,D,N,K,R,bias", [(1, 1, 1, 2, 1, False), (3, 7, 5, 4, 2, True), (0, 4, 2, 3, 1, True)])
def test_step_matches_the_oracle(B, D, N, K, R, bias, dtype, tol):
    m = make(1, D, N, K, R, B, dtype)
    t, p = m["token"], m["proj"]
    conv = dict(conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"] if bias else None)
    if not bias:
        p["dt_bias"] = None
    want = O.step(**t, **conv, **p, A=m["A"], Dp=m["Dp"])
    states = t["conv_state"], t["ssm_state"]
    out = mamba.mamba_step(**t, **conv, **p, A=m["A"], Dp=m["Dp"])
    assert out.dtype == dtype and rel(out, want[0]) <= tol
    assert torch.equal(states[0].double(), want[1]) and rel(states[1], want[2]) <= min(tol, 1e-5)


def test_prompt_then_steps_is_the_whole_sequence():
    """Packed prompts, then tokens: what mamba_conv and mamba_ssm give over the whole sequences, in float64 to 1e-11."""
    D, N, K, R, lengths, more = 6, 4, 4, 2, (5, 0, 9), 3
    m = make(sum(lengths) + len(lengths) * more, D, N, K, R, len(lengths), F64, seed=1)
    conv, p, A, Dp = m["conv"], m["proj"], m["A"], m["Dp"]
    whole_x, whole_z = ([t[i : i + n + more] for i, n in zip((0, 8, 11), lengths)] for t in (m["seq"]["x"], m["seq"]["z"]))

    def projections(u):
        dt, b, c = (u @ p["x_proj"].T).split([R, N, N], -1)
        return dt @ p["dt_proj"].T + p["dt_bias"], b, c

    want = []
    for x, z in zip(whole_x, whole_z):
        u = core.mamba_conv(x[None], x.new_zeros(1, D, K - 1), conv["weight"], conv["bias"])
        draw, b, c = projections(u)
        want.append(core.mamba_ssm(draw, A, b, c, u, z[None], Dp)[0][0])
    x, z = (torch.cat([t[:n] for t, n in zip(ts, lengths)]) for ts in (whole_x, whole_z))
    starts = torch.tensor([0, 5, 5, 14])
    u, conv_state = mamba.mamba_conv_packed(x, starts, conv["weight"], conv["bias"])
    draw, b, c = projections(u)
    y, ssm_state = mamba.mamba_ssm_packed(draw, A, b, c, u, z, Dp, starts)
    got = [[y[a:e]] for a, e in zip(starts[:-1], starts[1:])]
    for i in range(more):
        xi, zi = (torch.stack([t[n + i] for t, n in zip(ts, lengths)]) for ts in (whole_x, whole_z))
        out = mamba.mamba_step(xi, zi, conv_state, ssm_state, conv["weight"], conv["bias"], **p, A=A, Dp=Dp)
        for s, o in zip(got, out):
            s.append(o[None])
    for g, w in zip(got, want):
        assert rel(torch.cat(g), w) < 1e-11


def test_refusals():
    m = make(10, 4, 3, 4, 2, 2, F32)
    s, conv, at = m["seq"], m["conv"], torch.tensor([0, 4, 10])
    for bad in ([0, 5, 4], [0, 11], [-1, 3], [2, 1]):
        with pytest.raises(ValueError, match="starts"):
            mamba.mamba_conv_packed(s["x"], torch.tensor(bad), **conv)
        with pytest.raises(ValueError, match="starts"):
            mamba.mamba_ssm_packed(s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], torch.tensor(bad))
    tails, h0 = m["state"](2)
    for bad in (dict(x=s["x"][None]), dict(starts=at[None]), dict(starts=at.float()), dict(starts=at[:0]), dict(weight=conv["weight"][:, 0]),
                dict(weight=conv["weight"][..., :1]), dict(bias=conv["bias"][:3]), dict(tails=tails[:1]), dict(tails=tails.double())):
        with pytest.raises(ValueError):
            mamba.mamba_conv_packed(**{**dict(x=s["x"], starts=at, **conv, tails=tails), **bad})
    good = dict(draw=s["draw"], A=m["A"], B_t=s["B_t"], C_t=s["C_t"], u=s["u"], z=s["z"], Dp=m["Dp"], starts=at, h0=h0)
    for bad in (dict(draw=s["draw"][0]), dict(A=m["A"][:, :0]), dict(A=m["A"].double()), dict(B_t=s["B_t"][:, :2]), dict(u=s["u"][:5]), dict(z=s["z"].bfloat16()),
                dict(Dp=m["Dp"][:2]), dict(h0=h0[:1]), dict(h0=h0.bfloat16()), dict(starts=at.to(torch.int16))):
        with pytest.raises(ValueError):
            mamba.mamba_ssm_packed(**{**good, **bad})
    t, p = m["token"], m["proj"]
    step = dict(**t, conv_weight=conv["weight"], conv_bias=conv["bias"], **p, A=m["A"], Dp=m["Dp"])
    for bad in (dict(x=t["x"][0]), dict(z=t["z"][:1]), dict(z=t["z"].double()), dict(conv_state=t["conv_state"][..., :2]), dict(ssm_state=t["ssm_state"].bfloat16()),
                dict(x_proj=p["x_proj"][:-1]), dict(x_proj=p["x_proj"].double()), dict(dt_proj=p["dt_proj"][:, :0]), dict(dt_bias=p["dt_bias"][:1]), dict(A=m["A"][:2])):
        with pytest.raises(ValueError):
            mamba.mamba_step(**{**step, **bad})


@pytest.mark.parametrize("which", ["conv", "ssm", "step"])
def test_no_gradient(which):
    m = make(6, 4, 3, 4, 2, 2, F32)
    s, conv, at, p = m["seq"], m["conv"], torch.tensor([0, 6]), m["proj"]
    calls = dict(
        conv=lambda: mamba.mamba_conv_packed(s["x"], at, conv["weight"].requires_grad_(), conv["bias"]),
        ssm=lambda: mamba.mamba_ssm_packed(s["draw"], m["A"].requires_grad_(), s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at),
        step=lambda: mamba.mamba_step(**m["token"], conv_weight=conv["weight"], conv_bias=conv["bias"], x_proj=p["x_proj"].requires_grad_(),
                                      dt_proj=p["dt_proj"], dt_bias=p["dt_bias"], A=m["A"], Dp=m["Dp"]),
    )
    with pytest.raises(RuntimeError, match="no gradient"):
        calls[which]()
    with torch.no_grad():
        calls[which]()


def test_backend_declines_what_it_cannot_serve():
    m = make(6, 4, 3, 4, 2, 2, F32)
    s, at = m["seq"], torch.tensor([0, 6])
    assert "GPU-only" in packed_hip.supports_conv(s["x"], at, *m["conv"].values(), None)
    assert "GPU-only" in packed_hip.supports_ssm(s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, None)
    assert "GPU-only" in packed_hip.supports_step(**m["token"], conv_weight=m["conv"]["weight"], conv_bias=None, **m["proj"], A=m["A"], Dp=m["Dp"])


def test_abi_refuses_before_any_launch():
    lib = _lib.load()
    p = 1 << 20  # an address that is never read
    conv = lambda T=4, S=1, D=8, K=4, io=1, x=p, sx=8, starts=p, w=p, out=p, left=p: lib.tsfast_hip_conv_packed(  # noqa: E731
        T, S, D, K, io, 0, 0, 0, x, sx, starts, None, w, None, out, left, None)
    assert conv(T=-1) == conv(K=1) == conv(io=2) == conv(x=None) == conv(sx=-1) == conv(starts=None) == conv(w=None) == conv(left=None) == -1
    assert conv(K=9) == conv(D=(1 << 24) + 1) == conv(T=1 << 32, D=1 << 10) == -3 and conv(D=0) == conv(T=0, S=0) == 0
    size = lib.tsfast_hip_mamba_packed_workspace_bytes
    assert size(77, 1, 128, 16) == 0 < size(65536, 1, 256, 16) and size(10, 1, 8, 65) == -1 and size(0, 3, 8, 4) == 0
    scan = lambda T=4, S=1, D=8, N=4, io=1, sz=8, A=p, draw=p, last=p, ws=None, n=0: lib.tsfast_hip_mamba_packed(  # noqa: E731
        T, S, D, N, io, 0, draw, 8, A, p, 4, p, 4, p, 8, p, sz, p, p, None, p, last, ws, n, None)
    assert scan(N=0) == scan(io=3) == scan(sz=-1) == scan(A=None) == scan(draw=None) == scan(last=None) == -1
    assert scan(N=65) == -3 and scan(D=0) == 0 and scan(T=65536, D=256, N=16) == -2 == scan(T=65536, D=256, N=16, ws=p, n=100)
    step = lambda B=2, D=8, N=4, R=2, K=4, io=0, pt=0, bt=0, x=p, h=p, ws=p, n=0: lib.tsfast_hip_mamba_step(  # noqa: E731
        B, D, N, R, K, io, pt, bt, x, 8, p, 8, p, h, p, None, p, p, None, p, p, p, ws, n, None)
    assert step(B=-1) == step(R=0) == step(K=1) == step(io=2) == step(pt=2) == step(bt=-1) == step(x=None) == step(h=None) == -1
    assert step(K=9) == step(N=65) == step(R=1017) == -3 and step(B=0) == 0 and step() == step(ws=None, n=1 << 20) == -2
    assert lib.tsfast_hip_mamba_step_workspace_bytes(2, 8, 4, 2, 4) >= 2 * 10 * 4
