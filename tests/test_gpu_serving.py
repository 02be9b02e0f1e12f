"""Packed prompts and single tokens of a Mamba layer on the GPU against float64.

Bars, against the largest value: float32 to the package's 1e-5 (the steps' rounding decays with the state; sums of up to 64 states and, in the
step, of up to 2048 products in float32 matrix sums), states likewise; bfloat16 outputs half a step of each value (2^-8) and that."""

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_serving import BF, F32, make
from tsfast_amd import gated, mamba
from tsfast_amd.mamba import core, packed_hip

pytestmark = pytest.mark.gpu


def near(got, want, what, roundings=1):
    got, want = got.detach().double().cpu(), want.cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    if want.numel():
        half = 2.0**-8 if what.endswith("bf16") else 2.0**-24
        err = (got - want).abs() - roundings * half * want.abs() - 1e-5 * want.abs().max()
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


@pytest.mark.parametrize("dtype", [F32, BF])
def test_runs_of_one_wave_in_and_before_a_sequence(gpu, dtype):
    """Few channels: a wave's lanes have tokens before, in and behind the sequences."""
    check_packed(make(500, 8, 4, 4, 2, 1, dtype, dev="cuda", seed=3), [110, 114, 250, 400], True, dtype)
    check_packed(make(500, 3, 4, 8, 2, 1, dtype, dev="cuda", seed=3), [129, 131, 131, 499], True, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("S", [62, 63, 64, 65, 300])
def test_many_sequences(gpu, S, dtype):
    """As many starts as a wave has lanes, and more; every fifth sequence is empty, most are shorter than a segment."""
    r = torch.Generator().manual_seed(S)
    lengths = torch.randint(1, 1500 // S + 2, (S,), generator=r)
    lengths[::5] = 0
    starts = [2, *(2 + lengths.cumsum(0)).tolist()]
    check_packed(make(starts[-1] + 3, 20, 5, 4, 2, 1, dtype, dev="cuda", seed=4), starts, True, dtype)
    check_packed(make(starts[-1] + 3, 20, 5, 4, 2, 1, dtype, dev="cuda", seed=4), starts, False, dtype, torch.int64)


def packed(m, at, tails=None, h0=None, **other):
    s = {**m["seq"], **other}
    u, left = mamba.mamba_conv_packed(s["x"], at, **m["conv"], tails=tails)
    y, last = mamba.mamba_ssm_packed(s["draw"], m["A"], s["B_t"], s["C_t"], s["u"], s["z"], m["Dp"], at, h0)
    return u, left, y, last


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b, strict=True))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_layouts(gpu, dtype):
    """Halves of a wider projection, at odd offsets, transposed or expanded, parameters as views: as dense tensors."""
    T, D, N = 300, 37, 5
    m = make(T, D, N, 4, 2, 1, dtype, dev="cuda", seed=5)
    at = torch.tensor([0, 100, 100, 290], device="cuda")
    tails, h0 = m["state"](3)
    want = packed(m, at, tails, h0)
    wide = torch.randn(T, 2 * D + 2 * N + 9, device="cuda").to(dtype)
    views, i = {}, 1
    for k in ("x", "z", "B_t", "C_t"):
        t = m["seq"][k]
        wide[:, i : i + t.shape[1]] = t
        views[k], i = wide[:, i : i + t.shape[1]], i + t.shape[1]
    turned = {k: m["seq"][k].t().contiguous().t() for k in ("draw", "u")}
    spaced = torch.stack((at, at - 7), 1)[:, 0]
    others = dict(m, A=m["A"].t().contiguous().t(), Dp=torch.stack((m["Dp"], m["Dp"]), 1)[:, 0], conv=dict(m["conv"], weight=m["conv"]["weight"].flip(-1).flip(-1).transpose(0, 2).contiguous().transpose(0, 2)))
    assert same(packed(others, spaced, tails.transpose(1, 2).contiguous().transpose(1, 2), h0.transpose(0, 1).contiguous().transpose(0, 1), **views, **turned), want)
    one = {k: m["seq"][k][:1].expand_as(m["seq"][k]) for k in ("x", "draw", "B_t", "C_t", "u", "z")}
    assert same(packed(m, at, tails, h0, **one), packed(m, at, tails, h0, **{k: t.contiguous() for k, t in one.items()}))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_nothing_of_other_tokens_gets_in(gpu, dtype):
    """NaN in the tokens before and behind the sequences and in another sequence: this one's results and states keep their bits."""
    starts = [5, 90, 600, 1100]
    at = torch.tensor(starts, device="cuda")
    m = make(1200, 70, 16, 4, 2, 1, dtype, dev="cuda", seed=6)
    tails, h0 = m["state"](3)
    want = packed(m, at, tails, h0)
    for own in range(3):
        hurt = {k: t.clone() for k, t in m["seq"].items()}
        for t in hurt.values():
            t[: starts[own]] = t[starts[own + 1] :] = float("nan")
        with_nan, h_nan = tails.clone(), h0.clone()
        for t in (with_nan, h_nan):
            t[:own] = t[own + 1 :] = float("nan")
        u, left, y, last = packed(m, at, with_nan, h_nan, **hurt)
        a, e = starts[own], starts[own + 1]
        assert same((u[a:e], left[own], y[a:e], last[own]), (want[0][a:e], want[1][own], want[2][a:e], want[3][own])), own
        assert not any(t[: starts[0]].any() or t[starts[-1] :].any() for t in (u, y))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_each_sequence_as_alone(gpu, dtype):
    """A row in segments against its sequences alone (cut elsewhere) and one after another with carried states: to float32 rounding."""
    starts = [0, 5000, 5003, 12000]
    at = torch.tensor(starts, device="cuda")
    m = make(starts[-1], 130, 16, 4, 2, 1, dtype, dev="cuda", seed=7)
    u, left, y, last = packed(m, at)
    for s, (a, e) in enumerate(zip(starts, starts[1:])):
        cut = (a + e) // 2
        tails = h0 = None
        for t0, t1 in ((a, cut), (cut, e)):
            part = packed(m, torch.tensor([0, t1 - t0], device="cuda"), tails, h0, **{k: t[t0:t1] for k, t in m["seq"].items()})
            assert torch.equal(part[0], u[t0:t1])
            near(part[2], y[t0:t1].double(), tag("y", dtype), 2)  # both are rounded
            tails, h0 = part[1], part[3]
        assert torch.equal(tails[0], left[s])
        near(h0[0], last[s].double(), "last")


def _step_args(m):
    return dict(**m["token"], conv_weight=m["conv"]["weight"], conv_bias=m["conv"]["bias"], **m["proj"], A=m["A"], Dp=m["Dp"])


def _near_step(kw, dtype, what):
    want = O.step(**kw)
    out = mamba.mamba_step(**kw)
    near(out, want[0], tag(what, dtype))
    assert torch.equal(kw["conv_state"].double(), want[1])
    near(kw["ssm_state"], want[2], what + " h")


@pytest.mark.parametrize("B,D,N,K,R", [(2, 33, 6, 5, 3), (9, 96, 16, 6, 130), (4, 300, 16, 7, 257), (70, 24, 3, 4, 11), (1, 2050, 64, 4, 800), (3, 8, 1, 2, 1)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_step_sizes(gpu, B, D, N, K, R, dtype):
    _near_step(_step_args(make(1, D, N, K, R, B, dtype, dev="cuda", seed=8)), dtype, "step")


def test_step_types_and_layouts(gpu):
    """Parameters in float32 or the sequence's type one by one; x and z as halves of a projection; parameters as views."""
    for n in range(16):
        kw = _step_args(make(1, 40, 16, 4, 5, 6, BF, dev="cuda", seed=9))
        for i, k in enumerate(("conv_weight", "conv_bias", "x_proj", "dt_proj")):
            if n >> i & 1:
                kw[k] = kw[k].float()
        if n & 1:
            kw["dt_bias"] = kw["dt_bias"].bfloat16()
        wide = torch.randn(6, 83, device="cuda").to(BF)
        wide[:, 1:41], wide[:, 43:] = kw["x"], kw["z"]
        kw["x"], kw["z"] = wide[:, 1:41], wide[:, 43:]
        for k in ("x_proj", "dt_proj", "A"):
            kw[k] = kw[k].t().contiguous().t()
        _near_step(kw, BF, f"types {n}")
    kw = _step_args(make(1, 40, 16, 4, 5, 6, F32, dev="cuda", seed=9))
    kw["ssm_state"] = kw["ssm_state"].transpose(1, 2).contiguous().transpose(1, 2)  # the torch path
    _near_step(kw, F32, "a turned state")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_repeats_streams_and_graphs(gpu, dtype):
    """Repeats, two streams at once, and two captured graphs in turn on new inputs give the same bits."""
    m, at = make(2000, 40, 16, 4, 6, 20, dtype, dev="cuda", seed=10), torch.tensor([0, 700, 1990], device="cuda")
    tails, h0 = m["state"](2)
    t = m["token"]
    states = t["conv_state"].clone(), t["ssm_state"].clone()

    def work(own):
        args = dict(_step_args(m), conv_state=own[0], ssm_state=own[1])
        own[0].copy_(states[0]), own[1].copy_(states[1])
        return *packed(m, at, tails, h0), mamba.mamba_step(**args), mamba.mamba_step(**args), *own

    own = lambda: tuple(s.clone() for s in states)  # noqa: E731
    want = work(own())
    for _ in range(3):
        assert same(work(own()), want)
    sides, got = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for side in sides * 2:
        with torch.cuda.stream(side):
            got.append(work(own()))
    torch.cuda.synchronize()
    assert all(same(g, want) for g in got)
    graphs = []
    for _ in range(2):
        mine, graph = own(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work(mine)))
    for seed, starts in ((1, [0, 0, 2000]), (2, [3, 1500, 1501]), (3, [0, 256, 512])):
        new = make(2000, 40, 16, 4, 6, 20, dtype, dev="cuda", seed=seed)
        for k, v in new["seq"].items():
            m["seq"][k].copy_(v)
        t["x"].copy_(new["token"]["x"])
        at.copy_(torch.tensor(starts))
        want = work(own())
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert same(outs, want), seed


def test_prompts_then_tokens_then_the_feed_forward(gpu):
    """A layer in service as it is used: packed prompts, then tokens one by one, each through the gated feed-forward block, against the
    training operators over the whole sequences (float32, to 1e-5 of the largest value, twice that behind the second block)."""
    D, N, K, R, lengths, more, F = 64, 16, 4, 4, (300, 0, 41), 4, 96
    S = len(lengths)
    m = make(sum(lengths) + S * more, D, N, K, R, S, F32, dev="cuda", seed=11)
    p, r = m["proj"], torch.Generator(device="cuda").manual_seed(12)
    wg, wu = (torch.randn(F, D, generator=r, device="cuda") / D**0.5 for _ in range(2))
    ends = [sum(lengths[: i + 1]) + (i + 1) * more for i in range(S)]
    whole = [(m["seq"]["x"][e - n - more : e], m["seq"]["z"][e - n - more : e]) for e, n in zip(ends, lengths)]

    def projections(u):
        dt, b, c = (u @ p["x_proj"].T).split([R, N, N], -1)
        return dt @ p["dt_proj"].T + p["dt_bias"], b, c

    want = []
    for x, z in whole:
        u = core.mamba_conv(x[None], x.new_zeros(1, D, K - 1), m["conv"]["weight"], m["conv"]["bias"])
        y, _ = core.mamba_ssm(projections(u)[0], m["A"], *projections(u)[1:], u, z[None], m["Dp"])
        want.append(gated.gated_feed_forward(y, wg, wu)[0])
    with torch.no_grad():
        x, z = (torch.cat([w[i][:n] for w, n in zip(whole, lengths)]) for i in range(2))
        at = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda")
        u, conv_state = mamba.mamba_conv_packed(x, at, **m["conv"])
        draw, b, c = projections(u)
        y, ssm_state = mamba.mamba_ssm_packed(draw, m["A"], b, c, u, z, m["Dp"], at)
        rows = gated.gated_feed_forward(y, wg, wu)
        got = [[rows[a:e]] for a, e in zip(at.tolist(), at.tolist()[1:])]
        for i in range(more):
            xi, zi = (torch.stack([w[k][n + i] for w, n in zip(whole, lengths)]) for k in range(2))
            out = mamba.mamba_step(xi, zi, conv_state, ssm_state, m["conv"]["weight"], m["conv"]["bias"], **p, A=m["A"], Dp=m["Dp"])
            for s, o in zip(got, gated.gated_feed_forward(out, wg, wu)):
                s.append(o[None])
    for g, w in zip(got, want):
        assert float((torch.cat(g) - w).abs().max() / w.abs().max()) <= 2e-5


def test_beyond_32_bit_offsets(gpu):
    """More than 2^31 elements in a row tensor: the last sequence as it is alone."""
    T, D, N = 1_050_000, 2048, 1
    r = torch.Generator(device="cuda").manual_seed(13)
    big = {k: torch.randn(T, D, generator=r, device="cuda", dtype=BF) for k in ("x", "z")}
    big["draw"], big["u"] = big["z"], big["x"]
    big["B_t"], big["C_t"] = (torch.randn(T, N, generator=r, device="cuda", dtype=BF) for _ in range(2))
    m = dict(make(1, D, N, 4, 2, 1, BF, dev="cuda", seed=14), seq=big)
    first = T - 777
    u, left, y, last = packed(m, torch.tensor([0, first, T], device="cuda"))
    alone = packed(m, torch.tensor([0, 777], device="cuda"), **{k: t[first:] for k, t in big.items()})
    assert torch.equal(u[first:], alone[0]) and torch.equal(left[1], alone[1][0])
    near(y[first:], alone[2].double(), "y bf16", 2)
    near(last[1], alone[3][0].double(), "last")


def test_supports_reasons(gpu):
    m = make(6, 4, 3, 4, 2, 2, F32, dev="cuda")
    s, at, kw = m["seq"], torch.tensor([0, 6], device="cuda"), _step_args(m)
    conv = lambda **k: packed_hip.supports_conv(**{**dict(x=s["x"], starts=at, **m["conv"], tails=None), **k})  # noqa: E731
    ssm = lambda **k: packed_hip.supports_ssm(**{**dict(draw=s["draw"], A=m["A"], B_t=s["B_t"], C_t=s["C_t"], u=s["u"], z=s["z"], Dp=m["Dp"], starts=at, h0=None), **k})  # noqa: E731
    step = lambda **k: packed_hip.supports_step(**{**kw, **k})  # noqa: E731
    assert conv() is None and ssm() is None and step() is None
    assert "a tensor" in conv(starts=at.cpu()) and "float64" in conv(x=s["x"].double()) and "width" in conv(weight=torch.zeros(4, 1, 9, device="cuda"))
    assert "a tensor" in ssm(A=m["A"].cpu()) and "state size" in ssm(A=torch.zeros(4, 65, device="cuda"))
    assert "a tensor" in step(dt_bias=kw["dt_bias"].half()) and "contiguous" in step(ssm_state=kw["ssm_state"].transpose(0, 1))
    big = torch.randn(6, 65, device="cuda")  # more states than the kernels hold: the torch path
    y, _ = mamba.mamba_ssm_packed(s["draw"], -torch.rand(4, 65, device="cuda"), big, big, s["u"], s["z"], m["Dp"], at)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T", [127, 128, 129, 159, 160, 161, 193])
def test_around_the_first_cuts(gpu, T, dtype):
    """Rows that are just short enough for one segment, and the first ones that are not."""
    for starts in ([0, T], [0, 31, 32, 64, 97, T - 1], [33, 95, 95, 128 if T > 128 else 120, T]):
        check_packed(make(T, 70, 16, 4, 2, 1, dtype, dev="cuda", seed=15), starts, True, dtype)


def test_compile_traces_a_layer_in_service(gpu):
    m, at = make(300, 24, 8, 4, 3, 5, F32, dev="cuda", seed=16), torch.tensor([0, 130, 290], device="cuda")
    tails, h0 = m["state"](2)

    def f(conv_state, ssm_state):
        u, left, y, last = packed(m, at, tails, h0)
        out = mamba.mamba_step(**dict(_step_args(m), conv_state=conv_state, ssm_state=ssm_state))
        return u * 1.0, left, y + 0.0, last, out, conv_state + 0.0, ssm_state + 0.0

    t = m["token"]
    with torch.no_grad():
        a, b = (fn(t["conv_state"].clone(), t["ssm_state"].clone()) for fn in (f, torch.compile(f, fullgraph=True)))
    assert same(a, b)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_step_beyond_32_bit_offsets(gpu, dtype):
    """More than 2^31 states: the last rows as they are alone (they lie in other workgroups' rows there: to float32 rounding)."""
    B, D, N = 8200, 4096, 64
    m = make(1, D, N, 4, 8, 6, dtype, dev="cuda", seed=17)
    t = m["token"]
    big = {k: v[:1].expand(B, *v.shape[1:]).contiguous() for k, v in t.items()}
    for k, v in t.items():
        big[k][-6:] = v
    args = _step_args(m)
    y = mamba.mamba_step(**{**args, **big})
    _near_step(args, dtype, "step")
    want = mamba.mamba_step(**{**args, **{k: v.clone() for k, v in _fresh(m).items()}})
    near(y[-6:], want.double(), tag("rows", dtype), 2)
    near(big["ssm_state"][-6:], t["ssm_state"].double(), "h")
    assert torch.equal(big["conv_state"][-6:], t["conv_state"])


def _fresh(m):
    """The tokens of test_step_beyond_32_bit_offsets before its step."""
    t = make(1, *m["A"].shape, 4, 8, 6, m["token"]["x"].dtype, dev="cuda", seed=17)["token"]
    return t
