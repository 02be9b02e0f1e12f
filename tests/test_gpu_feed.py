"""The fused gated feed-forward block on the GPU against float64.

Bars. Forward, bfloat16: sums are float32 and the result is rounded once, so an element is off by half a step (2^-8 of it)
and float32's part. Gradients, bfloat16: da and db are rounded once more, each by up to 2^-8 of itself, so an element is off by up to
2^-8 of the sum of its terms' magnitudes (and half a step of itself); as the roundings are independent, the whole gradient is off by
less than 2^-8 of its norm. Biases' gradients are sums of unrounded values. float32: a sum of n products is off by up to
n 2^-24 of the sum of their magnitudes in the worst order and about sqrt(n) 2^-24 in the usual case; the pairs of bfloat16 parts
that are left out are below 2^-23 of a product; the activation adds about 3e-7 of its value: 1e-5
of the sum of the magnitudes covers n up to 65536. What enters a gradient's sum, da and db, is itself off by that part of what a's and b's sums
are formed of, which counts where they cancel (feed_oracle.reach; a gradient of one row has no other rows that even it out)."""

import pytest
import torch

from oracle import feed_oracle
from tsfast_amd import gated
from tsfast_amd.gated import feed_hip

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _inputs(shape, D, F, dtype, bias, seed=0, dev="cuda"):
    r = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, device=dev)  # noqa: E731
    x, wg, wu, gy = n(*shape, D).to(dtype), (n(F, D) / D**0.5).to(dtype), (n(F, D) / D**0.5).to(dtype), n(*shape, F).to(dtype)
    return x, wg, wu, *((n(F).to(dtype), n(F).to(dtype)) if bias else (None, None)), gy


def _near(got, want, sums, reach, dtype, roundings, what):
    got, want = got.detach().double(), want.reshape(got.shape)
    sums, reach = (t.reshape(got.shape) for t in (sums, reach))
    err = (got - want).abs()
    half = 2.0**-8 if dtype == BF else 2.0**-24
    bound = 1e-5 * reach + half * want.abs() + (half * sums if roundings > 1 else 0)
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
    mag, reaches = feed_oracle.reach(x.reshape(-1, D), wg, wu, bg, bu, act, gy.reshape(-1, gy.shape[-1]))
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], wg.shape[0])
    _near(served, want, mag, mag, dtype, 1, "y")
    _near(y, want, mag, mag, dtype, 1, "y of a training step")
    names = [n for n, t in zip(("dx", "dwg", "dwu", "dbg", "dbu"), (x, wg, wu, bg, bu)) if t is not None]
    by_name = dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), zip(wgrads, sums, reaches)))
    for n, g in zip(names, grads):
        assert g.dtype == dtype
        _near(g, *by_name[n], dtype, 1 if n in ("dbg", "dbu") else 2, n)
    return y, grads


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize(
    "rows,D,F,bias",
    [(1, 1, 1, True), (1, 8, 16, False), (5, 33, 47, True), (16, 64, 64, False), (17, 40, 130, True), (33, 195, 517, True), (49, 131, 70, True), (64, 64, 32, False), (257, 96, 264, True)],
)
def test_small_sizes(gpu, rows, D, F, bias, act, dtype):
    _check(*_inputs((rows,), D, F, dtype, bias), act, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,D,F,bias", [(2050, 130, 700, True), (4096, 512, 1024, False), (20000, 64, 256, True), (1000, 1032, 2056, False), (700, 2048, 40, True)])
def test_larger_sizes(gpu, rows, D, F, bias, dtype):
    _check(*_inputs((rows,), D, F, dtype, bias, seed=1), "silu", dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,D,F", [(20, 72, 100), (300, 72, 100), (300, 71, 99)])
def test_layouts(gpu, rows, D, F, dtype):
    """Rows of a wider tensor at odd offsets, weights that are halves of one or lie transposed, gradients that are expanded or turned: as dense ones."""
    x, wg, wu, _, _, gy = _inputs((rows,), D, F, dtype, False, seed=2)
    want = _run(x, wg, wu, gy)
    wide = torch.randn(rows, 3 * D + 1, device="cuda").to(dtype)
    wide[:, D + 1 : 2 * D + 1] = x
    both = torch.cat((wg, wu))
    stacked = torch.randn(2 * F, D + 3, device="cuda").to(dtype)
    stacked[:F, 1 : D + 1], stacked[F:, 2 : D + 2] = wg, wu
    for views in ((wide[:, D + 1 : 2 * D + 1], wg, wu), (x, *both.chunk(2)), (x, stacked[:F, 1 : D + 1], stacked[F:, 2 : D + 2]), (x.t().contiguous().t(), wg.t().contiguous().t(), wu)):
        assert all(torch.equal(a, b) for a, b in zip(_run(*views, gy), want))
    assert all(torch.equal(a, b) for a, b in zip(_run(x, wg, wu, gy.t().contiguous().t()), want))
    one = gy[:1].expand(rows, F)
    assert all(torch.equal(a, b) for a, b in zip(_run(x, wg, wu, one), _run(x, wg, wu, one.contiguous())))
    same = x[:1].expand(rows, D)
    assert all(torch.equal(a, b) for a, b in zip(_run(same, wg, wu, gy), _run(same.contiguous(), wg, wu, gy)))
    leaf = wg.clone().requires_grad_()  # one tensor as both weights
    (shared,) = torch.autograd.grad(gated.gated_feed_forward(x, leaf, leaf), leaf, gy)
    apart = _run(x, wg, wg.clone(), gy)
    assert torch.equal(shared, apart[2] + apart[3])


def _run(x, wg, wu, gy, act="silu"):
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    y = gated.gated_feed_forward(*leaves, activation=act)
    with torch.no_grad():
        served = gated.gated_feed_forward(x, wg, wu, activation=act)
    return (y.detach(), *torch.autograd.grad(y, leaves, gy), served)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_leading_dimensions_and_none(gpu, dtype):
    x, wg, wu, bg, bu, gy = _inputs((3, 7), 40, 56, dtype, True, seed=3)
    _check(x, wg, wu, bg, bu, gy, "gelu", dtype)
    _check(x.transpose(0, 1), wg, wu, bg, bu, gy.transpose(0, 1), "gelu", dtype)
    _check(x[0, 0], wg, wu, bg, bu, gy[0, 0], "gelu", dtype)
    none = x[:0].requires_grad_()
    w = [t.clone().requires_grad_() for t in (wg, wu, bg, bu)]
    y = gated.gated_feed_forward(none, *w)
    assert y.shape == (0, 7, 56) and gated.gated_feed_forward(none.detach(), wg, wu).shape == (0, 7, 56)
    grads = torch.autograd.grad(y, [none, *w], torch.empty_like(y))
    assert grads[0].shape == none.shape and all(not g.any() for g in grads[1:])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_any_subset_of_gradients(gpu, dtype):
    x, wg, wu, bg, bu, gy = _inputs((70,), 40, 56, dtype, True, seed=4)
    tensors = (x, wg, wu, bg, bu)

    def grads(want):
        leaves = [t.clone().requires_grad_(w) for t, w in zip(tensors, want)]
        y = gated.gated_feed_forward(*leaves)
        return dict(zip((i for i, w in enumerate(want) if w), torch.autograd.grad(y, [t for t in leaves if t.requires_grad], gy)))

    every = grads([True] * 5)
    for n in range(1, 32):
        some = grads([bool(n >> i & 1) for i in range(5)])
        assert all(torch.equal(g, every[i]) for i, g in some.items()), n


@pytest.mark.parametrize("dtype", [F32, BF])
def test_repeats_streams_and_graphs(gpu, dtype):
    """Every sum has a fixed order: repeats, another stream, two streams at once and replays on new inputs give the same bits."""
    x, wg, wu, _, _, gy = _inputs((900,), 96, 130, dtype, False, seed=5)
    few = x[:9].clone()

    def work():
        y, kept = feed_hip._feed_train_op(x, wg, wu, None, None, 0)
        return y, *feed_hip._feed_bwd_op(gy, kept, x, wg, wu, True, True, 0, True, True), feed_hip._feed_op(few, wg, wu, None, None, 0)

    want = work()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(work(), want))
    sides = torch.cuda.Stream(), torch.cuda.Stream()
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    got = []
    for side in sides * 2:
        with torch.cuda.stream(side):
            got.append(work())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work()))
    for seed in (1, 2, 3):
        new = _inputs((900,), 96, 130, dtype, False, seed=seed)
        for dst, src in zip((x, wg, wu, gy), (*new[:3], new[5])):
            dst.copy_(src)
        few.copy_(x[:9])
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs]
            assert all(torch.equal(a, b) for a, b in zip(got, work())), seed


def test_a_captured_training_step(gpu):
    x, wg, wu, bg, bu, gy = _inputs((600,), 64, 96, BF, True, seed=6)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    step = lambda: torch.autograd.grad(gated.gated_feed_forward(*leaves), leaves, gy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for seed in (7, 8, 9):
        with torch.no_grad():
            for t, new in zip(leaves, _inputs((600,), 64, 96, BF, True, seed=seed)):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in grads]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_compile_traces_the_block(gpu):
    x, wg, wu, bg, bu, _ = _inputs((40,), 24, 32, F32, True, seed=7)
    f = lambda *t: (gated.gated_feed_forward(t[0] * 1.5, *t[1:]) * 2).sum()  # noqa: E731
    grads = []
    for fn in (f, torch.compile(f, fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
        grads.append(torch.autograd.grad(fn(*leaves), leaves))
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)


def test_gradients_against_differences(gpu):
    """Along the gradient g by +-e: the difference is 2 e |g|^2 and what the third derivatives add (e^2 of it) and float32's rounding of
    the two sums (below 2^-20 of the sum of their terms' magnitudes, |y| . |gy|)."""
    x, wg, wu, bg, bu, gy = _inputs((200,), 48, 64, F32, True, seed=8)
    for act in ("silu", "gelu", "sigmoid"):
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
        y = gated.gated_feed_forward(*leaves, activation=act)
        for i, g in enumerate(torch.autograd.grad(y, leaves, gy)):
            e = 1e-2 / float(g.double().norm())
            loss = []
            for sign in (1, -1):
                moved = [t.detach() + sign * e * g if i == k else t.detach() for k, t in enumerate(leaves)]
                loss.append(float((gated.gated_feed_forward(*moved, activation=act).double() * gy.double()).sum()))
            want = 2 * e * float((g.double() ** 2).sum())
            noise = 2.0**-19 * float((y.detach().double() * gy.double()).abs().sum())
            assert abs(loss[0] - loss[1] - want) <= 1e-3 * want + noise, (act, i)


def test_large_values(gpu):
    """Saturated activations: exact zeros and the identity, no NaN, and zero gradients where the activation is flat."""
    x = torch.tensor([[1.0], [-1.0]], device="cuda")
    for dtype in (F32, BF):
        for act in ("silu", "gelu", "sigmoid"):
            w = torch.full((1, 1), 1e4, device="cuda", dtype=dtype)
            leaves = [x.to(dtype).requires_grad_(), w.clone().requires_grad_(), torch.ones_like(w).requires_grad_()]
            y = gated.gated_feed_forward(*leaves, activation=act)
            assert y.flatten().tolist() == [1.0 if act == "sigmoid" else float(w), 0.0]
            assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y.sum(), leaves))


def test_supports_reasons(gpu):
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    ok = lambda x, w, v=None, b=None: feed_hip.supports(x, w, w if v is None else v, b, None)  # noqa: E731
    assert ok(x, w) is None and ok(x.bfloat16(), w.bfloat16()) is None
    assert "GPU-only" in ok(x.cpu(), w) and "float64" in ok(x.double(), w.double()) and "parameter" in ok(x, w, w.cpu())
    y = gated.gated_feed_forward(x.double(), w.double(), w.double())  # the torch path
    assert y.dtype == torch.float64 and torch.allclose(y, feed_oracle.feed(x, w, w, None, None, "silu"))


def test_beyond_32_bit_offsets(gpu):
    """More than 2^31 outputs: the last rows against float64, and their gradients."""
    rows, D, F, n = 530_000, 16, 4096, 100
    x, wg, wu, _, _, gy = _inputs((rows,), D, F, BF, False, seed=9)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    y = gated.gated_feed_forward(*leaves)
    (gx,) = torch.autograd.grad(y, x, gy)
    want, wgrads, sums = feed_oracle.feed(x[-n:], wg, wu, None, None, "silu", gy[-n:])
    mag, reaches = feed_oracle.reach(x[-n:], wg, wu, None, None, "silu", gy[-n:])
    _near(y[-n:], want, mag, mag, BF, 1, "y")
    _near(gx[-n:], wgrads[0], sums[0], reaches[0], BF, 2, "dx")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,D,F,bias", [(33, 2048, 61, True), (100, 2000, 517, True), (200, 1031, 64, False), (130, 4096, 1000, True), (65, 1536, 9, True)])
def test_parts_of_a_long_contraction(gpu, rows, D, F, bias, dtype):
    """Few tiles and a long k: every product is taken in parts, joined behind them."""
    _check(*_inputs((rows,), D, F, dtype, bias, seed=10), "gelu", dtype)
