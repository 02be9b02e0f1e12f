"""GPU parity of the gated and the residual norm (HIP) against the float64 oracle.

Bars, relative to the largest value of each result: float32 1e-5 (the package's bar; sums over up to 8192 columns in float32
trees, and over up to 3000 rows for the parameters). bfloat16 outputs are rounded once, 2^-9 of their own size: 2^-8; float32 results
from bfloat16 inputs (parameter gradients, a float32 stream) keep 1e-5.
"""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import dispatch, gated
from tsfast_amd.gated import core, norm_hip

pytestmark = pytest.mark.gpu

_EPS = 1e-5


def _rel(a, b):
    if not b.numel():
        return 0.0
    assert torch.isfinite(a).all()
    return float((a.detach().cpu().double() - b).abs().max() / b.abs().max().clamp_min(1e-30))


def _tol(t):
    return 2**-8 if t.dtype == torch.bfloat16 else 1e-5


def _rand(r, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=r).to("cuda", dtype)


_GATED = [
    ((3,), 7, 1), ((2, 5), 24, 3), ((4,), 195, 1), ((70,), 128, 1), ((33,), 256, 2), ((9,), 1536, 12), ((5,), 1536, 1),
    ((3,), 1000, 1), ((2,), 2047, 1), ((3,), 4096, 1), ((2,), 8192, 1), ((2,), 4500, 1), ((3000,), 64, 4), ((1100,), 520, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("lead,D,groups", _GATED)
def test_gated_norm(gpu, lead, D, groups, first, dtype):
    r = torch.Generator().manual_seed(D + groups)
    x, z, gy = (_rand(r, *lead, D, dtype=dtype) for _ in range(3))
    w = torch.rand(D, generator=r).cuda() + 0.5
    leaves = [t.requires_grad_() for t in (x, z, w)]
    with dispatch.use_backend("hip"):
        assert dispatch.resolve("gated.norm", core._NORM_BACKENDS, (), (x, z, (w,), D // groups)) is norm_hip
        y = gated.gated_norm(x, z, w, groups=groups, eps=_EPS, gate_first=first)
    want, *grads = G.gated_norm(x, z, w, groups, _EPS, first, gy)
    assert y.dtype == dtype and _rel(y, want) < _tol(y)
    for got, ref in zip(torch.autograd.grad(y, leaves, gy), grads):
        assert _rel(got, ref) < _tol(got)


@pytest.mark.parametrize("D,groups", [(1, 1), (36, 36)])
def test_one_column(gpu, D, groups):
    """Groups of one column, with an eps at which x's gradient, d (1 - rms(x)^2), is no small difference."""
    r = torch.Generator().manual_seed(7)
    x, z, gn, gy = (_rand(r, 3, D) for _ in range(4))
    w = torch.rand(D, generator=r).cuda() + 0.5
    leaves = [t.requires_grad_() for t in (x, z, w)]
    y = gated.gated_norm(x, z, w, groups=groups, eps=0.5)
    for got, ref in zip([y, *torch.autograd.grad(y, leaves, gy)], G.gated_norm(x, z, w, groups, 0.5, False, gy)):
        assert _rel(got, ref) < 1e-5
    if D == 1:
        new, y = gated.residual_norm(x, z, w, post_weight=w, eps=0.5)
        want = G.residual_norm(x, z, w, w, None, 0.5, gn, gy)
        gx, gz, gw = torch.autograd.grad([new, y], leaves, [gn, gy])
        for got, ref in zip((new, y, gx, gz, gw), (*want[:4], want[4] + want[5])):
            assert _rel(got, ref) < 1e-5


@pytest.mark.parametrize("gate,weight", [(False, True), (True, False), (False, False)])
def test_gated_norm_parts_may_be_absent(gpu, gate, weight):
    r = torch.Generator().manual_seed(1)
    x, z, gy = (_rand(r, 50, 96) for _ in range(3))
    z, w = z if gate else None, torch.rand(96, generator=r).cuda() if weight else None
    leaves = [t.requires_grad_() for t in (x, z, w) if t is not None]
    y = gated.gated_norm(x, z, w, groups=2, gate_first=True)
    want, gx, gz, gw = G.gated_norm(x, z, w, 2, 1e-5, gate, gy)
    assert _rel(y, want) < 1e-5
    refs = [t for t, there in ((gx, True), (gz, gate), (gw, weight)) if there]
    for got, ref in zip(torch.autograd.grad(y, leaves, gy), refs):
        assert _rel(got, ref) < 1e-5


_RESIDUAL = [(3, 7), (10, 195), (70, 128), (33, 256), (9, 1536), (600, 1000), (2, 2047), (3, 4096), (2, 8192), (3, 4501), (3000, 64)]
_KINDS = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dtype,res", _KINDS)
@pytest.mark.parametrize("rows,D", _RESIDUAL)
def test_residual_norm(gpu, rows, D, dtype, res):
    r = torch.Generator().manual_seed(D)
    x, gy = _rand(r, rows, D, dtype=dtype), _rand(r, rows, D, dtype=dtype)
    s, gn = _rand(r, rows, D, dtype=res), _rand(r, rows, D, dtype=res)
    w, p, c = (torch.rand(D, generator=r).cuda() + 0.5 for _ in range(3))
    leaves = [t.requires_grad_() for t in (x, s, w, p, c)]
    with dispatch.use_backend("hip"):
        new, y = gated.residual_norm(x, s, w, post_weight=p, scale=c, eps=_EPS)
    want_new, want_y, *grads = G.residual_norm(x, s, w, p, c, _EPS, gn, gy)
    assert new.dtype == res and y.dtype == dtype
    assert _rel(new, want_new) < _tol(new) and _rel(y, want_y) < _tol(y)
    for got, ref in zip(torch.autograd.grad([new, y], leaves, [gn, gy]), grads):
        assert _rel(got, ref) < _tol(got)


@pytest.mark.parametrize("weight,post,scale", [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
def test_residual_norm_parts_may_be_absent(gpu, weight, post, scale):
    r = torch.Generator().manual_seed(2)
    x, s, gn, gy = (_rand(r, 40, 100) for _ in range(4))
    w, p, c = (torch.rand(100, generator=r).cuda() + 0.5 if there else None for there in (weight, post, scale))
    leaves = [t.requires_grad_() for t in (x, s, w, p, c) if t is not None]
    new, y = gated.residual_norm(x, s, w, post_weight=p, scale=c)
    want_new, want_y, gx, gs, gw, gp, gc = G.residual_norm(x, s, w, p, c, 1e-5, gn, gy)
    assert _rel(new, want_new) < 1e-5 and _rel(y, want_y) < 1e-5
    refs = [t for t, there in ((gx, True), (gs, True), (gw, weight), (gp, post), (gc, scale)) if there]
    for got, ref in zip(torch.autograd.grad([new, y], leaves, [gn, gy]), refs):
        assert _rel(got, ref) < 1e-5


def test_residual_norm_with_one_output_differentiated(gpu):
    r = torch.Generator().manual_seed(3)
    x, s, g = (_rand(r, 20, 64) for _ in range(3))
    w, zero = torch.rand(64, generator=r).cuda(), torch.zeros(20, 64)
    for which in (0, 1):
        leaves = [t.detach().requires_grad_() for t in (x, s, w)]
        out = gated.residual_norm(*leaves)[which]
        grads = torch.autograd.grad(out, leaves, g, allow_unused=True)
        want = G.residual_norm(x, s, w, None, None, 1e-5, *((g, zero) if which == 0 else (zero, g)))[2:5]
        for got, ref in zip(grads, want):
            assert (got == 0).all() if (ref == 0).all() else _rel(got, ref) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [15, 64, 195])
def test_strides_and_alignment(gpu, D, dtype):
    """Slices of one projection at odd offsets, transposed rows and expanded ones give the contiguous rows' bits."""
    r = torch.Generator().manual_seed(4)
    both = _rand(r, 6, 9, 2 * D + 1, dtype=dtype)
    w = torch.rand(D, generator=r).cuda()
    x, z = both[..., 1 : D + 1], both[..., D + 1 :]
    forms = [(x, z), (x.transpose(0, 1).contiguous().transpose(0, 1), z.mT.contiguous().mT), (x[:1].expand_as(x), z)]
    gy = _rand(r, 6, 9, D, dtype=dtype).mT.contiguous().mT
    for a, b in forms:
        results = []
        for u, v in ((a, b), (a.contiguous(), b.contiguous())):
            u, v = u.detach().requires_grad_(), v.detach().requires_grad_()
            y = gated.gated_norm(u, v, w)
            new, y2 = gated.residual_norm(u, v, w, post_weight=w, scale=w)
            results.append([y, new, y2, *torch.autograd.grad([y, new, y2], [u, v], [gy, gy, gy])])
        assert all(torch.equal(p, q) for p, q in zip(*results))


def test_empty_rows_and_rows_of_zeros(gpu):
    w = torch.ones(12, device="cuda", requires_grad=True)
    x = torch.zeros(0, 5, 12, device="cuda", requires_grad=True)
    y = gated.gated_norm(x, x, w)
    new, z = gated.residual_norm(x, x, w, post_weight=w, scale=w)
    assert y.shape == new.shape == z.shape == (0, 5, 12)
    (gw,) = torch.autograd.grad(y.sum() + new.sum() + z.sum(), [w])
    assert (gw == 0).all()
    x = torch.zeros(3, 12, device="cuda", requires_grad=True)
    y = gated.gated_norm(x, x, w)
    new, z = gated.residual_norm(x, x, w, post_weight=w)
    grads = torch.autograd.grad(y.sum() + new.sum() + z.sum(), [x, w])
    assert (y == 0).all() and (z == 0).all() and all(torch.isfinite(t).all() for t in grads)


def test_large_and_small_values(gpu):
    """Gates far out on both sides, rows of very different size."""
    r = torch.Generator().manual_seed(8)
    x, z, gy = _rand(r, 64, 96), _rand(r, 64, 96) * 60, _rand(r, 64, 96)
    x = x * torch.logspace(-8, 8, 64, device="cuda")[:, None]
    x.requires_grad_(), z.requires_grad_()
    y = gated.gated_norm(x, z, None)
    want, gx, gz, _ = G.gated_norm(x, z, None, 1, 1e-5, False, gy)
    got = torch.autograd.grad(y, [x, z], gy)
    assert _rel(y, want) < 1e-5 and _rel(got[0], gx) < 1e-5 and _rel(got[1], gz) < 1e-5


def test_repeats_streams_and_graphs(gpu):
    """Parameter gradients are sums in a fixed order; captured passes equal eager ones, replay after replay."""
    r = torch.Generator().manual_seed(9)
    x, z, gy = (_rand(r, 2000, 260, dtype=torch.bfloat16) for _ in range(3))
    w = torch.rand(260, generator=r).cuda()

    def work():
        y = norm_hip._gated_op(x, z, w, 4, _EPS, False)
        new, y2 = norm_hip._residual_op(y, z, w, w, w, _EPS)
        return y, new, y2, *norm_hip._gated_bwd_op(gy, x, z, w, 4, _EPS, False), *norm_hip._residual_bwd_op(gy, gy, y, z, w, w, w, _EPS)

    a, b = work(), work()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for seed in (1, 2, 3):
        x.copy_(_rand(torch.Generator().manual_seed(seed), 2000, 260))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(p, q) for p, q in zip(got, work())), seed


def test_supports_reasons_and_wide_rows(gpu):
    x, w = torch.randn(2, 8200, device="cuda"), torch.ones(8200, device="cuda")
    assert "columns" in norm_hip.supports(x, x, (w,), 8200) and norm_hip.supports(x, x, (w,), 4100) is None
    assert "GPU-only" in norm_hip.supports(x.cpu(), None, (None,), 8)
    assert "float64" in norm_hip.supports(x.double(), None, (None,), 8)
    assert "parameters" in norm_hip.supports(x, None, (w.double(),), 8)
    assert _rel(gated.gated_norm(x, x, w), G.gated_norm(x, x, w, 1, 1e-5, False)) < 1e-5  # the torch path
    half = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = gated.gated_norm(torch.randn(4, 64, device="cuda"), None, half)
    assert torch.autograd.grad(y.sum(), half)[0].dtype == torch.bfloat16


def test_compile_traces_the_norms(gpu):
    r = torch.Generator().manual_seed(10)
    x, z = _rand(r, 30, 64), _rand(r, 30, 64)
    w = torch.rand(64, generator=r).cuda()

    def f(x, z, w):
        y = gated.gated_norm(x * 2, z, w, groups=2)
        new, y = gated.residual_norm(y, z, w, scale=w)
        return new.sum() + (y * y).sum()

    grads = []
    for fn in (f, torch.compile(f, fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_() for t in (x, z, w)]
        grads.append(torch.autograd.grad(fn(*leaves), leaves))
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
