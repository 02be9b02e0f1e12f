"""The gated and the residual norm over more rows than units of threads (HIP): each unit walks several rows, not all of them as
many, with the next row's loads in flight, its column sums in registers and its sums' places in LDS taken in turn.

Bars, relative to the largest value of each result: float32 1e-5, the package's (a column sum of 40001 rows is 5 rows in turn, then
512 units in turn, then 16 parts: roundings of random sign leave sqrt(512) 2^-24 = 1.3e-6 of it); bfloat16 outputs are rounded
once, 2^-9 of their own size: 2^-8.
"""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import dispatch, gated

pytestmark = pytest.mark.gpu

_EPS = 1e-5


def _rel(a, b):
    assert torch.isfinite(a).all()
    return float((a.detach().cpu().double() - b).abs().max() / b.abs().max())


def _tol(t):
    return 2**-8 if t.dtype == torch.bfloat16 else 1e-5


def _rand(r, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=r).to("cuda", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D,groups,first", [(40001, 64, 4, False), (9001, 195, 1, True), (1500, 4096, 2, False), (1200, 8192, 1, True)])
def test_gated_norm_over_many_rows(gpu, rows, D, groups, first, dtype):
    r = torch.Generator().manual_seed(rows)
    x, z, gy = (_rand(r, rows, D, dtype=dtype) for _ in range(3))
    w = torch.rand(D, generator=r).cuda() + 0.5
    leaves = [t.requires_grad_() for t in (x, z, w)]
    with dispatch.use_backend("hip"):
        y = gated.gated_norm(x, z, w, groups=groups, eps=_EPS, gate_first=first)
    want, *grads = G.gated_norm(x, z, w, groups, _EPS, first, gy)
    assert _rel(y, want) < _tol(y)
    for got, ref in zip(torch.autograd.grad(y, leaves, gy), grads):
        assert _rel(got, ref) < _tol(got)


@pytest.mark.parametrize("dtype,res", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("rows,D", [(40001, 64), (8401, 1536), (2500, 2047), (1200, 8192)])
def test_residual_norm_over_many_rows(gpu, rows, D, post, dtype, res):
    r = torch.Generator().manual_seed(D)
    x, gy = _rand(r, rows, D, dtype=dtype), _rand(r, rows, D, dtype=dtype)
    s, gn = _rand(r, rows, D, dtype=res), _rand(r, rows, D, dtype=res)
    w, p, c = (torch.rand(D, generator=r).cuda() + 0.5 for _ in range(3))
    p = p if post else None
    leaves = [t.requires_grad_() for t in (x, s, w, p, c) if t is not None]
    with dispatch.use_backend("hip"):
        new, y = gated.residual_norm(x, s, w, post_weight=p, scale=c, eps=_EPS)
    want_new, want_y, *grads = G.residual_norm(x, s, w, p, c, _EPS, gn, gy)
    grads = [t for t, there in zip(grads, (True, True, True, post, True)) if there]
    assert _rel(new, want_new) < _tol(new) and _rel(y, want_y) < _tol(y)
    for got, ref in zip(torch.autograd.grad([new, y], leaves, [gn, gy]), grads):
        assert _rel(got, ref) < _tol(got)
