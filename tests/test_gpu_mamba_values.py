"""The training scan of a Mamba layer on the GPU with a NaN among its step sizes: it shows where float64 has it, and nowhere else."""

import pytest
import torch

from tsfast_amd import mamba

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16


def _inputs(B, L, D, N, dtype):
    r = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=r, device="cuda")  # noqa: E731
    A = -torch.rand(D, N, generator=r, device="cuda") * 4 - 0.1
    return [(n(B, L, D) - 3).to(dtype), A, n(B, L, N).to(dtype), n(B, L, N).to(dtype), n(B, L, D).to(dtype), n(B, L, D).to(dtype), n(D), n(B, D, N)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,L,D,N", [(2, 50, 70, 16), (1, 3000, 64, 8), (3, 700, 96, 16)])
def test_a_nan_step_size_stays_in_its_sequence_and_channel(gpu, B, L, D, N, dtype):
    tensors = _inputs(B, L, D, N, dtype)
    b, t, d = B - 1, L // 3, D - 2
    hurt = tensors[0].clone()
    hurt[b, t, d] = float("nan")
    mask = torch.ones(B, L, D, dtype=torch.bool, device="cuda")
    mask[b, t:, d] = False
    g = torch.randn(B, L, D, device="cuda").to(dtype)
    results = []
    for draw in (tensors[0], hurt):
        with torch.no_grad():
            served, last = mamba.mamba_ssm(draw, *tensors[1:])
        leaves = [v.clone().requires_grad_() for v in (draw, tensors[4], tensors[5])]
        out, _ = mamba.mamba_ssm(leaves[0], *tensors[1:4], *leaves[1:], *tensors[6:])
        results.append((served, out.detach(), last.view(B, D, N), *torch.autograd.grad(out, leaves, g)))
    want, got = results
    for w, h in zip(want[:2], got[:2]):
        assert h[~mask].isnan().all() and torch.equal(h[mask], w[mask])
    assert got[2][b, d].isnan().all() and int(got[2].isnan().any(-1).sum()) == 1
    assert got[3][b, t, d].isnan()
    whole = torch.ones(B, L, D, dtype=torch.bool, device="cuda")
    whole[b, :, d] = False  # a gradient goes back to the row's start
    for w, h in zip(want[3:], got[3:]):
        assert torch.equal(h[whole], w[whole])
