"""Calls at the edges of the gated recurrence's arguments (HIP): results are the contiguous tensors' bits."""

import pytest
import torch

from tsfast_amd import dispatch, gated
from tsfast_amd.gated import recurrence_hip

pytestmark = pytest.mark.gpu


def _inputs(B, L, H, Hk, K, V, dtype, seed=0):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    g = -torch.rand(B, L, H, generator=r) * 0.05
    seq = (n(B, L, Hk, K), n(B, L, Hk, K) / K**0.5, n(B, L, H, V), g)
    return *(t.to("cuda", dtype) for t in seq), n(B, H, K, V).cuda(), n(B, L, H, V).to("cuda", dtype), n(B, H, K, V).cuda()


def _run(q, k, v, g, state, go, gl):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state)]
    with dispatch.use_backend("hip"):
        o, last = gated.gated_recurrence(*leaves)
    return o, last, *torch.autograd.grad([o, last], leaves, [go, gl])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [0, 1])
def test_steps_of_any_distance_where_there_is_no_second_one(gpu, L, dtype):
    """One token of a time-major or cached tensor: the distance to the next step, which is not there, may be beyond the 32-bit
    offsets of a chunk (and no copy changes it: such a tensor counts as contiguous where there is one row)."""
    args = _inputs(1, L, 2, 1, 16, 24, dtype)
    far = 2 * recurrence_hip._MAX_STEP

    def apart(t):
        return t.as_strided(t.shape, (t.stride(0), far, *t.stride()[2:]))

    q, k, v, g, s, go, gl = args
    want, got = _run(*args), _run(*(apart(t) for t in (q, k, v, g)), s, apart(go), gl)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
