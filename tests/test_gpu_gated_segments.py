"""The gated recurrence on few long rows (HIP), whose segments' states are joined 16 at a time: as many segments as that,
one more, two more and several times as many, with the forward's states kept for the backward and without.

Bars as for the recurrence on short rows, relative to the largest value of each result: float32 1e-5; bfloat16 2^-8 where outputs are rounded
to it and 2e-5 for the float32 states.
"""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import _lib
from tsfast_amd.gated import recurrence_hip

pytestmark = pytest.mark.gpu


def _rel(a, b):
    assert torch.isfinite(a).all()
    return float((a.detach().cpu().double() - b).abs().max() / b.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("segments,L,K,V", [(16, 4096, 24, 100), (17, 4352, 20, 16), (17, 4300, 100, 24), (18, 4608, 72, 80), (34, 8704, 33, 64),
                                            (34, 8700, 40, 70)])
def test_many_segments(gpu, segments, L, K, V, dtype):
    r = torch.Generator().manual_seed(L + K)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    # heads that remember for over a segment (256 steps), and a reset inside one
    g = -torch.rand(1, L, 2, generator=r) * torch.tensor([2e-3, 0.05])
    g[:, 1000, 1] = float("-inf")
    q, k, v, g, go = (t.to("cuda", dtype) for t in (n(1, L, 1, K), n(1, L, 1, K) / K**0.5, n(1, L, 2, V), g, n(1, L, 2, V)))
    state, gl = n(1, 2, K, V).cuda(), n(1, 2, K, V).cuda()
    io = _lib.TSF_DTYPE_BF16 if dtype == torch.bfloat16 else _lib.TSF_DTYPE_F32
    padded = (64 if K <= 64 else 128) * (64 if V <= 64 else 128) * 4
    assert _lib.load().tsfast_hip_gated_kept_bytes(1, L, 2, 1, K, V, io) == 2 * segments * padded
    with torch.no_grad():
        o, last, kept = recurrence_hip._recurrence_train_op(q, k, v, g, state)
        results = [recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, state, *how) for how in ((kept,), ())]
    want_o, want_last, _ = G.recurrence(q, k, v, g, state)
    wants = G.recurrence_grads(go, gl, q, k, v, g, state)
    tol, tol32 = (2**-8, 2e-5) if dtype == torch.bfloat16 else (1e-5, 1e-5)
    assert _rel(o, want_o) < tol and _rel(last, want_last) < tol32
    for grads in results:
        for name, got, want in zip("qkvgs", grads, wants):
            assert _rel(got, want) < (tol32 if name == "s" else tol), name
