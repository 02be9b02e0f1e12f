"""Which sizes the packed operators of a Mamba layer in service take, without a GPU."""

from types import SimpleNamespace

import pytest
import torch

from tsfast_amd import _lib
from tsfast_amd.mamba import packed_hip

P = 1 << 20  # an address that is never read


def _tensor(dtype, *shape):
    """A stand-in for a tensor that fits no memory here."""
    return SimpleNamespace(dtype=dtype, device="cuda:0", shape=shape, get_device=lambda: 0)


def _supports(T, D, N, S=1):
    row, wide = (lambda n: _tensor(torch.bfloat16, T, n)), lambda *s: _tensor(torch.float32, *s)
    return packed_hip.supports_ssm(row(D), wide(D, N), row(N), row(N), row(D), row(D), wide(D), _tensor(torch.int32, S + 1), None)


def _library(T, D, N, S=1):
    """The library's status of such a call without a workspace: -2 where it needs one, that is, it would run; -3: declined."""
    return _lib.load().tsfast_hip_mamba_packed(T, S, D, N, 1, 0, P, D, P, P, N, P, N, P, D, P, D, P, P, None, P, P, None, 0, None)


@pytest.mark.parametrize("T,D,N", [(1 << 20, 1 << 14, 16), (1 << 25, 512, 8), (1 << 30, 64, 64), (1 << 26, 1 << 10, 16)])
def test_long_and_wide_rows_are_for_the_kernel(T, D, N):
    assert _library(T, D, N) == -2 and _supports(T, D, N) is None


def test_sizes_beyond_the_kernels():
    for T, D, N in ((1 << 20, 64, 65), ((1 << 30) + 1, 64, 16), (1 << 20, (1 << 24) + 1, 16)):
        assert _library(T, D, N) == -3 and _supports(T, D, N) is not None
