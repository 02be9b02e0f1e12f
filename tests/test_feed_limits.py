"""Which sizes of the feed-forward block are declined, without a GPU: those that one launch of less than 2^32 threads does not hold, by the
library and by the Python side alike."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from tsfast_amd import _lib
from tsfast_amd.gated import feed_hip

SIZES = [
    (1, 1, 1), (64, 8, 8), (65, 2048, 5461), (1 << 20, 1536, 4096), (1 << 24, 1, 1), ((1 << 30) - 64, 8, 8), ((1 << 30) - 63, 8, 8), (1 << 30, 8, 8),
    (1 << 30, 64, 32), (1 << 30, 65, 8), ((1 << 31) - 64, 1, 1), ((1 << 31) - 63, 1, 1), (1 << 29, 128, 32), (1 << 29, 64, 64), (1 << 29, 129, 8),
    (1, 1 << 20, 1 << 20), (1, 1 << 20, 1 << 16), (64, 1 << 18, 1 << 18), (64, 1 << 19, 1 << 19), (64, 1 << 20, 1 << 18), (4096, 1 << 20, 1 << 10),
    (1 << 15, 1 << 15, 1 << 15), (1, (1 << 20) + 1, 1),
]  # fmt: skip


def plan(rows, D, F, io, train):
    out = (ctypes.c_int64 * 12)()
    status = _lib.load().tsfast_hip_feed_plan(rows, D, F, io, train, ctypes.addressof(out))
    return status, [out[4 * i : 4 * i + 4] for i in range(3)]


def _tensors(rows, D, F, dtype):
    """Stand-ins for tensors that fit no memory."""
    one = lambda *shape: SimpleNamespace(dtype=dtype, device="cuda:0", shape=shape, get_device=lambda: 0, numel=lambda: torch.Size(shape).numel())  # noqa: E731
    return one(rows, D), one(F, D), one(F, D), None, None


@pytest.mark.parametrize("dtype,io", feed_hip._IO_DTYPES.items())
@pytest.mark.parametrize("rows,D,F", SIZES)
def test_every_size_is_launched_whole_or_declined(rows, D, F, dtype, io):
    declined = _lib.load().tsfast_hip_feed_kept_bytes(rows, D, F, io) < 0
    assert (feed_hip.supports(*_tensors(rows, D, F, dtype)) is not None) == declined
    for train in (0, 1):
        status, plans = plan(rows, D, F, io, train)
        assert status == (-3 if declined else 0)
        if not declined:
            for edge, parts, workgroups, threads in plans:
                assert edge in (0, 64, 128, 256) and 1 <= parts <= 64 and 0 < workgroups * threads < 1 << 32


def test_the_largest_sizes():
    declined = lambda *size: _lib.load().tsfast_hip_feed_kept_bytes(*size, 1) < 0  # noqa: E731
    assert not declined((1 << 30) - 64, 8, 8) and declined((1 << 30) - 63, 8, 8)  # 2^24 workgroups of 256 threads are one launch too many
    assert not declined(64, 1 << 18, 1 << 18) and declined(64, 1 << 20, 1 << 20)


def test_plan_queries():
    assert plan(20, 64, 32, 1, 0)[1][0] == [0, 1, 2, 256] and plan(20, 64, 32, 1, 1)[1][0][0] == 64
    assert plan(0, 8, 8, 0, 0)[0] == plan(1, 0, 8, 0, 0)[0] == plan(1, 8, 8, 2, 0)[0] == -1
    assert _lib.load().tsfast_hip_feed_plan(1, 8, 8, 0, 0, None) == -1
