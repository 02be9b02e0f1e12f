"""A token of float32 sequences through parameters kept in bfloat16, on the GPU against float64: as ``test_gpu_serving`` has it for the other types."""

import pytest
import torch

from tests.test_gpu_serving import _near_step, _step_args
from tests.test_serving import BF, F32, make
from tsfast_amd import dispatch

pytestmark = pytest.mark.gpu

PARAMETERS = ("conv_weight", "conv_bias", "x_proj", "dt_proj", "dt_bias")


def _args(B, D, N, K, R, which):
    kw = _step_args(make(1, D, N, K, R, B, F32, dev="cuda", seed=11))
    for k in which:
        kw[k] = kw[k].bfloat16()
    return kw


@pytest.fixture(autouse=True)
def _fused_only(monkeypatch):
    """The torch path would do too: no test here may take it."""

    def declined(key, message):
        raise AssertionError(message)

    monkeypatch.setattr(dispatch, "warn_fallback", declined)


@pytest.mark.parametrize("B,D,N,K,R", [(1, 1, 1, 2, 1), (1, 128, 16, 4, 8), (17, 130, 33, 3, 9), (33, 200, 64, 8, 40), (5, 1100, 16, 4, 69), (3, 70, 20, 5, 130), (256, 96, 16, 4, 6)])
def test_float32_tokens_with_bfloat16_parameters(gpu, B, D, N, K, R):
    _near_step(_args(B, D, N, K, R, PARAMETERS), F32, "step")


@pytest.mark.parametrize("which", range(1, 31))
def test_float32_tokens_with_parameters_of_both_types(gpu, which):
    _near_step(_args(3, 40, 16, 4, 5, [k for i, k in enumerate(PARAMETERS) if which >> i & 1]), F32, "step")
