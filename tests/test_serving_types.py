"""The types that a token's parameters may have, without a GPU."""

import itertools

import pytest
import torch

from oracle import serving_oracle as O
from tests.test_serving import BF, F32, F64, make, rel
from tsfast_amd import mamba
from tsfast_amd.mamba import packed_hip


def _args(dtype, other):
    m = make(1, 7, 5, 4, 2, 3, dtype, seed=2)
    p = {k: v.to(other) for k, v in m["proj"].items()}
    return dict(**m["token"], conv_weight=m["conv"]["weight"].to(other), conv_bias=m["conv"]["bias"].to(other), **p, A=m["A"], Dp=m["Dp"])


@pytest.mark.parametrize("dtype,other", itertools.product((F32, BF, F64), (F32, BF)))
def test_parameters_in_float32_or_bfloat16_whatever_the_tokens_are(dtype, other):
    """To 1e-5 of the largest value (sums of at most 7 products in float32), bfloat16 outputs half a step more."""
    kw = _args(dtype, other)
    want = O.step(**kw)
    out = mamba.mamba_step(**kw)
    tol = 1e-5 + (2.0**-8 if dtype == BF else 0)
    assert out.dtype == dtype and rel(out, want[0]) <= tol and rel(kw["ssm_state"], want[2]) <= 1e-5


def test_other_types_are_refused_by_name():
    for dtype in (F32, BF):
        for other in (torch.float16, F64):
            with pytest.raises(ValueError, match="float32, bfloat16 or"):
                mamba.mamba_step(**_args(dtype, other))


def test_the_kernels_take_what_the_public_step_takes():
    gpu = lambda t: type("T", (), dict(dtype=t.dtype, device="cuda:0", shape=t.shape, get_device=lambda s: 0, is_contiguous=lambda s: True))()  # noqa: E731
    for dtype, other in itertools.product((F32, BF), (F32, BF)):
        assert packed_hip.supports_step(*(gpu(t) for t in _args(dtype, other).values())) is None
