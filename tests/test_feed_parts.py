"""Three bfloat16 parts of a float32 and six products of them, emulated in float64: what the pairs that are left out cost, and that the GPU's
bars show the loss of any one that is kept."""

import pytest
import torch

from tests.test_gpu_feed_plans import SIZES, bars

PAIRS = ((2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0))  # of parts, the largest first


def parts(t):
    """Each the nearest bfloat16 to what the ones before leave."""
    left, found = t.double(), []
    for _ in range(3):
        found.append(left.float().bfloat16().double())
        left = left - found[-1]
    return found


def off(pairs):
    r = torch.Generator().manual_seed(0)
    x, w = torch.randn(400, 300, generator=r), torch.randn(300, 400, generator=r)
    px, pw, want = parts(x), parts(w), x.double() @ w.double()
    return float((sum(px[i] @ pw[j] for i, j in pairs) - want).norm() / want.norm())


def test_a_float_is_the_sum_of_its_parts():
    t = torch.randn(10_000, generator=torch.Generator().manual_seed(1))
    assert (sum(parts(t)) - t.double()).abs().max() <= 2.0**-24 * t.abs().max()


def test_six_products_keep_float32s_accuracy():
    """Left out are products of 2^-9 and 2^-18 of a value each, 2^-27 and less, rms."""
    assert off(PAIRS) < 2.0**-26


@pytest.mark.parametrize("dropped", PAIRS)
def test_the_bars_show_every_pair(dropped):
    loss = off([p for p in PAIRS if p != dropped])
    for rows, D, F, *_ in SIZES:
        b = bars(rows, D, F)
        assert loss > max(b["dx"], b["dwg"], b["dwu"]), (rows, D, F)
        assert 2**0.5 * loss > b["y"], (rows, D, F)  # both a and b are off
