"""The fused feed-forward block on the GPU against float64 in every way that its products can be cut: each tile, whole and in parts of k, for y in
service and in training, dx, and dWg and dWu, in both types (``test_feed_plans`` pins that these sizes select them all).

Element by element the bars are ``test_gpu_feed``'s. They do not show whether float32 products have all six pairs of parts, so float32 has a bar on
the norm of the error too. Without a pair a product is off by 1.66e-3 squared, 2.7e-6 of its norm, as a bfloat16 is off by 1.66e-3 rms (``test_feed_parts``).
With all of them a sum of n products is off by what its rounding leaves: one for every 16 products, of 2^-24 / sqrt 3 rms of a partial sum whose
mean square is half the last one's, 2^-24 sqrt(n / 96), under 2^-25 sqrt(n / 16); and by 2e-7 for the parts of which products are left out and the
activation. Gradients take a's and b's errors along, at most three times (act', its slope and b)."""

import pytest
import torch

from oracle import feed_oracle
from tests.test_gpu_feed import BF, F32, _check, _inputs

pytestmark = pytest.mark.gpu

# rows, D, F, activation, biases
SIZES = [
    (9001, 768, 1500, "silu", False),
    (6000, 1000, 2049, "gelu", True),
    (17003, 1537, 1030, "sigmoid", True),
    (16385, 1536, 4104, "silu", False),
    (25555, 3457, 36, "gelu", True),
    (31, 69, 34, "silu", True),
    (1248, 3307, 33, "sigmoid", True),
    (647, 1357, 4450, "gelu", False),
    (132, 678, 4186, "silu", True),
    (3242, 71, 5920, "sigmoid", False),
    (5608, 134, 6046, "gelu", True),
]


def sums(n):
    """The error of a float32 sum of n products, relative to the norm of many such sums."""
    return 2e-7 + 2.0**-25 * (n / 16) ** 0.5


def bars(rows, D, F):
    a = sums(D)
    return dict(y=2 * a, **{n: (sums(k) ** 2 + 3 * a**2) ** 0.5 for n, k in (("dx", 2 * F), ("dwg", rows), ("dwu", rows), ("dbg", rows), ("dbu", rows))})


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,D,F,act,bias", SIZES)
def test_every_cut(gpu, rows, D, F, act, bias, dtype):
    x, wg, wu, bg, bu, gy = _inputs((rows,), D, F, dtype, bias, seed=12)
    y, grads = _check(x, wg, wu, bg, bu, gy, act, dtype)
    if dtype == F32:
        want, wgrads, _ = feed_oracle.feed(x, wg, wu, bg, bu, act, gy)
        got = dict(y=y.detach(), **dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), grads)))
        for n, w in zip(("y", "dx", "dwg", "dwu", "dbg", "dbu"), (want, *wgrads)):
            if n in got:
                off = float((got[n].double() - w).norm() / w.norm())
                assert off <= bars(rows, D, F)[n], f"{n}: {off:.2e} of {bars(rows, D, F)[n]:.2e}"


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_the_largest_tile_with_every_activation(gpu, dtype, act):
    x, wg, wu, bg, bu, gy = _inputs((6000,), 1000, 2049, dtype, True, seed=13)
    _check(x, wg, wu, bg, bu, gy, act, dtype)
