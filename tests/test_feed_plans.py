"""Which cuts of the feed-forward block's products the rule selects, without a GPU: the GPU's tests have a size for each of them."""

import math
import random

from tests.test_feed_limits import plan
from tests.test_gpu_feed_plans import SIZES

PRODUCTS = ("y", "dx", "dW")


def cuts(rows, D, F):
    """(product, type, edge of the tile, in parts): all that the calls of this size are."""
    found = set()
    for io in (0, 1):
        for train in (0, 1):
            status, plans = plan(rows, D, F, io, train)
            assert status == 0
            for name, (edge, parts, _, _) in zip(PRODUCTS, plans):
                if train or name == "y":
                    found.add((name + (" in training" if train and name == "y" else ""), io, edge, parts > 1))
    return found


def test_the_gpu_tests_have_every_cut():
    """46 ways: three tiles whole and in parts for dx and dW; for y without the largest in parts, and the kernel of few rows in service."""
    tested = set().union(*(cuts(*size[:3]) for size in SIZES))
    rng = random.Random(0)
    sizes = [[round(math.exp(rng.uniform(0, math.log(most)))) for most in (200_000, 5000, 10_000)] for _ in range(4000)]
    selected = set().union(*(cuts(*size) for size in sizes))
    assert selected <= tested, sorted(selected - tested)
    assert len(tested) == 2 * (6 + 6 + 5 + 6)


def test_the_largest_tile_is_tested_with_more_than_a_stage():
    """256 x 256 tiles, 64 k a stage, with remainders of rows, D and F, in both types and every product."""
    large = [(s, c) for s in SIZES for c in cuts(*s[:3]) if c[2] == 256 and not c[3]]
    for product, contraction in (("y", 1), ("y in training", 1), ("dx", 2), ("dW", 0)):
        for io in (0, 1):
            assert any(c[:2] == (product, io) and s[contraction] > 192 and s[0] % 256 and s[1] % 256 and s[2] % 256 for s, c in large), (product, io)
