"""Tree attention where one CTA works through many short items one after the
other: items of one and of two tiles of query vectors in turn, whose K/V slots
and Q tiles share memory."""

import numpy as np
import pytest

from tests import tree_bounds
from tests import tree_cases as T

pytestmark = pytest.mark.gpu

# (cached positions, nodes) in turn; four query heads to a KV head, so more than 32 nodes are two tiles of vectors.
# 200 sequences of 8 KV heads are 11 to 14 items to a CTA.  In each pattern a large item is followed by short ones that
# fit the ring's own slots, and only a later one reaches the slots inside the second Q tile.
TURNS = {
    "large_short": [(300, 64), (60, 8)],
    "two_tiles_short": [(190, 64), (60, 8)],
    "large_two_tiny": [(300, 60), (50, 5), (50, 5)],
    "one_tile_large": [(60, 8), (40, 64), (300, 8)],
    "one_tile_large_first": [(40, 40), (400, 8), (20, 3)],
    "large_many_short": [(100, 64), (60, 8), (60, 8), (60, 8), (60, 8)],
}


@pytest.mark.parametrize("turns", TURNS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bt", [16, 12])  # with and without TMA
def test_items_in_turn(capi, turns, d, bt):
    rng = np.random.default_rng(41)
    pattern = TURNS[turns] * (200 // len(TURNS[turns]))
    c = T.AttentionCase(rng, "f16", [a for a, _ in pattern], [n for _, n in pattern], 32, 8, d, bt=bt, layers=1, layer=0)
    c.upload().run(capi)
    tree_bounds.check_case(c)
    first = c.dev.keep["out"][:c.total].clone()
    for _ in range(20):
        c.dev.keep["out"].zero_()
        c.run(capi)
        assert (c.dev.keep["out"][:c.total] == first).all()


@pytest.mark.parametrize("kv", ["f16", "f32", "i8"])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_ragged_short_contexts(capi, kv, seed):
    """A serving batch just after its prompts."""
    rng = np.random.default_rng(seed)
    lengths = [int(x) for x in rng.integers(1, 301, 120)]
    nodes = [int(x) for x in rng.integers(0, 65, 120)]
    c = T.AttentionCase(rng, kv, lengths, nodes, 32, 8, 64, layers=1, layer=0).upload().run(capi)
    if kv == "f16":
        tree_bounds.check_case(c)
    first = c.dev.keep["out"][:c.total].clone()
    assert np.isfinite(first.cpu().numpy()).all()
    for _ in range(10):
        c.dev.keep["out"].zero_()
        c.run(capi)
        assert (c.dev.keep["out"][:c.total] == first).all()
