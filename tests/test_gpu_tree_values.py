"""Tree attention on values that stretch its F16 operands: rows of zeros, rows
far above or below the others, seen or masked."""

import numpy as np
import pytest

from tests import tree_cases as T

pytestmark = pytest.mark.gpu


def set_row(c, s, index, kind, row, scale=None):
    """K (kind 0) or V (1) of index `index` (cached positions, then nodes) of
    sequence s, every KV head, in the pool and in the case's 64-bit copy."""
    length = c.lengths[s]
    slot = int(c.slots[c.cu[s] + index - length]) if index >= length else \
        int(c.tables[s][index // c.bt]) * c.bt + index % c.bt
    c.pool[slot // c.bt, 1, kind, :, slot % c.bt] = row
    value = np.broadcast_to(row, (c.kv_heads, c.d)).astype(c.pool.dtype).astype(np.float64)
    if c.scales is not None:
        c.scales[slot // c.bt, 1, kind, :, slot % c.bt] = scale
        value = value * np.float64(np.float32(scale))
    (c.k, c.v)[kind][s][:, index] = value


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_zeros(capi, kv, d):
    """Positions whose K, V or both are zero count with their weights."""
    rng = np.random.default_rng(50)
    c = T.AttentionCase(rng, kv, [300, 70, 5], [20, 9, 3], 8, 2, d)
    for s, index in ((0, 7), (0, 8), (0, 64), (0, 299), (0, 300), (0, 311), (1, 0), (1, 71), (2, 0), (2, 6)):
        set_row(c, s, index, 1, 0, 0.02)
        if index % 2:
            set_row(c, s, index, 0, 0, 0.02)
    c.upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_all_values_zero(capi, kv):
    rng = np.random.default_rng(51)
    c = T.AttentionCase(rng, kv, [40, 0], [5, 3], 8, 2, 64)
    for s in range(2):
        for index in range(c.lengths[s] + c.nodes[s]):
            set_row(c, s, index, 1, 0, 0.0)
    c.upload().run(capi).check()
    assert (c.dev.get("out")[:c.total, :c.heads * c.d] == 0).all()
