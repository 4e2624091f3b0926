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


@pytest.mark.parametrize("kv,q_scale,k_scale", [
    ("f32", 1.5, 1e9), ("f32", 1.5, 1e20), ("f32", 1e-3, 1e36), ("f32", 1e9, 1.0), ("f32", 1e34, 1.0), ("f32", 1e20, 1e12),
    ("f16", 1e9, 1.0), ("f16", 1e20, 1.0), ("f16", 1e5, 1e4), ("i8", 1e9, 1.0), ("i8", 1.5, 1e12)])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_any_size(capi, kv, q_scale, k_scale, d):
    """Scores so large that one position takes all the weight: its V comes out,
    whole items and cut ones alike."""
    rng = np.random.default_rng(57)
    c = T.AttentionCase(rng, kv, [300, 20, 3000], [20, 33, 2], 8, 2, d, q_scale=q_scale)
    if kv == "i8":
        c.scales[:, :, 0] *= np.float32(k_scale)
    else:
        c.pool[:, :, 0] *= c.pool.dtype.type(k_scale)
    c.upload().run(capi)
    got = c.dev.get("out").astype(np.float64)
    assert c.dev.get("status")[0] == 0
    clear = 0
    for s, n in enumerate(c.nodes):
        k = c.k[s] * k_scale  # to rounding, far below the gaps that count
        for i in range(n):
            seen = np.flatnonzero(c.mask[s][i])
            for h in range(8):
                q = c.q[c.cu[s] + i, h * d:(h + 1) * d].astype(np.float64)
                scores = k[h // 4][seen] @ q / np.sqrt(d)
                size = (np.abs(k[h // 4][seen]) @ np.abs(q)).max() / np.sqrt(d)
                first, second = np.argsort(scores)[-1], np.sort(scores)[-2:][0]
                row = got[c.cu[s] + i, h * d:(h + 1) * d]
                assert np.isfinite(row).all()
                # 2 d/16 + 1 truncations and the roundings of q and k: below 2^-18 of the sum for d 128
                if scores[first] - second > 2.0 ** -16 * size + 100:
                    clear += 1
                    want = c.v[s][h // 4][seen[first]]
                    # hi + lo parts: 2^-21 of the element (V and weight), 2^-23 of the row's largest
                    assert (np.abs(row - want) <= 2.0 ** -20 * np.abs(want) + 2.0 ** -23 * np.abs(want).max()).all()
    assert clear > 300
