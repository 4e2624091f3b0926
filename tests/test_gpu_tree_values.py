"""Tree attention on values that stretch its F16 operands: rows of zeros, rows
far above or below the others, seen or masked."""

import numpy as np
import pytest

from tests import tree_bounds
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


LARGE = [1e4, 1e8, 1e10, 1e12, 1e20, 1e30]


@pytest.mark.parametrize("kv", ["f32", "i8"])
@pytest.mark.parametrize("large", LARGE)
def test_masked_node_with_large_values(capi, kv, large):
    """A node that most rows do not see holds finite V far above the rest."""
    rng = np.random.default_rng(52)
    c = T.AttentionCase(rng, kv, [90, 0, 300], [40, 20, 7], 8, 2, 128, masks="any")
    for s, node in ((0, 7), (0, 33), (1, 2), (2, 6)):
        length = c.lengths[s]
        c.mask[s][:, length + node] = False
        c.mask[s][node, length + node] = True  # itself only
        row = rng.integers(-127, 128, c.d) if kv == "i8" else rng.standard_normal(c.d) * large
        for kind in (0, 1):
            set_row(c, s, length + node, kind, row, large)
        r = slice(c.cu[s], c.cu[s + 1])
        c.words[r] = T.mask_words(c.mask[s][:, length:], c.words.shape[1])
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


def test_masked_node_with_nan_scales(capi):
    rng = np.random.default_rng(53)
    c = T.AttentionCase(rng, "i8", [90, 0], [40, 20], 8, 2, 64, masks="any")
    unseen = []
    for s, node, scale in ((0, 7, np.nan), (0, 33, np.inf), (1, 2, -np.inf)):
        c.mask[s][:, c.lengths[s] + node] = False
        slot = c.slots[c.cu[s] + node]
        c.scales[slot // c.bt, 1, :, :, slot % c.bt] = scale
        unseen.append((s, c.lengths[s] + node))
    for s, index in unseen:
        c.k[s][:, index] = c.v[s][:, index] = 0
        c.words[c.cu[s]:c.cu[s + 1]] = T.mask_words(c.mask[s][:, c.lengths[s]:], c.words.shape[1])
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


@pytest.mark.parametrize("kv", ["f32", "i8"])
@pytest.mark.parametrize("large", LARGE)
def test_seen_position_of_large_values_and_no_weight(capi, kv, large):
    """Cached positions with V far above the rest and scores far below: what
    they add is small, and the others keep their digits."""
    rng = np.random.default_rng(54)
    c = T.AttentionCase(rng, kv, [90, 700], [9, 30], 8, 2, 64)
    c.q = np.abs(c.q)
    far = 1.6 * (np.log(large) + 10) / (0.8 * 1.5 * 8)  # scores near -1.6 (ln large + 10)
    for s, index in ((0, 5), (0, 64), (1, 3), (1, 699)):
        set_row(c, s, index, 0, -127 if kv == "i8" else -far, far / 127)
        row = rng.integers(-127, 128, c.d) if kv == "i8" else rng.standard_normal(c.d) * large
        set_row(c, s, index, 1, row, large / 127)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-28, 1e28, 1), (1e28, 1e-28, 1e-20), (1e-20, 1e20, 1e36)])
@pytest.mark.parametrize("d", [64, 128])
def test_f32_extreme_magnitudes(capi, q_scale, k_scale, v_scale, d):
    """Ordinary scores from factors far from one."""
    rng = np.random.default_rng(56)
    c = T.AttentionCase(rng, "f32", [300, 20], [20, 33], 8, 2, d, q_scale=q_scale)
    c.pool[:, :, 0] *= np.float32(k_scale)
    c.pool[:, :, 1] *= np.float32(v_scale)
    for s, length in enumerate(c.lengths):
        p = np.arange(length)
        slot = np.concatenate([c.tables[s][p // c.bt].astype(np.int64) * c.bt + p % c.bt, c.slots[c.cu[s]:c.cu[s + 1]]])
        for kind, to in ((0, c.k), (1, c.v)):
            to[s] = np.moveaxis(c.pool[slot // c.bt, 1, kind, :, slot % c.bt].astype(np.float64), 1, 0)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


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


@pytest.mark.parametrize("times", [300, 3000])
@pytest.mark.parametrize("side", ["k", "v", "both"])
@pytest.mark.parametrize("d", [64, 128])
def test_f32_outlier_channel(capi, times, side, d):
    """One channel far above the others, as keys of trained models have: the
    other channels keep the digits of their own size."""
    rng = np.random.default_rng(55)
    lengths, nodes = [0, 2, 40, 300], [1, 1, 20, 30]
    c = T.AttentionCase(rng, "f32", lengths, nodes, 8, 2, d, q_scale=0.01 if side == "v" else 1.5)
    c.q.reshape(-1, 8, d)[:, :, 5] /= times  # scores stay ordinary
    for kind, name, to in ((0, "k", c.k), (1, "v", c.v)):
        if side in (name, "both"):
            c.pool[:, :, kind, ..., 5] *= np.float32(times)
            for s, length in enumerate(lengths):
                p = np.arange(length)
                slot = np.concatenate([c.tables[s][p // c.bt].astype(np.int64) * c.bt + p % c.bt, c.slots[c.cu[s]:c.cu[s + 1]]])
                to[s] = np.moveaxis(c.pool[slot // c.bt, 1, kind, :, slot % c.bt].astype(np.float64), 1, 0)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


@pytest.mark.parametrize("kv,scale", [("f32", 0), ("i8", 0.0), ("i8", 1.0), ("i8", 1e6)])
@pytest.mark.parametrize("v_size", [1, 1e-5])
@pytest.mark.parametrize("strength", [1, 3, 8])
def test_row_of_zeros_with_all_the_weight(capi, kv, scale, v_size, strength):
    """A position whose V is zero (codes of zero with any scale) takes nearly all
    of every row's weight; what is left keeps its digits."""
    rng = np.random.default_rng(58)
    c = T.AttentionCase(rng, kv, [90, 700, 3], [9, 30, 4], 8, 2, 64)
    c.q = np.abs(c.q)
    if kv == "i8":
        c.scales[:, :, 1] *= np.float32(v_size)
    else:
        c.pool[:, :, 1] *= np.float32(v_size)
    for s, length in enumerate(c.lengths):
        p = np.arange(length)
        slot = np.concatenate([c.tables[s][p // c.bt].astype(np.int64) * c.bt + p % c.bt, c.slots[c.cu[s]:c.cu[s + 1]]])
        v = c.pool[slot // c.bt, 1, 1, :, slot % c.bt].astype(np.float64)
        if kv == "i8":
            v = v * c.scales[slot // c.bt, 1, 1, :, slot % c.bt].astype(np.float64)[..., None]
        c.v[s] = np.moveaxis(v, 1, 0)
    for s, index in ((0, 5), (1, 3), (1, 699), (2, 1)):
        set_row(c, s, index, 0, 127 if kv == "i8" else strength, strength / 127)
        set_row(c, s, index, 1, 0, scale)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


@pytest.mark.parametrize("kv", ["f32", "i8"])
@pytest.mark.parametrize("large", [1e11, 1e18, 1e30])
@pytest.mark.parametrize("lengths", [[100], [40, 2000], [130, 30], [20000]])
def test_weight_on_zeros_beside_large_values(capi, kv, large, lengths):
    """Nodes share the weight but have V zero, and the tiles before hold V of up
    to 1e30: sums of weights and of products are in units far apart, within a
    stream, between streams and between the parts of a cut item."""
    rng = np.random.default_rng(59)
    c = T.AttentionCase(rng, kv, lengths, [128] * len(lengths), 4, 2, 64, masks="any", q_scale=0.3)
    for s, length in enumerate(lengths):
        row = rng.integers(-127, 128, c.d) if kv == "i8" else rng.standard_normal(c.d) * large
        for index in range(min(length, 300)):
            set_row(c, s, index, 1, row, large / 100)
        for node in range(128):
            set_row(c, s, length + node, 1, 0, 1.0)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)


@pytest.mark.parametrize("kv", ["f32", "i8"])
@pytest.mark.parametrize("lengths", [[100], [40, 2000], [20000]])
def test_values_of_all_sizes(capi, kv, lengths):
    """V from 1e-18 to 1e18 among positions of like weight."""
    rng = np.random.default_rng(64)
    c = T.AttentionCase(rng, kv, lengths, [33] * len(lengths), 4, 2, 64, masks="any", q_scale=0.3)
    for s, length in enumerate(lengths):
        for index in range(min(length, 500)):
            size = 10.0 ** rng.uniform(-18, 18)
            row = rng.integers(-127, 128, c.d) if kv == "i8" else rng.standard_normal(c.d) * size
            set_row(c, s, index, 1, row, size / 100)
    tree_bounds.check_case(c.upload().run(capi), tree_bounds.rows_and_bound_by_element)
