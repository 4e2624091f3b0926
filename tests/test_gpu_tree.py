"""Drafted-token tree operators on the GPU (include/tvara_kernels.h
tvara_tree_plan, tvara_tree_attention, tvara_tree_commit) against their plain
64-bit forms in tests/tree_cases.py."""

import ctypes as C

import numpy as np
import pytest

from tests import tree_cases as T
from tvara_b200 import _bindings as B

pytestmark = pytest.mark.gpu


def sync():
    import torch
    torch.cuda.synchronize()


def check(lib, status):
    assert status == 0, lib.tvara_last_error().decode()


# ------------------------------------------------------------------ attention
SHAPES = [  # heads, kv_heads, head_dim
    (9, 3, 64), (32, 8, 128), (8, 2, 32), (4, 4, 128), (7, 1, 64), (6, 2, 80), (3, 1, 96), (2, 2, 17), (4, 2, 256),
    (5, 5, 8), (10, 2, 128),
]


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("heads,kv_heads,d", SHAPES)
def test_attention_shapes(capi, kv, heads, kv_heads, d):
    rng = np.random.default_rng(heads * 1000 + d)
    T.AttentionCase(rng, kv, [0, 1, 77, 128, 300], [3, 1, 17, 2, 40], heads, kv_heads, d).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("bt", [1, 3, 8, 16, 24, 64, 200])
def test_attention_block_sizes(capi, kv, bt):
    rng = np.random.default_rng(bt)
    T.AttentionCase(rng, kv, [255, 33, 0], [5, 31, 1], 8, 2, 64, bt=bt).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("n", [1, 2, 32, 33, 63, 64, 65, 128])
def test_attention_edges(capi, kv, length, n):
    rng = np.random.default_rng(length * 131 + n)
    T.AttentionCase(rng, kv, [length], [n], 4, 1, 64, spare_rows=1).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
def test_attention_masks(capi, kv, masks):
    rng = np.random.default_rng(5)
    T.AttentionCase(rng, kv, [0, 40, 0, 200], [70, 20, 1, 130], 8, 2, 128, masks=masks).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_attention_many_ragged_sequences(capi, kv):
    rng = np.random.default_rng(6)
    lengths = [int(x) for x in rng.integers(0, 700, 40)]
    nodes = [int(x) for x in rng.integers(0, 20, 40)]
    nodes[0] = nodes[17] = nodes[39] = 0
    T.AttentionCase(rng, kv, lengths, nodes, 8, 2, 64).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_attention_large_trees_long_context(capi, kv):
    rng = np.random.default_rng(7)
    T.AttentionCase(rng, kv, [5000, 3], [300, 1024], 4, 2, 128, bt=32).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("pad", [4, 3])
def test_attention_strided_rows(capi, kv, pad):
    """Padded rows; pad 3 leaves rows unaligned for wide loads."""
    rng = np.random.default_rng(8)
    T.AttentionCase(rng, kv, [100, 31], [9, 12], 8, 2, 64, pad=pad).upload().run(capi).check()


def test_attention_mask_words_wider_than_needed(capi):
    rng = np.random.default_rng(9)
    T.AttentionCase(rng, "f16", [50, 10], [9, 12], 8, 2, 64, max_nodes=700).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_attention_masked_node_holds_nan_or_infinity(capi, kv):
    """A node's NaN or infinite K and V reach only the rows that attend to it."""
    rng = np.random.default_rng(10)
    c = T.AttentionCase(rng, kv, [90, 0], [40, 20], 8, 2, 128, masks="any")
    bad = []
    for s, node, value in ((0, 7, np.nan), (0, 33, np.inf), (1, 2, -np.inf)):
        slot = c.slots[c.cu[s] + node]
        c.pool[slot // c.bt, 1, :, :, slot % c.bt] = value
        bad.append((s, node))
    c.upload().run(capi)
    got = c.dev.get("out")
    want, tol = c.want()  # computed without the bad values: only rows that do not see them count
    width = c.heads * c.d
    for s in range(2):
        for i in range(c.nodes[s]):
            if any(s == bs and c.mask[s][i, c.lengths[s] + j] for bs, j in bad):
                assert not np.isfinite(got[c.cu[s] + i, :width]).any()
            else:
                r = c.cu[s] + i
                assert (np.abs(got[r] - want[r]) <= tol[r]).all()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_attention_bad_blocks_count_as_masked(capi, kv):
    """A table entry or slot outside the pool: reported, and the rest unharmed."""
    rng = np.random.default_rng(11)
    c = T.AttentionCase(rng, kv, [100, 64], [9, 12], 8, 2, 64)
    c.tables[0, 2] = 1 << 30
    c.mask[0][:, 32:48] = False
    c.slots[c.cu[1] + 4] = 1 << 40
    c.mask[1][:, 64 + 4] = False
    c.upload().run(capi)
    want, tol = c.want()
    assert (np.abs(c.dev.get("out") - want) <= tol).all()
    assert c.dev.get("status")[0] == 1


def test_attention_bad_lengths_skip_the_sequence(capi):
    rng = np.random.default_rng(12)
    c = T.AttentionCase(rng, "f16", [100, 64, 30], [9, 12, 5], 8, 2, 64)
    good = list(c.lengths)
    c.lengths = [100, 1 << 20, -3]
    c.upload().run(capi)
    c.lengths = good
    want, tol = c.want()
    got = c.dev.get("out")
    assert (np.abs(got - want)[:9] <= tol[:9]).all()
    assert (got[9:] == 123.0).all()
    assert c.dev.get("status")[0] == 2


def test_attention_repeats_bit_for_bit_on_another_stream(capi):
    import torch
    rng = np.random.default_rng(13)
    c = T.AttentionCase(rng, "f16", [3000, 500], [30, 64], 32, 8, 128).upload().run(capi)
    sync()
    one = c.dev.get("out").copy()
    c.dev.keep["out"].fill_(7)
    stream = torch.cuda.Stream()
    sync()
    c.run(capi, stream.cuda_stream)
    stream.synchronize()
    assert np.array_equal(c.dev.get("out")[:94], one[:94])
    c.dev.keep["out"].copy_(torch.from_numpy(c.out))
    c.run(capi).check()


def test_attention_captured_with_changing_lengths(capi):
    """One captured launch replayed with other lengths, masks and queries."""
    import torch
    rng = np.random.default_rng(14)
    cases = [T.AttentionCase(np.random.default_rng(s), "f16", lengths, [5, 20, 3], 8, 2, 128, bt=16, max_nodes=20)
             for s, lengths in ((1, [700, 40, 300]), (2, [20, 900, 120]))]
    first = cases[0].upload()
    room = max(c.dev.a.max_blocks for c in cases)
    stride = max(c.stride for c in cases)
    pool = torch.zeros((room,) + first.pool.shape[1:], dtype=torch.float16, device="cuda")
    tables = torch.zeros(3, stride, dtype=torch.int32, device="cuda")
    first.dev.set(pool=pool, tables=tables, max_blocks=room, table_stride=stride)
    size = capi.tvara_tree_attention_workspace(first.dev.by)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        check(capi, capi.tvara_tree_attention(first.dev.by, work.data_ptr(), size,
                                              torch.cuda.current_stream().cuda_stream))
    for c in cases + cases[:1]:
        pool[:len(c.pool)].copy_(torch.from_numpy(c.pool))
        tables[:, :c.stride].copy_(torch.from_numpy(c.tables))
        for name, value in (("q", c.q), ("out", c.out), ("lengths", np.asarray(c.lengths, np.int32)),
                            ("cu_nodes", c.cu), ("slots", c.slots), ("ancestors", c.words.view(np.int64))):
            first.dev.keep[name].copy_(torch.from_numpy(value))
        graph.replay()
        sync()
        got = first.dev.get("out")
        want, tol = c.want()
        assert (np.abs(got - want) <= tol).all()
    del graph


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("bt", [8, 16, 32, 48, 128, 12])
def test_attention_wide_heads_by_block_size(capi, kv, bt):
    """head_dim 128 with boxes of 8, 16 and 32 rows, and a size with none."""
    rng = np.random.default_rng(100 + bt)
    T.AttentionCase(rng, kv, [700, 129, 64], [33, 5, 40], 8, 2, 128, bt=bt, layers=3).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("n_seq", [513, 2000])
def test_attention_more_sequences_than_threads(capi, kv, n_seq):
    rng = np.random.default_rng(n_seq)
    lengths = [int(x) for x in rng.integers(0, 40, n_seq)]
    nodes = [int(x) for x in rng.integers(0, 4, n_seq)]
    T.AttentionCase(rng, kv, lengths, nodes, 4, 2, 64, layers=1, layer=0).upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_attention_one_long_sequence(capi, kv):
    """One item cut into pieces for every SM."""
    rng = np.random.default_rng(15)
    T.AttentionCase(rng, kv, [30000], [3], 4, 1, 64, layers=1, layer=0).upload().run(capi).check()


@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-6, 1, 1), (30, 1, 1), (1e-12, 1e12, 1e10), (1, 1, 1e-12)])
def test_attention_f32_magnitudes(capi, q_scale, k_scale, v_scale):
    """F32 values far outside F16's range: every row has its own power of two."""
    rng = np.random.default_rng(16)
    c = T.AttentionCase(rng, "f32", [300, 20], [20, 33], 8, 2, 64, q_scale=q_scale)
    rows = np.exp(rng.uniform(-3, 3, c.pool.shape[0] * c.pool.shape[4])).reshape(c.pool.shape[0], 1, 1, c.pool.shape[4], 1)
    rows = np.exp2(np.round(np.log2(rows))).astype(np.float32)  # uneven rows, by powers of two
    c.pool[:, :, 0] *= (k_scale * rows).astype(np.float32)
    c.pool[:, :, 1] *= (v_scale * rows).astype(np.float32)
    for s, length in enumerate(c.lengths):
        p = np.arange(length)
        slot = np.concatenate([c.tables[s][p // c.bt].astype(np.int64) * c.bt + p % c.bt, c.slots[c.cu[s]:c.cu[s + 1]]])
        for kind, to in ((0, c.k), (1, c.v)):
            to[s] = np.moveaxis(c.pool[slot // c.bt, 1, kind, :, slot % c.bt].astype(np.float64), 1, 0)
    c.upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_attention_and_commit_beyond_32_bit_offsets(capi, kv):
    """Blocks more than 2^32 bytes (and 2^32 elements of int8) into the pool."""
    import torch
    rng = np.random.default_rng(17)
    c = T.AttentionCase(rng, kv, [100, 33], [9, 20], 8, 2, 128, bt=16, layers=2)
    per_block = int(np.prod(c.pool.shape[1:]))
    far = (1 << 32) // per_block + 7
    blocks = far + len(c.pool)
    pool = torch.empty((blocks,) + c.pool.shape[1:], dtype=torch.from_numpy(c.pool).dtype, device="cuda")
    pool[far:].copy_(torch.from_numpy(c.pool))
    c.tables[c.tables >= 0] += far
    c.slots[c.slots >= 0] += far * c.bt
    c.upload()
    c.dev.set(pool=pool, max_blocks=blocks)
    scales = None
    if kv == "i8":
        scales = torch.empty((blocks,) + c.scales.shape[1:], device="cuda")
        scales[far:].copy_(torch.from_numpy(c.scales))
        c.dev.set(kv_scales=scales)
    c.run(capi).check()
    # move node 5's row of sequence 0 over node 0's
    dev = T.Dev(B.TreeCommitArgs, kv_dtype=T.KV[kv][0], kv_heads=2, head_dim=128, block_tokens=16, layers=2, n_seq=1,
                capacity=9, max_nodes=9, max_blocks=blocks)
    parents = np.full(9, -1, np.int32)
    dev.set(lengths=np.array([100], np.int32), cu_nodes=np.array([0, 9], np.int32), parents=parents,
            tokens=np.arange(9, dtype=np.uint32), choices=np.full(9, 77, np.uint32), first=np.array([5], np.uint32),
            slots=c.slots[:9].copy(), pool=pool, path=np.zeros(9, np.int32), accepted=np.zeros(1, np.int32),
            next=np.zeros(1, np.uint32), lengths_out=np.zeros(1, np.int32), status=np.zeros(1, np.int32))
    if scales is not None:
        dev.set(kv_scales=scales)
    check(capi, capi.tvara_tree_commit(dev.by, None))
    assert dev.get("accepted")[0] == 1 and dev.get("status")[0] == 0
    a, b = c.slots[5] - far * 16, c.slots[0]
    want = c.pool[a // 16, :, :, :, a % 16]
    assert np.array_equal(pool[int(b // 16), :, :, :, int(b % 16)].cpu().numpy().view(np.uint8), want.view(np.uint8))


def test_attention_shared_prefix_and_shared_slots(capi):
    """Sequences that share cached blocks, and nodes that share a slot."""
    rng = np.random.default_rng(18)
    c = T.AttentionCase(rng, "f16", [64, 64, 80], [9, 9, 4], 8, 2, 128, masks="any")
    c.tables[1, :4] = c.tables[0, :4]
    c.k[1][:, :64], c.v[1][:, :64] = c.k[0][:, :64], c.v[0][:, :64]
    c.slots[c.cu[0] + 3] = c.slots[c.cu[0] + 8]
    c.k[0][:, 64 + 3], c.v[0][:, 64 + 3] = c.k[0][:, 64 + 8], c.v[0][:, 64 + 8]
    c.upload().run(capi).check()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("bt", [16, 12])
def test_attention_alternating_tree_sizes(capi, kv, bt):
    """Neighbouring sequences with one and with two tiles of query vectors, few
    positions each, so that a CTA changes between the two many times; repeated
    calls agree bit for bit."""
    rng = np.random.default_rng(19)
    nodes = [64 if i % 2 else 3 for i in range(120)]
    lengths = [int(x) for x in rng.integers(0, 300, 120)]
    c = T.AttentionCase(rng, kv, lengths, nodes, 8, 2, 128, bt=bt, layers=1, layer=0).upload().run(capi)
    c.check()
    first = c.dev.get("out").copy()
    for _ in range(20):
        c.dev.keep["out"].zero_()
        c.run(capi)
        assert np.array_equal(c.dev.get("out")[:c.total], first[:c.total])


def test_attention_calls_on_two_streams(capi):
    """Concurrent calls, each with its own workspace and status."""
    import torch
    cases = [T.AttentionCase(np.random.default_rng(s), kv, [900, 40], [20, 64], 8, 2, 128).upload()
             for s, kv in ((1, "f16"), (2, "i8"), (3, "f32"), (4, "f16"))]
    streams = [torch.cuda.Stream() for _ in cases]
    sync()
    for _ in range(3):
        for c, s in zip(cases, streams):
            c.run(capi, s.cuda_stream)
            c.hold = getattr(c, "hold", []) + [c.workspace]
    sync()
    for c in cases:
        c.check()


def test_attention_refuses_an_unaligned_workspace(capi):
    import torch
    c = T.AttentionCase(np.random.default_rng(1), "f16", [9], [2], 4, 2, 64).upload()
    size = capi.tvara_tree_attention_workspace(c.dev.by)
    work = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    assert capi.tvara_tree_attention(c.dev.by, work.data_ptr() + 4, size, None) == -1
    assert b"aligned" in capi.tvara_last_error()


# ----------------------------------------------------------------------- plan
def plan_case(rng, lengths, nodes, bt, tree, spare_free=5, extra_held=0, max_nodes=None, spare_rows=2):
    n_seq = len(lengths)
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    held = np.array([-(-a // bt) + (int(rng.integers(0, extra_held + 1)) if extra_held else 0) for a in lengths],
                    np.int32)
    need = [max(0, -(-(a + b) // bt) - h) for a, b, h in zip(lengths, nodes, held)]
    stride = max(1, max(int(h) + x for h, x in zip(held, need)))
    blocks = int(held.sum()) + sum(need) + spare_free
    ids = rng.permutation(blocks).astype(np.int32)
    tables = np.full((n_seq, stride), -1, np.int32)
    at = 0
    for s in range(n_seq):
        tables[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    free = np.concatenate([ids[at:], np.full(3, -9, np.int32)])  # entries behind the count are no blocks
    count = blocks - at
    parents = None
    if tree:
        parents = np.concatenate([T.random_tree(rng, n) for n in nodes] + [np.full(spare_rows, 99, np.int32)])
    most = max_nodes or max(1, max(nodes))
    words = -(-most // 64)
    rows = int(cu[-1]) + spare_rows
    d = T.Dev(B.TreePlanArgs, block_tokens=bt, n_seq=n_seq, capacity=rows, max_nodes=most,
              max_blocks=blocks, table_stride=stride, free_capacity=len(free))
    d.set(lengths=np.asarray(lengths, np.int32), held=held, cu_nodes=cu, free_blocks=free,
          free_count=np.array([count], np.int32), tables=tables, slots=np.full(rows, -5, np.int64),
          positions=np.full(rows, -5, np.int32), held_out=np.zeros(n_seq, np.int32),
          free_left=np.zeros(1, np.int32), status=np.zeros(1, np.int32))
    if tree:
        d.set(parents=parents, ancestors=np.full((rows, words), 0x55, np.uint64))
    want = T.plan(np.asarray(lengths), held, cu, parents, tables, free, count, bt)
    return d, want, cu, words


def check_plan(d, want, cu, words, tree):
    total = int(cu[-1])
    assert d.get("status")[0] == 0
    assert np.array_equal(d.get("tables"), want["tables"])
    assert np.array_equal(d.get("slots")[:total], want["slots"]) and (d.get("slots")[total:] == -5).all()
    assert np.array_equal(d.get("positions")[:total], want["positions"]) and (d.get("positions")[total:] == -5).all()
    assert np.array_equal(d.get("held_out"), want["held"])
    assert d.get("free_left")[0] == want["free_left"]
    if tree:
        got = d.get("ancestors").view(np.uint64)
        for s, m in enumerate(want["masks"]):
            if len(m):
                assert np.array_equal(got[cu[s]:cu[s + 1]], T.mask_words(m, words)), s
        assert (got[total:] == 0x55).all()


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("bt", [1, 16, 24])
@pytest.mark.parametrize("n_seq,top,nodes", [(1, 0, 1), (1, 40, 26), (7, 90, 64), (33, 500, 65), (200, 60, 5), (3, 50, 1024)])
def test_plan(capi, tree, bt, n_seq, top, nodes):
    rng = np.random.default_rng(n_seq * 7 + nodes)
    lengths = rng.integers(0, top + 1, n_seq).tolist()
    counts = rng.integers(0, nodes + 1, n_seq).tolist()
    counts[0] = nodes
    d, want, cu, words = plan_case(rng, lengths, counts, bt, tree)
    check(capi, capi.tvara_tree_plan(d.by, None))
    check_plan(d, want, cu, words, tree)
    check(capi, capi.tvara_tree_plan(d.by, None))  # inputs are not consumed: the same step again
    check_plan(d, want, cu, words, tree)


def test_plan_chain_of_parents_is_a_triangle(capi):
    rng = np.random.default_rng(3)
    d, want, cu, words = plan_case(rng, [5], [300], 16, True)
    chain = T.random_tree(rng, 300, chain=True)
    d.set(parents=np.concatenate([chain, np.zeros(2, np.int32)]))
    check(capi, capi.tvara_tree_plan(d.by, None))
    got = d.get("ancestors").view(np.uint64)[:300]
    assert np.array_equal(got, T.mask_words(np.tril(np.ones((300, 300), bool)), words))
    assert np.array_equal(d.get("positions")[:300], 5 + np.arange(300))


def test_plan_most_sequences_and_held_blocks_are_used_first(capi):
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 100, 8192).tolist()
    nodes = rng.integers(0, 9, 8192).tolist()
    d, want, cu, words = plan_case(rng, lengths, nodes, 16, True, extra_held=2)
    check(capi, capi.tvara_tree_plan(d.by, None))
    check_plan(d, want, cu, words, True)


def test_plan_prompt_rows_beyond_a_trees_limit(capi):
    rng = np.random.default_rng(5)
    d, want, cu, words = plan_case(rng, [0, 7, 4000], [5000, 1, 3001], 16, False)
    check(capi, capi.tvara_tree_plan(d.by, None))
    check_plan(d, want, cu, words, False)


def test_plan_counts_in_place_and_captured(capi):
    """held_out = held and free_left = free_count: a captured step that grows
    its own tables from replay to replay."""
    import torch
    rng = np.random.default_rng(6)
    d, _, cu, words = plan_case(rng, [10, 0, 33], [7, 20, 1], 16, True, spare_free=40)
    stride = 12
    tables = np.full((3, stride), -1, np.int32)
    old = d.get("tables")
    tables[:, :old.shape[1]] = old
    d.set(tables=tables, table_stride=stride)
    d.set(held_out=d.keep["held"], free_left=d.keep["free_count"])
    held, count, lengths = d.get("held").copy(), int(d.get("free_count")[0]), d.get("lengths").copy()
    free, parents = d.get("free_blocks"), d.get("parents")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        check(capi, capi.tvara_tree_plan(d.by, torch.cuda.current_stream().cuda_stream))
    for _ in range(3):
        want = T.plan(lengths, held, cu, parents[:cu[-1]], tables, free, count, 16)
        graph.replay()
        sync()
        assert np.array_equal(d.get("tables"), want["tables"])
        assert np.array_equal(d.get("slots")[:cu[-1]], want["slots"])
        assert np.array_equal(d.get("held"), want["held"]) and d.get("free_count")[0] == want["free_left"]
        tables, held, count = want["tables"], want["held"], want["free_left"]
        lengths = lengths + np.diff(cu)  # every drafted row kept
        d.keep["lengths"].copy_(torch.from_numpy(lengths.astype(np.int32)))
    del graph


@pytest.mark.parametrize("fault,bit", [("blocks", 4), ("decreasing", 2), ("rows", 2), ("negative", 2), ("held", 2),
                                       ("table", 2), ("count", 2), ("nodes", 2)])
def test_plan_refused_on_the_device_writes_nothing(capi, fault, bit):
    rng = np.random.default_rng(7)
    d, _, cu, words = plan_case(rng, [20, 3, 50], [9, 30, 12], 16, True)
    edit = {"blocks": ("free_count", 0, 1), "decreasing": ("cu_nodes", 1, 45), "rows": ("cu_nodes", 3, 60),
            "negative": ("lengths", 1, -1), "held": ("held", 0, 1), "table": ("lengths", 2, 5000),
            "count": ("free_count", 0, 1000), "nodes": None}[fault]
    if edit:
        d.keep[edit[0]][edit[1]] = edit[2]
    else:
        d.set(max_nodes=20)
    before = {name: d.get(name).copy() for name in ("tables", "slots", "positions", "ancestors", "held_out", "free_left")}
    check(capi, capi.tvara_tree_plan(d.by, None))
    sync()
    assert d.get("status")[0] == bit
    for name, was in before.items():
        assert np.array_equal(d.get(name), was), name


def test_plan_bad_parents_and_blocks_are_reported(capi):
    rng = np.random.default_rng(8)
    d, want, cu, words = plan_case(rng, [20, 3], [9, 30], 16, True)
    d.keep["parents"][3] = 3
    d.keep["parents"][5] = -2
    d.keep["parents"][9 + 4] = 29
    d.keep["tables"][0, 1] = 1 << 20
    check(capi, capi.tvara_tree_plan(d.by, None))
    assert d.get("status")[0] == 1 | 8
    assert (d.get("slots")[:9] == -1).all() and (d.get("slots")[9:39] >= 0).all()
    assert d.get("positions")[3] == 20 and d.get("positions")[5] == 20 and d.get("positions")[9 + 4] == 3


# --------------------------------------------------------------------- commit
def commit_case(rng, kv, nodes, layers, kv_heads, d, bt, in_place, first=True, spare_rows=2, keep_going=0.85,
                twins=False):
    n_seq = len(nodes)
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    total = int(cu[-1])
    rows = total + spare_rows
    parents = np.concatenate([T.random_tree(rng, n) for n in nodes] + [np.full(spare_rows, 99, np.int32)])
    tokens = rng.integers(0, 1000, rows).astype(np.uint32)
    choices = rng.integers(2000, 3000, rows).astype(np.uint32)
    firsts = rng.integers(2000, 3000, n_seq).astype(np.uint32)
    for s, n in enumerate(nodes):  # a path of matches down each tree
        p, at = parents[cu[s]:cu[s + 1]], -1
        while True:
            kids = [c for c in range(n) if p[c] == at]
            if not kids or rng.random() > keep_going:
                break
            kid = kids[int(rng.integers(len(kids)))]
            if twins:
                tokens[cu[s] + np.array(kids)] = tokens[cu[s] + kid]
            if at < 0:
                firsts[s] = tokens[cu[s] + kid]
            else:
                choices[cu[s] + at] = tokens[cu[s] + kid]
            at = kid
    per = [-(-n // bt) + 1 for n in nodes]
    blocks = 2 * sum(per) + 1
    ids = rng.permutation(blocks)
    slots, dest = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    at = 0
    for s, n in enumerate(nodes):
        for to in (slots, dest):
            mine = ids[at:at + per[s]].astype(np.int64)
            at += per[s]
            p = int(rng.integers(bt)) + np.arange(n)
            to[cu[s]:cu[s + 1]] = mine[p // bt] * bt + p % bt
    shape = (blocks, layers, 2, kv_heads, bt, d)
    if kv == "i8":
        pool = rng.integers(-127, 128, shape).astype(np.int8)
    else:
        pool = rng.standard_normal(shape).astype(T.KV[kv][1])
    scales = rng.random(shape[:-1]).astype(np.float32) if kv == "i8" else None
    dev = T.Dev(B.TreeCommitArgs, kv_dtype=T.KV[kv][0], kv_heads=kv_heads, head_dim=d, block_tokens=bt, layers=layers,
                n_seq=n_seq, capacity=rows, max_nodes=max(1, max(nodes)), max_blocks=blocks)
    lengths = rng.integers(0, 5000, n_seq).astype(np.int32)
    dev.set(lengths=lengths, cu_nodes=cu, parents=parents, tokens=tokens, choices=choices, slots=slots, pool=pool,
            path=np.full(rows, -5, np.int32), accepted=np.full(n_seq, -5, np.int32),
            next=np.zeros(n_seq, np.uint32), lengths_out=np.zeros(n_seq, np.int32), status=np.zeros(1, np.int32))
    if first:
        dev.set(first=firsts)
    if scales is not None:
        dev.set(kv_scales=scales)
    if not in_place:
        dev.set(dest=dest)
    want_pool, want_scales = pool.copy(), None if scales is None else scales.copy()
    want = dict(path=np.full(rows, -5, np.int32), accepted=[], next=[])
    for s, n in enumerate(nodes):
        r = slice(cu[s], cu[s + 1])
        path, nxt = T.walk(parents[r], tokens[r], choices[r], int(firsts[s]) if first else None)
        want["path"][r] = -1
        want["path"][cu[s]:cu[s] + len(path)] = path
        want["accepted"].append(len(path))
        want["next"].append(nxt)
        for k, node in enumerate(path):
            f, t = slots[cu[s] + node], (slots if in_place else dest)[cu[s] + k]
            want_pool[t // bt, ..., t % bt, :] = pool[f // bt, ..., f % bt, :]
            if scales is not None:
                want_scales[t // bt, ..., t % bt] = scales[f // bt, ..., f % bt]
    want.update(pool=want_pool, kv_scales=want_scales, lengths_out=lengths + np.array(want["accepted"]))
    return dev, want


def check_commit(dev, want, status=0):
    assert dev.get("status")[0] == status
    assert np.array_equal(dev.get("path"), want["path"])
    assert dev.get("accepted").tolist() == want["accepted"]
    assert dev.get("next").view(np.uint32).tolist() == want["next"]
    assert np.array_equal(dev.get("lengths_out"), want["lengths_out"])
    assert np.array_equal(dev.get("pool"), want["pool"])
    if want["kv_scales"] is not None:
        assert np.array_equal(dev.get("kv_scales"), want["kv_scales"])


@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("nodes,layers,kv_heads,d,bt", [
    ([1], 1, 1, 64, 16), ([26], 3, 3, 64, 16), ([0, 5, 64, 1, 33, 0], 2, 8, 128, 16), ([70, 130], 2, 2, 17, 8),
    ([9, 14], 2, 1, 6, 1), ([40, 3], 1, 2, 5, 24), ([1024, 300], 1, 1, 32, 64)])
def test_commit(capi, kv, in_place, nodes, layers, kv_heads, d, bt):
    rng = np.random.default_rng(sum(nodes) + d)
    dev, want = commit_case(rng, kv, nodes, layers, kv_heads, d, bt, in_place, keep_going=0.97)
    check(capi, capi.tvara_tree_commit(dev.by, None))
    check_commit(dev, want)


def test_commit_without_first_accepts_node_zero(capi):
    rng = np.random.default_rng(3)
    dev, want = commit_case(rng, "f16", [12, 0, 30], 2, 2, 64, 16, True, first=False)
    check(capi, capi.tvara_tree_commit(dev.by, None))
    check_commit(dev, want)
    assert want["accepted"][0] >= 1 and want["accepted"][1] == 0 and want["next"][1] == T.NONE


def test_commit_equal_siblings_take_the_lowest(capi):
    rng = np.random.default_rng(4)
    dev, want = commit_case(rng, "f32", [40, 64, 17], 1, 2, 32, 16, False, twins=True)
    check(capi, capi.tvara_tree_commit(dev.by, None))
    check_commit(dev, want)


def test_commit_long_chain_closes_up_in_place(capi):
    """A path longer than one batch of rows, moved over its own sources."""
    rng = np.random.default_rng(5)
    n = 200
    dev, _ = commit_case(rng, "f32", [n], 2, 2, 16, 16, True)
    parents = np.concatenate([np.array([-1, -1] + [i - 2 for i in range(2, n)], np.int32), np.full(2, 99, np.int32)])
    tokens = np.arange(n + 2, dtype=np.uint32)
    choices = np.concatenate([np.arange(2, n + 2, dtype=np.uint32), np.zeros(2, np.uint32)])
    choices[n - 1] = T.NONE  # a non-finite row's argmax: the walk ends there
    dev.set(parents=parents, tokens=tokens, choices=choices, first=np.array([1], np.uint32))
    pool, slots = dev.get("pool").copy(), dev.get("slots")
    check(capi, capi.tvara_tree_commit(dev.by, None))
    path = np.arange(1, n, 2)
    assert dev.get("accepted")[0] == len(path) and np.array_equal(dev.get("path")[:len(path)], path)
    assert dev.get("next").view(np.uint32)[0] == T.NONE
    want = pool.copy()
    for k, node in enumerate(path):
        want[slots[k] // 16, :, :, :, slots[k] % 16] = pool[slots[node] // 16, :, :, :, slots[node] % 16]
    assert np.array_equal(dev.get("pool"), want)


def test_commit_bad_parents_slots_and_lengths_are_reported(capi):
    rng = np.random.default_rng(6)
    dev, want = commit_case(rng, "f16", [30, 20, 10], 2, 2, 64, 16, False, keep_going=1.0)
    dev.keep["cu_nodes"][3] = 1 << 20  # the last sequence reaches behind the rows
    path0 = want["path"][0]
    dev.keep["slots"][int(path0)] = -1
    dev.keep["parents"][30 + 19] = 40
    pool = dev.get("pool").copy()
    check(capi, capi.tvara_tree_commit(dev.by, None))
    assert dev.get("status")[0] == 1 | 2 | 8
    assert dev.get("accepted")[0] == want["accepted"][0] and dev.get("accepted")[2] == -5
    t = dev.get("dest")[0]
    assert np.array_equal(dev.get("pool")[t // 16, :, :, :, t % 16], pool[t // 16, :, :, :, t % 16])


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_commit_next_over_first_and_lengths_in_place(capi, kv):
    """Many slices per sequence, all walking from `first` while `next` replaces it."""
    for seed in range(5):
        rng = np.random.default_rng(30 + seed)
        dev, want = commit_case(rng, kv, [40, 64, 3], 16, 8, 128, 16, True, keep_going=1.0)
        dev.set(next=dev.keep["first"], lengths_out=dev.keep["lengths"])
        check(capi, capi.tvara_tree_commit(dev.by, None))
        check_commit(dev, want)


def test_commit_without_a_pool_only_walks(capi):
    rng = np.random.default_rng(7)
    dev, want = commit_case(rng, "f16", [30, 20], 2, 2, 64, 16, True)
    pool, before = dev.keep["pool"], dev.get("pool").copy()
    dev.set(pool=None, slots=None)
    dev.set(lengths_out=dev.keep["lengths"])
    check(capi, capi.tvara_tree_commit(dev.by, None))
    assert np.array_equal(dev.get("path"), want["path"]) and np.array_equal(dev.get("lengths"), want["lengths_out"])
    assert np.array_equal(pool.cpu().numpy(), before)


# ------------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["f32", "f16", "i8"])
def test_speculative_steps_equal_the_plain_continuation(capi, kv):
    """Plan, K/V of the drafts into their slots, attention, choices, commit,
    captured once and replayed for several steps on its own device state: the
    cache, lengths and emitted tokens equal a host model that keeps each
    sequence's accepted K and V rows as lists."""
    import torch
    rng = np.random.default_rng(20)
    heads, kv_heads, d, bt, n_seq, n = 8, 2, 64, 16, 3, 12
    layers, layer = 1, 0
    total = n_seq * n
    blocks, stride = 64, 16
    cu = np.arange(n_seq + 1, dtype=np.int32) * n
    i8 = kv == "i8"
    pool = torch.zeros(blocks, layers, 2, kv_heads, bt, d, dtype=getattr(torch, {"f32": "float32", "f16": "float16",
                                                                                "i8": "int8"}[kv]), device="cuda")
    scales = torch.zeros(blocks, layers, 2, kv_heads, bt, device="cuda") if i8 else None
    lengths = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    held = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    count = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    shared = dict(lengths=lengths, cu_nodes=cu, status=status)
    plan = T.Dev(B.TreePlanArgs, block_tokens=bt, n_seq=n_seq, capacity=total, max_nodes=n, max_blocks=blocks,
                 table_stride=stride, free_capacity=blocks)
    plan.set(held=held, held_out=held, free_count=count, free_left=count,
             free_blocks=rng.permutation(blocks).astype(np.int32), tables=np.full((n_seq, stride), -1, np.int32),
             parents=np.full(total, -1, np.int32), slots=np.zeros(total, np.int64), positions=np.zeros(total, np.int32),
             ancestors=np.zeros((total, 1), np.uint64), **shared)
    att = T.Dev(B.TreeAttentionArgs, kv_dtype=T.KV[kv][0], heads=heads, kv_heads=kv_heads, head_dim=d, block_tokens=bt,
                layers=layers, layer=layer, n_seq=n_seq, capacity=total, max_nodes=n, max_blocks=blocks,
                table_stride=stride, q_stride=heads * d, out_stride=heads * d)
    att.set(q=np.zeros((total, heads * d), np.float32), out=np.zeros((total, heads * d), np.float32), pool=pool,
            tables=plan.keep["tables"], slots=plan.keep["slots"], ancestors=plan.keep["ancestors"], **shared)
    com = T.Dev(B.TreeCommitArgs, kv_dtype=T.KV[kv][0], kv_heads=kv_heads, head_dim=d, block_tokens=bt, layers=layers,
                n_seq=n_seq, capacity=total, max_nodes=n, max_blocks=blocks)
    first = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    com.set(parents=plan.keep["parents"], tokens=np.zeros(total, np.uint32), choices=np.zeros(total, np.uint32),
            first=first, slots=plan.keep["slots"], pool=pool, path=np.zeros(total, np.int32),
            accepted=np.zeros(n_seq, np.int32), next=first, lengths_out=lengths, **shared)
    if i8:
        att.set(kv_scales=scales)
        com.set(kv_scales=scales)
    fresh = torch.zeros(total, 2, kv_heads, d, dtype=pool.dtype, device="cuda")
    fresh_scales = torch.zeros(total, 2, kv_heads, device="cuda")
    head = torch.from_numpy(rng.standard_normal((heads * d, 3)).astype(np.float32)).cuda()  # three token ids
    size = capi.tvara_tree_attention_workspace(att.by)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        check(capi, capi.tvara_tree_plan(plan.by, s))
        slots = plan.keep["slots"]
        pool[slots // bt, layer, :, :, slots % bt] = fresh
        if i8:
            scales[slots // bt, layer, :, :, slots % bt] = fresh_scales
        check(capi, capi.tvara_tree_attention(att.by, work.data_ptr(), size, s))
        com.keep["choices"].copy_((att.keep["out"] @ head).argmax(1))
        check(capi, capi.tvara_tree_commit(com.by, s))

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    keep = [x.clone() for x in (lengths, held, count, pool, plan.keep["tables"], first)]
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    for x, was in zip((lengths, held, count, pool, plan.keep["tables"], first), keep):
        x.copy_(was)
    if i8:
        scales.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    model = [([], []) for _ in range(n_seq)]  # accepted K and V rows
    head_h = head.double().cpu().numpy()
    moved = 0
    for _ in range(6):
        parents = np.concatenate([T.random_tree(rng, n) for _ in range(n_seq)])
        tokens = rng.integers(0, 3, total).astype(np.int32)  # often equal to a choice
        q = rng.standard_normal((total, heads * d)).astype(np.float32)
        if i8:
            x = rng.integers(-127, 128, (total, 2, kv_heads, d)).astype(np.int8)
            sc = (rng.random((total, 2, kv_heads)) * 0.03 + 0.001).astype(np.float32)
            fresh_scales.copy_(torch.from_numpy(sc))
            real = x.astype(np.float64) * sc[..., None]
        else:
            x = rng.standard_normal((total, 2, kv_heads, d)).astype(T.KV[kv][1])
            real = x.astype(np.float64)
        fresh.copy_(torch.from_numpy(x))
        plan.keep["parents"].copy_(torch.from_numpy(parents))
        com.keep["tokens"].copy_(torch.from_numpy(tokens))
        att.keep["q"].copy_(torch.from_numpy(q))
        firsts = com.get("next").copy()
        graph.replay()
        sync()
        assert int(status.item()) == 0
        out, choices = att.get("out"), com.get("choices")
        for s in range(n_seq):
            r = slice(cu[s], cu[s + 1])
            k_rows, v_rows = model[s]
            mask = np.concatenate([np.ones((n, len(k_rows)), bool), T.ancestors(parents[r])], 1)
            k = np.concatenate([np.array(k_rows).reshape(-1, kv_heads, d), real[r, 0]]).transpose(1, 0, 2)
            v = np.concatenate([np.array(v_rows).reshape(-1, kv_heads, d), real[r, 1]]).transpose(1, 0, 2)
            o, tol = T.attention(q[r].reshape(n, heads, d), k, v, mask, heads // kv_heads, kv == "f32")
            assert (np.abs(out[r].reshape(n, heads, d) - o) <= tol).all()
            logits = o.reshape(n, -1) @ head_h
            # the device's choice is the largest logit, up to rounding of a near tie
            mine = choices[r]
            assert (logits[np.arange(n), mine] >= logits.max(1) - 1e-2).all()
            path, nxt = T.walk(parents[r], tokens[r], mine, int(firsts[s]))
            assert com.get("accepted")[s] == len(path) and int(com.get("next")[s]) == nxt
            for node in path:
                k_rows.append(real[cu[s] + node, 0])
                v_rows.append(real[cu[s] + node, 1])
            moved += len(path)
            assert int(lengths[s]) == len(k_rows)
    assert moved > 5
    # the cache holds exactly the accepted rows
    tables = plan.get("tables")
    for s in range(n_seq):
        p = np.arange(len(model[s][0]))
        b, o = tables[s][p // bt], p % bt
        got = pool.cpu().numpy()[b, layer, :, :, o].astype(np.float64)
        if i8:
            got = got * scales.cpu().numpy()[b, layer, :, :, o].astype(np.float64)[..., None]
        assert np.array_equal(got[:, 0], np.array(model[s][0]).reshape(-1, kv_heads, d))
        assert np.array_equal(got[:, 1], np.array(model[s][1]).reshape(-1, kv_heads, d))
    del graph
