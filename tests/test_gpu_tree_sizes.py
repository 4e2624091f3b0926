"""Sizes that only the device sees: what every form of the tree calls reports
and skips, on the tensor cores and (head_dim 256) beside them."""

import numpy as np
import pytest

from tests import tree_cases as T
from tests.test_gpu_tree import commit_case
from tvara_b200 import _bindings as B

pytestmark = pytest.mark.gpu


def run_and_compare(capi, c, given, skipped, status):
    """`given` replaces device sizes; rows of `skipped` sequences stay as they were."""
    c.upload()
    c.dev.set(**given)
    c.run(capi)
    assert c.dev.get("status")[0] == status
    want, tol = c.want()
    for s in skipped:
        r = slice(c.cu[s], c.cu[s + 1])
        want[r], tol[r] = c.out[r], 0
    assert (np.abs(c.dev.get("out") - want) <= tol).all()


def case(d, nodes=(9, 0, 12, 5)):
    return T.AttentionCase(np.random.default_rng(60), "f16", [100, 40, 64, 30], list(nodes), 8, 2, d)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("length", [-3, 1 << 20, 0x7fffffff])
def test_bad_length_of_an_empty_sequence(capi, d, length):
    c = case(d)
    run_and_compare(capi, c, dict(lengths=np.array([100, length, 64, 30], np.int32)), [], 2)


@pytest.mark.parametrize("d", [64, 256])
def test_bad_length_of_a_sequence(capi, d):
    c = case(d)
    run_and_compare(capi, c, dict(lengths=np.array([100, 40, -1, 30], np.int32)), [2], 2)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("last", [20, -1, 0])
def test_last_offset_too_small(capi, d, last):
    """The last sequence shrinks or goes, and so does what reaches behind it."""
    c = case(d)
    cu = c.cu.copy()
    cu[4] = last
    skipped = [0, 2, 3] if last <= 0 else [2, 3]
    run_and_compare(capi, c, dict(cu_nodes=cu), skipped, 2)


@pytest.mark.parametrize("d", [64, 256])
def test_offset_far_too_large_in_the_middle(capi, d):
    """Neighbours of the wrong offset are skipped, the sequences behind are not."""
    c = case(d, (9, 3, 12, 5))
    cu = c.cu.copy()
    cu[1] = 1000
    run_and_compare(capi, c, dict(cu_nodes=cu), [0, 1], 2)


@pytest.mark.parametrize("d", [64, 256])
def test_first_offset_not_zero(capi, d):
    """Reported; the rows before it are no sequence's."""
    c = T.AttentionCase(np.random.default_rng(61), "f16", [100, 64], [1, 12], 8, 2, d, masks="chain")
    cu = c.cu.copy()
    cu[0] = 1
    run_and_compare(capi, c, dict(cu_nodes=cu), [0], 2)


@pytest.mark.parametrize("d", [64, 256])
def test_empty_sequences_and_spare_rows_are_no_error(capi, d):
    c = T.AttentionCase(np.random.default_rng(62), "f16", [0, 40, 64, 0], [0, 3, 0, 0], 8, 2, d, spare_rows=300)
    run_and_compare(capi, c, {}, [], 0)


@pytest.mark.parametrize("edit,skipped", [((0, 1), []), ((3, 20), [1, 2]), ((3, -1), [0, 1, 2]), ((1, 1000), [0, 1])])
def test_commit_skips_and_reports_the_same(capi, edit, skipped):
    """Sequences of 9, 20 and 5 rows with one wrong offset."""
    rng = np.random.default_rng(63)
    dev, want = commit_case(rng, "f16", [9, 20, 5], 2, 2, 64, 16, False, keep_going=1.0)
    cu = dev.get("cu_nodes").copy()
    cu[edit[0]] = edit[1]
    if edit == (0, 1):
        skipped = [0]  # its nodes moved by one: another tree
    path, answers = dev.get("path").copy(), {name: dev.get(name).copy() for name in ("accepted", "next", "lengths_out")}
    before = dev.get("cu_nodes")
    dev.set(cu_nodes=cu)
    assert capi.tvara_tree_commit(dev.by, None) == 0
    assert dev.get("status")[0] & 2
    for s in range(3):
        r = slice(before[s], before[s + 1])
        if s not in skipped:
            assert np.array_equal(dev.get("path")[r], want["path"][r]) and dev.get("accepted")[s] == want["accepted"][s]
        elif edit != (0, 1):
            assert np.array_equal(dev.get("path")[r], path[r])
            assert all(dev.get(name)[s] == answers[name][s] for name in answers)


@pytest.mark.parametrize("bt", [1 << 20, 1])
def test_plan_of_nearly_two_to_the_31_rows(capi, bt):
    """Row (and, with blocks of one position, block) counts at the end of 32 bits."""
    import torch
    rows = 0x7fffffff
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    blocks = -(-rows // bt)
    free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device="cuda")  # so that block j of the sequence is j
    d = T.Dev(B.TreePlanArgs, block_tokens=bt, n_seq=2, capacity=rows, max_nodes=1, max_blocks=blocks, table_stride=blocks,
              free_capacity=blocks)
    d.set(lengths=np.zeros(2, np.int32), held=np.zeros(2, np.int32), cu_nodes=np.array([0, rows, rows], np.int32),
          free_blocks=free, free_count=np.array([blocks], np.int32), held_out=np.zeros(2, np.int32),
          free_left=np.zeros(1, np.int32), status=np.zeros(1, np.int32),
          tables=torch.full((2 * blocks,), -1, dtype=torch.int32, device="cuda"),
          slots=torch.full((rows,), -1, dtype=torch.int64, device="cuda"),
          positions=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    assert capi.tvara_tree_plan(d.by, None) == 0, capi.tvara_last_error()
    assert d.get("status")[0] == 0 and d.get("held_out").tolist() == [blocks, 0] and d.get("free_left")[0] == 0
    assert torch.equal(d.keep["tables"][:blocks], torch.arange(blocks, dtype=torch.int32, device="cuda"))
    assert (d.keep["tables"][blocks:] == -1).all()
    for at in range(0, rows, 1 << 27):
        want = torch.arange(at, min(at + (1 << 27), rows), device="cuda")
        assert torch.equal(d.keep["slots"][at:at + (1 << 27)], want)
        assert torch.equal(d.keep["positions"][at:at + (1 << 27)], want.int())
    d.keep.clear()
    torch.cuda.empty_cache()
