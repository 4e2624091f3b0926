"""Outputs of the tree calls that meet what the same call reads or writes are
refused (no GPU needed: nothing is launched)."""

import ctypes as C

import pytest

from tests.test_tree_host import SOME, attention, commit, plan, refused
from tvara_b200 import _bindings as B

# bytes of each array in the calls of test_tree_host: 4 sequences, 100 rows, 8 table entries, 10 free blocks
SIZES = {
    "plan": dict(lengths=16, held=16, cu_nodes=20, parents=400, free_blocks=40, free_count=4, tables=128, slots=800,
                 positions=400, ancestors=800, held_out=16, free_left=4, status=4),
    "attention": dict(q=204800, out=204800, pool=819200, tables=128, lengths=16, cu_nodes=20, slots=800, ancestors=800,
                      status=4),
    "commit": dict(lengths=16, cu_nodes=20, parents=400, tokens=400, choices=400, first=16, slots=800, dest=800,
                   pool=819200, path=400, accepted=16, next=16, lengths_out=16, status=4),
}
OUTPUTS = {"plan": ("tables", "slots", "positions", "ancestors", "held_out", "free_left", "status"),
           "attention": ("out", "status"), "commit": ("path", "accepted", "next", "lengths_out", "status", "pool")}
SAME = {("held_out", "held"), ("free_left", "free_count"), ("next", "first"), ("lengths_out", "lengths")}
BUILD = {"plan": (plan, B.TreePlanArgs), "attention": (attention, B.TreeAttentionArgs), "commit": (commit, B.TreeCommitArgs)}
PAIRS = [(call, out, other) for call in SIZES for out in OUTPUTS[call] for other in SIZES[call] if other != out]


def place(struct, name):
    return SOME * ([n for n, k in struct._fields_ if k is C.c_void_p].index(name) + 1)


def run(capi, call, **fields):
    build, _ = BUILD[call]
    a = build(**fields)
    if call == "attention":
        return capi.tvara_tree_attention(C.byref(a), C.c_void_p(SOME * 1000), 1 << 40, None)
    return {"plan": capi.tvara_tree_plan, "commit": capi.tvara_tree_commit}[call](C.byref(a), None)


@pytest.mark.parametrize("call,out,other", PAIRS)
def test_outputs_apart(capi, call, out, other):
    struct = BUILD[call][1]
    base, size = place(struct, other), SIZES[call][other]
    last = base + (size - 1) // 8 * 8
    first = base - (SIZES[call][out] - 1) // 8 * 8 if SIZES[call][out] > 8 else base
    if call == "attention":  # rows of 16-byte pieces
        last, first = base + (size - 1) // 16 * 16, base - (SIZES[call][out] - 1) // 16 * 16 if SIZES[call][out] > 16 else base
    for at in (base, last, first):
        if at == base and (out, other) in SAME:
            continue  # this very array: allowed
        refused(capi, run(capi, call, **{out: at}), "overlap")


@pytest.mark.parametrize("name", list(SIZES["attention"]))
def test_attention_workspace_apart(capi, name):
    a = attention()
    size = capi.tvara_tree_attention_workspace(C.byref(a))
    base = place(B.TreeAttentionArgs, name)
    for at in (base, base + (SIZES["attention"][name] - 1) // 16 * 16, base - size + 16):
        if at > 0:
            refused(capi, capi.tvara_tree_attention(C.byref(a), C.c_void_p(at), size, None), "overlap")


@pytest.mark.parametrize("name", ["out", "status"])
def test_attention_outputs_apart_from_scales(capi, name):
    refused(capi, run(capi, "attention", kv_dtype=2, **{name: place(B.TreeAttentionArgs, "kv_scales")}), "overlap")


@pytest.mark.parametrize("name", ["path", "accepted", "next", "lengths_out", "status"])
def test_commit_outputs_apart_from_scales(capi, name):
    refused(capi, run(capi, "commit", kv_dtype=2, **{name: place(B.TreeCommitArgs, "kv_scales")}), "overlap")


def test_one_array_for_two_outputs(capi):
    """held_out = held is allowed, free_left on top of it is not."""
    held = place(B.TreePlanArgs, "held")
    refused(capi, run(capi, "plan", held_out=held, free_left=held), "overlap")
    first = place(B.TreeCommitArgs, "first")
    refused(capi, run(capi, "commit", next=first, accepted=first), "overlap")


def test_arrays_without_rows_meet_nothing(capi):
    """capacity 0: row arrays may lie anywhere, even inside another."""
    at = place(B.TreeAttentionArgs, "pool") + 160
    a = attention(capacity=0, out=at, q=at, slots=at)
    size = capi.tvara_tree_attention_workspace(C.byref(a))
    assert capi.tvara_tree_attention(C.byref(a), C.c_void_p(SOME * 1000), size, None) == 0
