"""Refusals of the drafted-token tree calls that the host makes before any
device work (no GPU needed: nothing is launched)."""

import ctypes as C

import pytest

from tvara_b200 import _bindings as B

SOME = 1 << 20  # a pointer that is never followed


def filled(struct, **fields):
    a = struct()
    a.struct_size = C.sizeof(struct)
    for name, kind in struct._fields_:
        if kind is C.c_void_p:
            setattr(a, name, SOME)
    for i, name in enumerate(n for n, k in struct._fields_ if k is C.c_void_p):
        setattr(a, name, SOME * (i + 1))  # apart from one another
    for name, value in fields.items():
        setattr(a, name, value)
    return a


def plan(**fields):
    return filled(B.TreePlanArgs, **dict(dict(block_tokens=16, n_seq=4, capacity=100, max_nodes=64, max_blocks=50,
                                              table_stride=8, free_capacity=10), **fields))


def attention(**fields):
    return filled(B.TreeAttentionArgs, **dict(dict(
        kv_dtype=1, heads=8, kv_heads=2, head_dim=64, block_tokens=16, layers=2, layer=1, n_seq=4, capacity=100,
        max_nodes=64, max_blocks=50, table_stride=8, q_stride=512, out_stride=512), **fields))


def commit(**fields):
    return filled(B.TreeCommitArgs, **dict(dict(kv_dtype=1, kv_heads=2, head_dim=64, block_tokens=16, layers=2,
                                                n_seq=4, capacity=100, max_nodes=64, max_blocks=50), **fields))


def refused(lib, status, text):
    assert status != 0 and text in lib.tvara_last_error().decode()


SIZES = [(dict(n_seq=0), "sequences"), (dict(n_seq=8193), "sequences"), (dict(capacity=1 << 31), "capacity"),
         (dict(max_nodes=0), "nodes"), (dict(max_nodes=1025), "nodes"), (dict(max_blocks=0), "pool size"),
         (dict(max_blocks=1 << 31), "pool size"), (dict(block_tokens=0), "pool size"), (dict(struct_size=8), "arguments"),
         (dict(lengths=None), "arguments"), (dict(cu_nodes=None), "arguments"), (dict(status=None), "arguments")]


@pytest.mark.parametrize("fields,text", SIZES + [
    (dict(parents=None), "go together"), (dict(ancestors=None), "go together"), (dict(table_stride=0), "table width"),
    (dict(slots=None), "arguments"), (dict(free_blocks=None), "arguments"), (dict(held_out=SOME + 4), "overlap"),
    (dict(held_out=2 * SOME + 4), "overlap"), (dict(free_left=2 * SOME), "overlap"),
    (dict(held_out=3 * SOME + 16), "overlap"), (dict(free_left=SOME), "overlap"), (dict(free_left=6 * SOME + 2), "overlap")])
def test_plan_refusals(capi, fields, text):
    refused(capi, capi.tvara_tree_plan(C.byref(plan(**fields)), None), text)


def test_null_arguments(capi):
    refused(capi, capi.tvara_tree_plan(None, None), "arguments")
    refused(capi, capi.tvara_tree_commit(None, None), "arguments")
    refused(capi, capi.tvara_tree_attention(None, None, 0, None), "arguments")
    assert capi.tvara_tree_attention_workspace(None) == 0


@pytest.mark.parametrize("fields,text", SIZES + [
    (dict(kv_dtype=3), "dtype"), (dict(kv_dtype=2, kv_scales=None), "scales"), (dict(heads=7), "geometry"),
    (dict(kv_heads=0), "geometry"), (dict(head_dim=0), "geometry"), (dict(head_dim=257), "geometry"),
    (dict(layer=2), "geometry"), (dict(table_stride=0), "geometry"), (dict(q_stride=511), "shorter"),
    (dict(out_stride=511), "shorter"), (dict(q=None), "arguments"), (dict(out=None), "arguments"),
    (dict(pool=None), "arguments"), (dict(slots=None), "arguments"), (dict(tables=None), "arguments")])
def test_attention_refusals(capi, fields, text):
    refused(capi, capi.tvara_tree_attention(C.byref(attention(**fields)), C.c_void_p(SOME), 1 << 40, None), text)


def test_attention_workspace_is_required(capi):
    a = attention()
    size = capi.tvara_tree_attention_workspace(C.byref(a))
    assert size > 0
    refused(capi, capi.tvara_tree_attention(C.byref(a), None, size, None), "workspace")
    refused(capi, capi.tvara_tree_attention(C.byref(a), C.c_void_p(SOME), size - 1, None), "workspace")
    assert capi.tvara_tree_attention(C.byref(attention(capacity=0)), C.c_void_p(SOME), size, None) == 0  # no rows


@pytest.mark.parametrize("fields,text", SIZES + [
    (dict(kv_dtype=3), "dtype"), (dict(kv_dtype=2, kv_scales=None), "scales"), (dict(kv_heads=0), "geometry"),
    (dict(head_dim=0), "geometry"), (dict(layers=0), "geometry"), (dict(layers=65535, head_dim=65535), "geometry"),
    (dict(slots=None), "geometry"), (dict(parents=None), "arguments"), (dict(tokens=None), "arguments"),
    (dict(choices=None), "arguments"), (dict(path=None), "arguments"), (dict(accepted=None), "arguments"),
    (dict(next=None), "arguments"), (dict(lengths_out=None), "arguments"),
    (dict(next=SOME), "overlap"), (dict(next=6 * SOME + 4), "overlap"), (dict(accepted=6 * SOME), "overlap"),
    (dict(lengths_out=SOME + 8), "overlap"), (dict(accepted=2 * SOME + 16), "overlap")])
def test_commit_refusals(capi, fields, text):
    refused(capi, capi.tvara_tree_commit(C.byref(commit(**fields)), None), text)


# Arrays are read by their own types: an address off by half of one would fault on the device.
@pytest.mark.parametrize("call,fields", [
    ("plan", dict(lengths=SOME + 2)), ("plan", dict(tables=7 * SOME + 2)), ("plan", dict(slots=8 * SOME + 4)),
    ("plan", dict(ancestors=10 * SOME + 4)), ("plan", dict(status=13 * SOME + 1)),
    ("attention", dict(q=SOME + 2)), ("attention", dict(out=2 * SOME + 2)), ("attention", dict(pool=3 * SOME + 1)),
    ("attention", dict(kv_dtype=0, pool=3 * SOME + 2)), ("attention", dict(kv_dtype=2, kv_scales=4 * SOME + 2)),
    ("attention", dict(slots=8 * SOME + 4)), ("attention", dict(ancestors=9 * SOME + 4)),
    ("attention", dict(cu_nodes=7 * SOME + 3)),
    ("commit", dict(tokens=4 * SOME + 2)), ("commit", dict(slots=7 * SOME + 4)), ("commit", dict(dest=8 * SOME + 4)),
    ("commit", dict(pool=9 * SOME + 1)), ("commit", dict(kv_dtype=2, kv_scales=10 * SOME + 2)),
    ("commit", dict(path=11 * SOME + 2))])
def test_misaligned_arrays(capi, call, fields):
    if call == "attention":
        status = capi.tvara_tree_attention(C.byref(attention(**fields)), C.c_void_p(SOME), 1 << 40, None)
    else:
        status = {"plan": capi.tvara_tree_plan, "commit": capi.tvara_tree_commit}[call](
            C.byref({"plan": plan, "commit": commit}[call](**fields)), None)
    refused(capi, status, "aligned")


@pytest.mark.parametrize("name", ["parents", "tokens", "choices"])
def test_commit_path_apart_from_what_the_walk_reads(capi, name):
    at = [n for n, k in B.TreeCommitArgs._fields_ if k is C.c_void_p].index(name) + 1
    refused(capi, capi.tvara_tree_commit(C.byref(commit(path=at * SOME + 396)), None), "overlap")
    refused(capi, capi.tvara_tree_commit(C.byref(commit(path=at * SOME - 396)), None), "overlap")


# Rows of 512 floats out of 100; q begins at SOME.
@pytest.mark.parametrize("fields", [
    dict(out=SOME), dict(out=SOME + 2044), dict(out=SOME - 2044), dict(out=SOME + 99 * 2048 + 2044),
    dict(q_stride=1024, out_stride=1024, out=SOME + 2044), dict(q_stride=1024, out_stride=1024, out=SOME + 5 * 4096 - 2044),
    dict(q_stride=1024, out_stride=1028, out=SOME + 2048)])
def test_attention_out_apart_from_q(capi, fields):
    refused(capi, capi.tvara_tree_attention(C.byref(attention(**fields)), C.c_void_p(50 * SOME), 1 << 40, None), "overlap")


# Column slices of one buffer are apart: such a call is refused only for its missing workspace.
@pytest.mark.parametrize("fields", [
    dict(q_stride=1024, out_stride=1024, out=SOME + 2048), dict(q_stride=1024, out_stride=1024, out=SOME - 2048),
    dict(q_stride=1536, out_stride=1536, out=SOME + 4096), dict(out=SOME + 100 * 2048), dict(out=SOME - 100 * 2048)])
def test_attention_out_beside_q(capi, fields):
    refused(capi, capi.tvara_tree_attention(C.byref(attention(**fields)), None, 0, None), "workspace")
