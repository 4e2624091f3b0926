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
