"""What the calls of the serving operators refuse, without a GPU: every refusal comes before the device is touched, so a block of zeros
stands for the handle and numbers for the addresses."""
import ctypes as C
import math

import pytest

from tensorlisp_b200 import _lib, device_ops as ops
from tensorlisp_b200._lib import TlbError

HANDLE = C.create_string_buffer(1 << 16)
A = [0x100000000 * (i + 1) for i in range(12)]      # addresses far from each other


class Handle:
    ordinal = 0
    L = _lib.lib()
    dev = C.cast(HANDLE, C.c_void_p)


def call(entry, args, word, kind):
    st = getattr(_lib.lib(), entry)(HANDLE, C.byref(args), None)
    assert _lib.STATUS_NAMES[st] == kind and word in _lib.lib().tlb_last_error().decode(), (st, _lib.lib().tlb_last_error())


def packed(**kw):
    a = dict(type=1, seqs=2, heads=4, kv_heads=2, head_size=64, scale=0.125, q_rows=10, kv_rows=10, q=A[0], k=A[1], v=A[2], out=A[3], q_stride=512, k_stride=256,
             v_stride=256, out_stride=512, q_offsets=A[4], workspace=A[5], workspace_bytes=0)
    return _lib.tlb_packed_attention_args(**{**a, **kw})


@pytest.mark.parametrize("kind,word,change", [
    ("Unsupported", "f16 or bf16", dict(type=0)), ("Unsupported", "f16 or bf16", dict(type=26)), ("Unsupported", "head size", dict(head_size=12)),
    ("Unsupported", "head size", dict(head_size=520)), ("Unsupported", "head size", dict(head_size=0)), ("Unsupported", "kv heads", dict(kv_heads=3)),
    ("Unsupported", "kv heads", dict(kv_heads=0)), ("Unsupported", "kv heads", dict(heads=0)), ("Unsupported", "kv heads", dict(heads=2 ** 32 - 1, kv_heads=1)),
    ("Unsupported", "scale", dict(scale=0.0)), ("Unsupported", "scale", dict(scale=-1.0)), ("Unsupported", "scale", dict(scale=math.nan)),
    ("Unsupported", "scale", dict(scale=math.inf)), ("Unsupported", "rows", dict(q_rows=2 ** 31)), ("Unsupported", "rows", dict(kv_rows=2 ** 63)),
    ("Invalid", "null", dict(q=0)), ("Invalid", "null", dict(k=0)), ("Invalid", "null", dict(out=0)), ("Invalid", "null", dict(q_offsets=0)),
    ("Invalid", "16 bytes", dict(q_stride=520)), ("Invalid", "stride", dict(q_stride=496)), ("Invalid", "stride", dict(k_stride=0)), ("Invalid", "16 bytes", dict(v_stride=2 ** 41)),
    ("Invalid", "16-byte", dict(q=A[0] + 8)), ("Invalid", "16-byte", dict(out=A[3] + 2)), ("Invalid", "overlaps", dict(out=A[0])), ("Invalid", "overlaps", dict(out=A[1] + 256)),
    ("Invalid", "overlaps", dict(out=A[2] - 16))])
def test_packed_attention_refuses(kind, word, change):
    call("tlb_packed_attention", packed(**change), word, kind)


def tree(**kw):
    a = dict(seqs=2, drafts=4, heads=4, kv_heads=2, head_size=64, block_size=16, max_blocks=8, scale=0.125, pool_blocks=20, q=A[0], k_pool=A[1], v_pool=A[2], out=A[3],
             tables=A[4], context=A[5], counts=A[6], parents=A[7], workspace=A[8], workspace_bytes=0)
    return _lib.tlb_tree_attention_args(**{**a, **kw})


@pytest.mark.parametrize("kind,word,change", [
    ("Unsupported", "64 drafted", dict(drafts=0)), ("Unsupported", "64 drafted", dict(drafts=65)), ("Unsupported", "power of two", dict(block_size=12)),
    ("Unsupported", "power of two", dict(block_size=0)), ("Unsupported", "power of two", dict(max_blocks=0)), ("Unsupported", "2^31", dict(max_blocks=2 ** 30)),
    ("Unsupported", "pages", dict(pool_blocks=2 ** 40)), ("Unsupported", "kv heads", dict(kv_heads=3)), ("Unsupported", "head size", dict(head_size=20)),
    ("Unsupported", "scale", dict(scale=0.0)), ("Unsupported", "rows", dict(seqs=2 ** 31 - 1, drafts=64)), ("Invalid", "null", dict(parents=0)),
    ("Invalid", "null", dict(v_pool=0)), ("Invalid", "16-byte", dict(k_pool=A[1] + 2)), ("Invalid", "overlaps", dict(out=A[0] + 512)), ("Invalid", "overlaps", dict(out=A[2] + 4096))])
def test_tree_attention_refuses(kind, word, change):
    call("tlb_tree_attention", tree(**change), word, kind)


def keep(**kw):
    pool = 20 * 2 * 16 * 64 * 2
    a = dict(layers=3, seqs=2, drafts=4, kv_heads=2, head_size=64, block_size=16, max_blocks=8, pool_blocks=20, k_pools=A[0], v_pools=A[0] + pool, k_layer_stride=2 * pool,
             v_layer_stride=2 * pool, tables=A[4], context=A[5], counts=A[6], path=A[7])
    return _lib.tlb_cache_keep_args(**{**a, **kw})


@pytest.mark.parametrize("kind,word,change", [
    ("Unsupported", "head size", dict(head_size=4)), ("Unsupported", "64 drafted", dict(drafts=65)), ("Unsupported", "layers", dict(layers=70000)),
    ("Unsupported", "pages", dict(block_size=0)), ("Unsupported", "pages", dict(pool_blocks=2 ** 31)), ("Invalid", "null", dict(path=0)),
    ("Invalid", "16-byte", dict(k_pools=A[0] + 8)), ("Invalid", "16-byte", dict(k_layer_stride=8)), ("Invalid", "overlap", dict(k_layer_stride=16)),
    ("Invalid", "overlap", dict(v_pools=A[0])), ("Invalid", "overlap", dict(v_pools=A[0] + 16)), ("Invalid", "overlap", dict(layers=1, v_pools=A[0], k_layer_stride=0))])
def test_cache_keep_refuses(kind, word, change):
    call("tlb_cache_keep", keep(**change), word, kind)


def scores(**kw):
    a = dict(type=0, top=4, rows=3, vocab=100, logits=A[0], stride=400, tokens=A[1], logprob=A[2], entropy=A[3], top_ids=A[4], top_logprobs=A[5], workspace=A[6],
             workspace_bytes=1 << 20)
    return _lib.tlb_token_logprobs_args(**{**a, **kw})


@pytest.mark.parametrize("kind,word,change", [
    ("Unsupported", "f32, f16 or bf16", dict(type=26)), ("Unsupported", "32", dict(top=33)), ("Unsupported", "tokens", dict(vocab=0)), ("Unsupported", "tokens", dict(vocab=2 ** 31)),
    ("Unsupported", "rows", dict(rows=2 ** 31)), ("Invalid", "null", dict(logits=0)), ("Invalid", "null", dict(top_ids=0)), ("Invalid", "null", dict(logprob=0)),
    ("Invalid", "rows", dict(stride=396)), ("Invalid", "rows", dict(stride=402)), ("Invalid", "rows", dict(logits=A[0] + 2)), ("Invalid", "overlaps", dict(entropy=A[0] + 1100)),
    ("Invalid", "workspace", dict(workspace=0)), ("Invalid", "workspace", dict(workspace_bytes=15)), ("Invalid", "workspace", dict(workspace=A[6] + 4))])
def test_token_logprobs_refuses(kind, word, change):
    call("tlb_token_logprobs", scores(**change), word, kind)


def test_null_arguments_are_errors():
    for entry in ("tlb_packed_attention", "tlb_tree_attention", "tlb_cache_keep", "tlb_token_logprobs"):
        assert getattr(_lib.lib(), entry)(None, C.byref(packed()), None) == _lib.TLB_INVALID
        assert getattr(_lib.lib(), entry)(HANDLE, None, None) == _lib.TLB_INVALID
    for entry in ("tlb_packed_attention_workspace", "tlb_tree_attention_workspace", "tlb_token_logprobs_workspace"):
        assert getattr(_lib.lib(), entry)(HANDLE, None) == 0


def test_nothing_to_do_is_fine():
    for entry, args in (("tlb_packed_attention", packed(seqs=0)), ("tlb_packed_attention", packed(q_rows=0)), ("tlb_tree_attention", tree(seqs=0)),
                        ("tlb_cache_keep", keep(seqs=0)), ("tlb_cache_keep", keep(layers=0)), ("tlb_token_logprobs", scores(rows=0))):
        assert getattr(_lib.lib(), entry)(HANDLE, C.byref(args), None) == _lib.TLB_OK


# ------------------------------------------------------------------------------------------------ the checks of the Python calls
def array(i, shape, typestr, strides=None):
    return ops.DeviceArray(A[i], shape, typestr, strides)


def refused(word, f, *a, **kw):
    with pytest.raises(TlbError) as e:
        f(Handle, *a, **kw)
    assert e.value.kind == "Invalid" and word in str(e.value), str(e.value)


def test_arrays_of_the_wrong_kind_are_refused():
    q, k, at = array(0, (10, 4, 64), "<f2"), array(1, (10, 2, 64), "<f2"), array(2, (3,), "<i4")
    out = array(3, (10, 4, 64), "<f2")
    go = ops.packed_attention
    refused("not an array in device memory", go, [1, 2], k, k, at, out)
    refused("must be f16 or bf16", go, array(0, (10, 4, 64), "<f4"), k, k, at, out)
    refused("3 dimensions", go, array(0, (10, 256), "<f2"), k, k, at, out)
    refused("must be i32", go, q, k, k, array(2, (3,), "<i8"), out)
    refused("dense", go, array(0, (10, 4, 64), "<f2", (1024, 256, 2)), k, k, at, out)
    refused("dense", go, q, k, k, array(2, (3,), "<i4", (8,)), out)
    refused("kv heads, head size", go, q, array(1, (10, 2, 32), "<f2"), array(1, (10, 2, 32), "<f2"), at, out)
    refused("kv heads, head size", go, q, k, array(1, (11, 2, 64), "<f2"), at, out)
    refused("kv heads, head size", go, q, k, k, at, array(3, (9, 4, 64), "<f2"))
    refused("sequences + 1", go, q, k, k, array(2, (0,), "<i4"), out)
    refused("kv_offsets", go, q, k, k, at, out, kv_offsets=array(4, (4,), "<i4"))
    wide = array(0, (1, 2 ** 33, 64), "<f2")
    refused("out of range", go, wide, k, k, at, wide)
    refused("not an array", go, q, k, None, at, out)
    refused("whole elements", go, array(0, (10, 4, 64), "<f2", (513, 128, 2)), k, k, at, out)
    refused("status", go, q, k, k, at, out, status=array(4, (2,), "<i4"))
    x = array(0, (5, 100), "<f4")
    refused("shape", ops.token_logprobs, x, array(1, (4,), "<i4"), array(2, (5,), "<f4"))
    refused("come together", ops.token_logprobs, x, None, None, None, array(1, (5, 2), "<i4"))
    refused("shape", ops.token_logprobs, x, None, None, None, array(1, (5, 2), "<i4"), array(2, (5, 3), "<f4"))
    refused("dense", ops.token_logprobs, array(0, (5, 100), "<f4", (800, 8)), None, array(2, (5,), "<f4"))
    t = dict(q=array(0, (2, 4, 4, 64), "<f2"), p=array(1, (9, 2, 16, 64), "<f2"), tables=array(2, (2, 3), "<i4"), n=array(3, (2,), "<i4"), par=array(4, (2, 4), "<i4"))
    refused("one block-table row", ops.tree_attention, t["q"], t["p"], t["p"], array(2, (3, 3), "<i4"), t["n"], t["n"], t["par"], t["q"])
    refused("parents", ops.tree_attention, t["q"], t["p"], t["p"], t["tables"], t["n"], t["n"], array(4, (2, 5), "<i4"), t["q"])
    refused("4 dimensions", ops.tree_attention, q, t["p"], t["p"], t["tables"], t["n"], t["n"], t["par"], t["q"])
    refused("5 dimensions", ops.cache_keep, t["p"], t["p"], t["tables"], t["n"], t["par"], t["n"])


def test_a_cpu_tensor_is_refused():
    import torch
    refused("another device", ops.token_logprobs, torch.zeros(5, 100), None, array(2, (5,), "<f4"))


@pytest.mark.parametrize("word,entry,args", [
    # rows whose distance in memory does not fit 64 bits
    ("overflow", "tlb_packed_attention", packed(q_rows=2 ** 31 - 512, q_stride=2 ** 39)), ("overflow", "tlb_packed_attention", packed(kv_rows=2 ** 31 - 512, v_stride=2 ** 39)),
    ("overflow", "tlb_token_logprobs", scores(rows=2 ** 31 - 1, stride=2 ** 39)),
    # numbers between two places for numbers
    ("4-byte", "tlb_packed_attention", packed(q_offsets=A[4] + 2)), ("4-byte", "tlb_packed_attention", packed(kv_offsets=A[6] + 1)), ("4-byte", "tlb_packed_attention", packed(status=A[6] + 2)),
    ("4-byte", "tlb_tree_attention", tree(tables=A[4] + 2)), ("4-byte", "tlb_tree_attention", tree(context=A[5] + 2)), ("4-byte", "tlb_tree_attention", tree(counts=A[6] + 2)),
    ("4-byte", "tlb_tree_attention", tree(parents=A[7] + 2)), ("4-byte", "tlb_cache_keep", keep(tables=A[4] + 2)), ("4-byte", "tlb_cache_keep", keep(path=A[7] + 2)),
    ("4-byte", "tlb_cache_keep", keep(counts=A[6] + 2)), ("4-byte", "tlb_cache_keep", keep(context=A[5] + 2)), ("4-byte", "tlb_token_logprobs", scores(tokens=A[1] + 2)),
    ("4-byte", "tlb_token_logprobs", scores(logprob=A[2] + 2)), ("4-byte", "tlb_token_logprobs", scores(top_ids=A[4] + 2)), ("4-byte", "tlb_token_logprobs", scores(top_logprobs=A[5] + 2)),
    # results on top of one another, of the numbers that are read, or of the workspace
    ("overlaps", "tlb_packed_attention", packed(q_offsets=A[3] + 512)), ("overlaps", "tlb_packed_attention", packed(kv_offsets=A[3])), ("overlaps", "tlb_packed_attention", packed(status=A[4] + 8)),
    ("overlaps", "tlb_tree_attention", tree(tables=A[3])), ("overlaps", "tlb_tree_attention", tree(parents=A[3] + 4096 - 4)), ("overlaps", "tlb_tree_attention", tree(status=A[6] + 4)),
    ("overlaps", "tlb_token_logprobs", scores(entropy=A[2] + 8)), ("overlaps", "tlb_token_logprobs", scores(top_ids=A[5] + 44)), ("overlaps", "tlb_token_logprobs", scores(logprob=A[1] + 8)),
    ("overlaps", "tlb_token_logprobs", scores(workspace=A[5] + 32)), ("overlaps", "tlb_token_logprobs", scores(workspace=A[0] + 1184))])
def test_arrays_in_impossible_places(word, entry, args):
    call(entry, args, word, "Invalid")


def test_results_side_by_side_are_fine():
    # what a refusal must not take for an overlap: arrays that touch; the refusal that follows is another one
    call("tlb_token_logprobs", scores(entropy=A[2] + 12, workspace=A[5] + 48, workspace_bytes=16), "workspace of", "Invalid")
    call("tlb_token_logprobs", scores(tokens=A[2] - 12, workspace_bytes=16), "workspace of", "Invalid")
