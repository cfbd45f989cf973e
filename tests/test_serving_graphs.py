"""Host-side checks of the serving programs (no GPU): nodes, shapes, the planner's arena, what the constructors refuse."""
import ctypes as C

import numpy as np
import pytest

from tensorlisp_b200 import _lib
from tensorlisp_b200.graph import BF16, F16, F32, I32, Graph, align256
from tensorlisp_b200.programs import DecoderConfig, TreeDecodeLoop, packed_prefill_step, verify_step

CFG = DecoderConfig(n_layers=3, d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, d_ffn=1024, vocab=2048)


def count(g, op):
    return sum(g.tensors[t].op == op for t in g.nodes)


def arena(dg):
    """The planner takes the graph; the size of its arena."""
    g, keep = dg.graph.to_c()
    offs = np.cumsum([0] + [align256(w.nbytes()) for w in dg.weights]).tolist()
    states = np.cumsum([0] + [align256(b) for b in dg.state_bytes]).tolist()
    nw, ns = len(dg.weights), len(dg.state_bytes)
    leaves = _lib.tlb_leaves((C.c_uint32 * nw)(), (C.c_uint64 * nw)(*offs[:nw]), nw, (C.c_uint64 * ns)(*states[:ns]), ns)
    a, io, n = C.c_uint64(), C.c_uint64(), len(dg.graph.tensors)
    st = _lib.lib().tlb_plan_only(C.byref(g), C.byref(leaves), None, C.byref(a), C.byref(io), (C.c_uint8 * n)(), (C.c_uint64 * n)(), (C.c_int64 * len(dg.graph.nodes))())
    assert st == 0, _lib.lib().tlb_last_error()
    del keep
    return a.value


def test_packed_prefill_graph():
    dg = packed_prefill_step(CFG, 5, 77, 40)
    g = dg.graph
    assert count(g, "PACKED_ATTN") == 3 and count(g, "CUSTOM") == 3 and count(g, "MUL_MAT") == 7 * 3 + 1 and count(g, "FLASH_ATTN_EXT") == 0
    assert g.tensors[dg.logits].ne[:2] == [2048, 5]
    a = next(g.tensors[t] for t in g.nodes if g.tensors[t].op == "PACKED_ATTN")
    assert a.ty == F16 and a.ne == [128, 4, 77, 1] and a.src[4] == -1
    assert g.tensors[a.src[1]].ne == [128, 2, 77, 1] and g.tensors[a.src[3]].ne[0] == 6
    assert dg.state_bytes == [40 * 2 * 16 * 128 * 2] * 6
    assert arena(dg) > 0


def test_verify_graph():
    dg = verify_step(CFG, 4, 8, 100, 60, top=5)
    g = dg.graph
    assert count(g, "PAGED_TREE_ATTENTION") == 3 and count(g, "TOKEN_LOGPROBS") == 1 and count(g, "ARGMAX") == 1
    a = next(g.tensors[t] for t in g.nodes if g.tensors[t].op == "PAGED_TREE_ATTENTION")
    assert a.ty == F16 and a.ne == [128, 4, 8, 4] and a.op_params[1:3] == [2, 16]
    assert [g.tensors[s].ne[:2] for s in a.src[3:7]] == [[7, 4], [4, 1], [4, 1], [8, 4]]
    assert g.tensors[dg.extras["scores"]].ne[:2] == [12, 32] and g.tensors[dg.logits].ne[:2] == [2048, 32]
    assert sorted(dg.inputs.values()) == list(range(8)) and arena(dg) > 0


def test_constructors_refuse():
    g = Graph()
    q, k, at = g.input(F16, [64, 4, 10], "q"), g.input(F16, [64, 3, 10], "k"), g.input(I32, [3], "at")
    with pytest.raises(AssertionError):
        g.packed_attention(q, k, k, at, 0.1)            # 4 heads over 3
    k2 = g.input(BF16, [64, 2, 10], "k2")
    with pytest.raises(AssertionError):
        g.packed_attention(q, k2, k, at, 0.1)           # values of another shape
    with pytest.raises(AssertionError):
        g.packed_attention(q, k2, k2, at, 0.0)
    y = g.token_logprobs(g.input(F32, [100, 7], "x"), None, 3)
    assert g.tensors[y].ne == [8, 7, 1, 1] and g.tensors[y].src[1] == -1


def test_tree_loop_checks_drafts():
    loop = TreeDecodeLoop.__new__(TreeDecodeLoop)       # without a device: what step() checks before it runs anything
    loop.batch, loop.drafts, loop.max_ctx, loop.cfg = 1, 4, 32, CFG
    loop.tables, loop.due, loop.context = np.zeros((1, 2), np.int32), np.array([1], np.int32), np.array([29], np.int32)
    for bad in ([[(5, -1)], []], [[(1, -1), (2, 0), (3, 1), (4, 2)]], [[(1, 0)]], [[(1, -1), (2, 1)]], [[(1, -1), (2, -1), (3, -1)]]):
        with pytest.raises(AssertionError):
            loop.step(bad)
