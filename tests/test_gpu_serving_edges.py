"""The serving operators at the edges of what they take, and with values that are not finite where a query sees them."""
import math

import numpy as np
import pytest
import torch

from tensorlisp_b200 import device_ops as ops
from tensorlisp_b200 import graph as G
from tensorlisp_b200._lib import TlbError
from tensorlisp_b200.native import Native, NativeProgram

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def room(n):
    return torch.full((max(int(n), 16),), 0xCD, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("dtype,first", [(torch.float32, 0), (torch.bfloat16, 0), (torch.float16, 3)], ids=["f32", "bf16", "f16"])
def test_the_largest_vocabulary(native, dtype, first):
    """All but four logits are 60 below or more: their part in the sums, 2^31 e^-60 < 2^-55, is nothing, so the results are those of the four
    alone, to the accuracy of a sum of four (exponents and logarithm: 2^-20)."""
    vocab = 2 ** 31 - 2048
    memory = torch.full((vocab + first,), -57.0, dtype=dtype, device="cuda")
    x = memory[first:].unsqueeze(0)
    at, value = [5, 2 ** 30 + 1, vocab - 600, vocab - 1], [3.0, 2.5, 2.0, 3.0]
    for i, y in zip(at, value):
        x[0, i] = y
    lp, ent, ids, top = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros((1, 4), dtype=torch.int32, device="cuda"), torch.zeros((1, 4), device="cuda")
    ops.token_logprobs(native, x, i32([vocab - 1]), lp, ent, ids, top, workspace=room(ops.token_logprobs_workspace(native, x, 4)), stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    lse = math.log(sum(math.exp(y) for y in value))
    want = sorted((lse - y, i) for i, y in zip(at, value))
    assert ids.tolist() == [[i for _, i in want]]
    assert abs(lp.item() - (3.0 - lse)) < 2.0 ** -20 and abs(ent.item() - sum(math.exp(-d) * d for d, _ in want)) < 2.0 ** -19
    assert np.abs(top.cpu().numpy()[0] + [d for d, _ in want]).max() < 2.0 ** -20


def randn(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def packed(native, q, k, v, q_at, kv_at=None):
    out = torch.full_like(q, 77.0)
    ws = room(ops.packed_attention_workspace(native, q, k, len(q_at) - 1))
    ops.packed_attention(native, q, k, v, i32(q_at), out, kv_offsets=None if kv_at is None else i32(kv_at), workspace=ws, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return out


def tree(native, q, k_pool, v_pool, tables, context, counts, parents):
    out = torch.full_like(q, 77.0)
    ws = room(ops.tree_attention_workspace(native, q, k_pool, tables))
    ops.tree_attention(native, q, k_pool, v_pool, tables, context, counts, parents, out, workspace=ws, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    return out


# Row tiles over many keys are cut between CTAs, so parts of the rows are joined by a launch behind: in the first, third and last of these
SHAPES = [([3000], None), ([40], None), ([300, 1, 200], [4000, 1, 1000]), ([2, 5], [3, 600]), ([1], [20000])]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,keys", SHAPES)
def test_a_query_that_is_no_number(native, lens, keys, D):
    """Every weight of its row is NaN and so is its result; the other rows and heads have theirs, to the last bit."""
    q_at, kv_at = [0] + list(np.cumsum(lens)), [0] + list(np.cumsum(keys or lens))
    q, k, v = randn((q_at[-1], 4, D), 1), randn((kv_at[-1], 1, D), 2), randn((kv_at[-1], 1, D), 3)
    want = packed(native, q, k, v, q_at, kv_at)
    rows = sorted({0, q_at[-1] // 2, q_at[-1] - 1})
    for i in rows:
        q[i, i % 4, D // 3] = float("nan")
        want[i, i % 4] = float("nan")
    out = packed(native, q, k, v, q_at, kv_at)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [10, 3000])
def test_a_draft_that_is_no_number(native, ctx, D):
    pages = -(-(ctx + 8) // 16)
    q, kp, vp = randn((1, 8, 4, D), 4), randn((pages, 2, 16, D), 5), randn((pages, 2, 16, D), 6)
    numbers = i32(np.random.default_rng(7).permutation(pages)[None]), i32([ctx]), i32([8]), i32([[-1, 0, 0, 1, 3, -1, 5, 2]])
    want = tree(native, q, kp, vp, *numbers)
    q[0, 5, 2, 7] = float("nan")
    want[0, 5, 2] = float("nan")
    out = tree(native, q, kp, vp, *numbers)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
@pytest.mark.parametrize("lens,keys", SHAPES + [([5], [3])])
def test_a_query_with_an_infinite_value(native, lens, keys, bad, D):
    """Its scores are infinite, of either sign: the weights are exp(inf - inf), or 0 / 0 where all are -inf. A row that sees nothing is zero all the same."""
    q_at, kv_at = [0] + list(np.cumsum(lens)), [0] + list(np.cumsum(keys or lens))
    q, k, v = randn((q_at[-1], 4, D), 1), randn((kv_at[-1], 1, D), 2), randn((kv_at[-1], 1, D), 3)
    assert (k != 0).all()
    want = packed(native, q, k, v, q_at, kv_at)
    sees = torch.cat([torch.arange(n) + (m - n) >= 0 for n, m in zip(lens, keys or lens)]).cuda()
    for i in sorted({0, q_at[-1] // 2, q_at[-1] - 1}):
        q[i, i % 4, D // 3] = bad
        want[i, i % 4] = float("nan") if sees[i] else 0.0
    out = packed(native, q, k, v, q_at, kv_at)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("behind", [0, 1000])
def test_keys_of_infinite_distance(native, behind, D):
    """Scores of -inf beside others have no weight; where a row has no other, its result is 0 / 0."""
    n = 200
    q, k, v = randn((n, 4, D), 1).abs(), randn((behind + n, 1, D), 2), randn((behind + n, 1, D), 3)
    q[:, :, 5] = 1.0
    k[:behind + 90, 0, 5] = -float("inf")
    want = packed(native, q, k.clamp(min=-65504), v, [0, n], [0, behind + n])
    out = packed(native, q, k, v, [0, n], [0, behind + n])
    assert torch.isnan(out[:90]).all() and torch.equal(out[90:], want[90:])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [10, 3000])
def test_a_draft_whose_scores_are_infinite(native, ctx, D):
    pages = -(-(ctx + 8) // 16)
    q, kp, vp = randn((1, 8, 4, D), 4), randn((pages, 2, 16, D), 5), randn((pages, 2, 16, D), 6)
    numbers = i32(np.random.default_rng(7).permutation(pages)[None]), i32([ctx]), i32([7]), i32([[-1, 0, 0, 1, 3, -1, 5, 2]])
    want = tree(native, q, kp, vp, *numbers)
    assert (want[0, 7] == 0).all()
    q[0, 5, 2, 7], q[0, 7, 1, 7] = float("inf"), float("inf")      # the last one is padding
    want[0, 5, 2] = float("nan")
    out = tree(native, q, kp, vp, *numbers)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])
    kp[:, :, :, 3] = -float("inf")
    q = q.abs().clamp(min=0.5)
    out = tree(native, q, kp, vp, *numbers)
    assert torch.isnan(out[0, :7]).all() and (out[0, 7] == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_result_beside_its_operands(native, D):
    """Queries, keys, values and the result are column blocks of one buffer: no byte of the result is one of theirs."""
    H, Gr, rows = 4, 2, 300
    wide = randn((rows, 2 * H + 2 * Gr, D), 8)
    q, k, v, out = wide[:, :H], wide[:, H:H + Gr], wide[:, H + Gr:H + 2 * Gr], wide[:, H + 2 * Gr:]
    want, before = packed(native, q.contiguous(), k.contiguous(), v.contiguous(), [0, 40, 300]), wide.clone()
    ws = room(ops.packed_attention_workspace(native, q, k, 2))
    go = lambda o: ops.packed_attention(native, q, k, v, i32([0, 40, 300]), o, workspace=ws, stream=torch.cuda.current_stream())  # noqa: E731
    go(out)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(wide[:, :H + 2 * Gr], before[:, :H + 2 * Gr])
    for o in (q, wide[:, H - 1:2 * H - 1], wide[:, 1:H + 1], wide[:, H + 2 * Gr - 1:-1]):
        with pytest.raises(TlbError):
            go(o)


def test_nodes_of_impossible_sizes_are_refused():
    """KV heads x tokens of a page x head size that pass 64 bits, sizes that pass 32: refusals of the compiler."""
    n = Native.load([])
    n.alloc_states([1 << 17, 1 << 17])

    def refused(change, word, block_size=16):
        g = G.Graph()
        q, kc, vc = g.input(G.F16, [16, 4, 8, 2], "q"), g.state(G.F16, [1 << 16], "k"), g.state(G.F16, [1 << 16], "v")
        ins = [g.input(G.I32, x, "x") for x in ([4, 2], [2], [2], [8, 2])]
        y = g.output(g.paged_tree_attention(q, kc, vc, *ins, block_size, 0.25, 4))
        change(g.tensors[y])
        with pytest.raises(TlbError) as e:
            NativeProgram.compile(n, g)
        assert e.value.kind == "Unsupported" and word in str(e.value), str(e.value)

    def kv_heads(x):
        def change(t):
            t.op_params[1] = x
        return change

    refused(kv_heads(1 << 30), "kv heads", 1 << 30)     # 2^64 values a page
    refused(kv_heads(1 << 30), "kv heads", 3)
    refused(kv_heads(0), "kv heads")
    refused(kv_heads(4), "2^31", 1 << 30)
    refused(kv_heads(4), "power of two", 24)
    n.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [8, 64, 72, 128])
def test_head_sizes_up_to_128_are_on_the_tensor_cores(native, D, dtype):
    """The kernel that is not turned off where it does not fit: it alone asks for scratch memory."""
    for rows in (3, 900):
        q, k = torch.empty((rows, 4, D), dtype=dtype, device="cuda"), torch.empty((rows, 2, D), dtype=dtype, device="cuda")
        assert ops.packed_attention_workspace(native, q, k, 1) > 0
    q, kp = torch.empty((2, 4, 4, D), dtype=torch.float16, device="cuda"), torch.empty((9, 2, 16, D), dtype=torch.float16, device="cuda")
    assert ops.tree_attention_workspace(native, q, kp, torch.empty((2, 4), dtype=torch.int32, device="cuda")) > 0
