"""The serving operators on device arrays against their definitions in 64 bits (numpy), at the sizes and masks where they can go wrong.

Tolerance of attention, with u the type's half step: the weights are rounded to the type once, in the numerator and in the sum that divides
it, and so is the result: |error| <= u |o| + 2 u A with A = sum_j p_j |v_j|. Weights below the type's smallest normal number lose at
most 2^-25 each (f16; the largest weight is 1 or more). Scores are f32 sums of hs products (relative to sum |q k|: hs 2^-24) and exp2 is
good to 2^-22; both enter as a relative error of the weights."""
import ctypes as C

import numpy as np
import pytest
import torch

from tensorlisp_b200 import device_ops as ops
from tensorlisp_b200 import graph as G
from tensorlisp_b200._lib import TlbError
from tensorlisp_b200.native import Native, NativeProgram

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def room(n):
    return torch.full((max(int(n), 16),), 0xCD, dtype=torch.uint8, device="cuda")     # its content does not matter


def randn(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def f64(t):
    return t.double().cpu().numpy()


def attend(q, k, v, seen, scale, u):
    """q [rows, D], k and v [keys, D], seen [rows, keys] -> (result, allowed error), rows that see nothing zero."""
    out, tol = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    for i in range(len(q)):
        at = seen[i]
        if not at.any():
            continue
        s = (k[at] @ q[i]) * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        with np.errstate(invalid="ignore"):
            out[i] = w @ v[at]
            a = w @ np.abs(v[at])
            scores = scale * (np.abs(k[at]) @ np.abs(q[i])).max() * q.shape[1] * 2.0 ** -24 * 2 + np.abs(s).max() * 2.0 ** -22 + 2.0 ** -20
            tol[i] = u * np.abs(out[i]) + (2 * u + 2 * scores) * a + at.sum() * 2.0 ** -25 * np.abs(v[at]).max(0) + 2.0 ** -24
    return out, tol


def check_close(got, want, tol, what):
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine), "%s: %d values are not finite, %d should not be" % (what, (~np.isfinite(got)).sum(), (~fine).sum())
    over = np.abs(got[fine] - want[fine]) - tol[fine]
    assert over.size == 0 or over.max() <= 0, "%s: error %.3e beyond the bound (largest bound %.3e)" % (what, over.max(), tol[fine].max())


# ------------------------------------------------------------------------------------------------ packed sequences
def packed(native, q, k, v, q_at, out, kv_at=None, scale=None, status=None):
    n = len(q_at) - 1
    ws = room(ops.packed_attention_workspace(native, q, k, n))
    ops.packed_attention(native, q, k, v, i32(q_at), out, scale, kv_offsets=None if kv_at is None else i32(kv_at), workspace=ws, status=status, stream=stream())
    torch.cuda.synchronize()


def packed_oracle(q, k, v, q_at, kv_at, scale, u):
    H, Gr = q.shape[1], k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for a, b, c, e in zip(q_at, q_at[1:], kv_at, kv_at[1:]):
        seen = np.arange(e - c)[None, :] <= (np.arange(b - a)[:, None] + (e - c) - (b - a))
        for h in range(H):
            out[a:b, h], tol[a:b, h] = attend(q[a:b, h], k[c:e, h // (H // Gr)], v[c:e, h // (H // Gr)], seen, scale, u)
    return out, tol


def offsets(lens, first=0):
    return [first] + [first + int(n) for n in np.cumsum(lens)]


PACKED = [
    # heads, kv heads, head size, query lengths, key lengths (None: the same)
    (4, 2, 128, [1], None), (4, 1, 128, [37], None), (8, 8, 128, [129, 1, 0, 255], None), (4, 4, 64, [256, 257], None),
    (7, 1, 128, [18, 19, 36, 37, 100], None), (16, 2, 64, [5, 64, 0, 0, 130], None), (12, 4, 96, [43, 42, 85, 86], None), (6, 2, 72, [31, 300], None),
    (2, 1, 8, [70], None), (3, 3, 256, [65, 3], None), (2, 2, 512, [20], None), (4, 2, 136, [33], None), (32, 8, 128, [333], None), (130, 1, 64, [3], None),
    (4, 1, 128, [1, 3, 40], [1000, 129, 40]), (4, 2, 64, [5, 7], [3, 7]), (2, 1, 128, [300, 2], [10, 0]), (8, 2, 128, [64, 65], [700, 2000]),
    (128, 1, 64, [2, 3], [130, 500]), (1, 1, 128, [1], [5000]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", PACKED, ids=lambda c: "%d-%d-%d-%s-%s" % (c[0], c[1], c[2], sum(c[3]), sum(c[4]) if c[4] else "same"))
def test_packed_attention(native, case, dtype):
    H, Gr, D, lens, keys = case
    q_at, kv_at = offsets(lens), offsets(keys if keys else lens)
    q, k, v = randn((q_at[-1], H, D), 1, dtype), randn((kv_at[-1], Gr, D), 2, dtype), randn((kv_at[-1], Gr, D), 3, dtype)
    out = torch.full_like(q, 77.0)
    packed(native, q, k, v, q_at, out, kv_at if keys else None)
    want, tol = packed_oracle(f64(q), f64(k), f64(v), q_at, kv_at, D ** -0.5, U[dtype])
    check_close(f64(out), want, tol, "packed")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_packed_attention_of_strided_rows_and_rows_outside(native, D):
    """q, k and v are columns of one projection's result, the result a column of a wider buffer; rows in front of the first sequence and
    behind the last hold NaN and are neither read nor written."""
    H, Gr, lens, first = 6, 2, [40, 0, 131], 3
    q_at = offsets(lens, first)
    rows = q_at[-1] + 5
    both = randn((rows, (H + 2 * Gr) * D), 4)
    both[:first] = float("nan")
    both[q_at[-1]:] = float("nan")
    cut = both.view(rows, H + 2 * Gr, D)
    q, k, v = cut[:, :H], cut[:, H:H + Gr], cut[:, H + Gr:]
    wide = torch.full((rows, H + 1, D), 77.0, dtype=torch.float16, device="cuda")
    packed(native, q, k, v, q_at, wide[:, :H])
    want, tol = packed_oracle(f64(q), f64(k), f64(v), q_at, q_at, D ** -0.5, U[torch.float16])
    got = f64(wide)
    check_close(got[first:q_at[-1], :H], want[first:q_at[-1]], tol[first:q_at[-1]], "strided")
    assert (got[:first] == 77).all() and (got[q_at[-1]:] == 77).all() and (got[:, H] == 77).all()


@pytest.mark.parametrize("D", [64, 128, 160])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_query_does_not_see_has_no_part_in_its_result(native, bad, D):
    """Keys and values of later tokens and of the neighbours that are not finite: earlier queries do not notice."""
    lens = [100, 200, 50]
    q_at = offsets(lens)
    q, k, v = randn((350, 4, D), 5), randn((350, 2, D), 6), randn((350, 2, D), 7)
    v[100 + 130:300] = bad          # of the second sequence, from its token 130 on
    k[300:] = bad                   # the third one's
    v[300:] = bad
    out = torch.zeros_like(q)
    packed(native, q, k, v, q_at, out)
    want, tol = packed_oracle(f64(q)[:230], f64(k)[:230], f64(v)[:230], [0, 100, 230], [0, 100, 230], D ** -0.5, U[torch.float16])
    check_close(f64(out)[:230], want, tol, "rows in front")
    assert not torch.isfinite(out[230:]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,keys", [([3], [3000]), ([700], [700]), ([40, 1], [900, 6000])])
def test_single_values_that_are_not_finite(native, bad, lens, keys):
    """One value of one late key: in its column it reaches the queries that see the key, and nothing else. Row tiles over many keys are cut
    between CTAs, so parts are joined too."""
    H, Gr, D = 4, 2, 128
    q_at, kv_at = offsets(lens), offsets(keys)
    q, k, v = randn((q_at[-1], H, D), 15), randn((kv_at[-1], Gr, D), 16), randn((kv_at[-1], Gr, D), 17)
    for e in kv_at[1:]:
        v[e - 2, 1, 77] = bad
        v[e - 1, 0, 5] = -bad
    out = torch.zeros_like(q)
    packed(native, q, k, v, q_at, out, kv_at)
    want, tol = packed_oracle(f64(q), f64(k), f64(v), q_at, kv_at, D ** -0.5, U[torch.float16])
    check_close(f64(out), want, tol, "values")
    assert (~np.isfinite(want)).sum() > 0 and np.isfinite(want).mean() > 0.9


@pytest.mark.parametrize("D", [128, 256])
def test_packed_attention_of_large_scores(native, D):
    """Scores of hundreds, rising along the keys: the running maximum moves at every tile."""
    n, H = 700, 2
    q, k, v = randn((n, H, D), 8) * 4, randn((n, 1, D), 9), randn((n, 1, D), 10)
    k = (k * torch.linspace(0.1, 4, n, device="cuda")[:, None, None]).half()
    q = q.half()
    out = torch.zeros_like(q)
    packed(native, q, k, v, [0, n], out)
    want, tol = packed_oracle(f64(q), f64(k), f64(v), [0, n], [0, n], D ** -0.5, U[torch.float16])
    check_close(f64(out), want, tol, "large scores")


@pytest.mark.parametrize("q_at", [[0, 5, 3, 10], [0, 5, 11], [-1, 5, 10], [0, 2 ** 31 - 1, 10]])
@pytest.mark.parametrize("D", [128, 256])
def test_packed_offsets_outside_are_reported(native, q_at, D):
    q = randn((10, 2, D), 11)
    out, status = torch.full_like(q, 77.0), i32([0])
    packed(native, q, q, q, q_at, out, status=status)
    assert status.item() == 4
    # sequences with offsets in order are computed
    want, tol = packed_oracle(f64(q), f64(q), f64(q), [0, 5], [0, 5], D ** -0.5, U[torch.float16])
    if q_at[:2] == [0, 5]:
        check_close(f64(out)[:3], want[:3], tol[:3], "the first sequence")


# ------------------------------------------------------------------------------------------------ drafted tokens
def make_tree(seqs, drafts, H, Gr, D, bs, ctxs, counts, seed, parents=None, spare=1):
    """Pools whose slots that no sequence has filled hold NaN."""
    rng = np.random.default_rng(seed)
    need = [-(-(c + n) // bs) for c, n in zip(ctxs, counts)]
    mb = max(max(need), 1)
    pages = rng.permutation(sum(need) + spare)
    tables, at = np.zeros((seqs, mb), np.int32), 0
    for s in range(seqs):
        tables[s, :need[s]] = pages[at:at + need[s]]
        at += need[s]
    kp = np.full((sum(need) + spare, Gr, bs, D), np.nan, np.float16)
    vp = kp.copy()
    for s in range(seqs):
        for t in range(ctxs[s] + counts[s]):
            kp[tables[s, t // bs], :, t % bs] = rng.standard_normal((Gr, D)).astype(np.float16)
            vp[tables[s, t // bs], :, t % bs] = rng.standard_normal((Gr, D)).astype(np.float16)
    if parents is None:
        parents = np.array([[rng.integers(-1, i) if i else -1 for i in range(drafts)] for _ in range(seqs)], np.int32).reshape(seqs, drafts)
    q = rng.standard_normal((seqs, drafts, H, D)).astype(np.float16)
    return q, kp, vp, tables, np.asarray(ctxs, np.int32), np.asarray(counts, np.int32), np.asarray(parents, np.int32)


def tree_oracle(q, kp, vp, tables, ctxs, counts, parents, scale):
    seqs, drafts, H, D = q.shape
    Gr, bs = kp.shape[1], kp.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(seqs):
        n = int(ctxs[s] + counts[s])
        t = np.arange(n)
        k, v = (p[tables[s, t // bs], :, t % bs].astype(np.float64) for p in (kp, vp))
        seen = np.zeros((int(counts[s]), n), bool)
        seen[:, :ctxs[s]] = True
        for i in range(int(counts[s])):
            a = i
            while a >= 0:
                seen[i, ctxs[s] + a] = True
                a = parents[s, a]
        for h in range(H):
            g = h // (H // Gr)
            out[s, :counts[s], h], tol[s, :counts[s], h] = attend(q[s, :counts[s], h].astype(np.float64), k[:, g], v[:, g], seen, scale, U[torch.float16])
    return out, tol


def tree(native, q, kp, vp, tables, ctxs, counts, parents, scale=None, status=None, out=None):
    dev = [torch.tensor(x).cuda() for x in (q, kp, vp, tables, ctxs, counts, parents)]
    out = torch.full(q.shape, 77.0, dtype=torch.float16, device="cuda")
    ws = room(ops.tree_attention_workspace(native, dev[0], dev[1], dev[3]))
    ops.tree_attention(native, *dev, out, scale, workspace=ws, status=status, stream=stream())
    torch.cuda.synchronize()
    return f64(out)


TREES = [
    # drafts, heads, kv heads, head size, block size, contexts, counts
    (1, 4, 1, 128, 16, [0], [1]), (1, 32, 8, 128, 16, [1000], [1]), (8, 32, 8, 128, 16, [1000], [8]), (16, 8, 2, 128, 16, [0, 1, 100, 127, 128, 129], [16, 15, 1, 16, 0, 9]),
    (5, 4, 4, 64, 8, [3, 300], [5, 2]), (64, 4, 1, 128, 32, [200, 64, 500], [64, 63, 33]), (64, 8, 1, 64, 16, [70, 1], [64, 64]), (33, 7, 1, 128, 16, [260], [33]),
    (7, 6, 2, 72, 1, [40, 0], [7, 7]), (9, 4, 2, 256, 16, [70, 5], [9, 8]), (4, 2, 2, 512, 4, [30], [4]), (3, 12, 12, 96, 64, [130, 17], [3, 1]), (12, 28, 4, 128, 16, [2000], [12]),
    (6, 4, 1, 128, 128, [700, 120, 122, 123], [6, 6, 6, 6]), (6, 4, 1, 64, 256, [700, 120], [6, 6]), (2, 160, 1, 64, 16, [300], [2]), (40, 16, 2, 128, 16, [30, 3000], [40, 1]),
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "%d-%d-%d-%d-%d-%d" % (c[0], c[1], c[2], c[3], c[4], sum(c[5])))
def test_tree_attention(native, case):
    d, H, Gr, D, bs, ctxs, counts = case
    t = make_tree(len(ctxs), d, H, Gr, D, bs, ctxs, counts, seed=d)
    status = i32([0])
    got = tree(native, *t, status=status)
    want, tol = tree_oracle(*t, D ** -0.5)
    check_close(got, want, tol, "tree")      # rows from counts on are zero
    assert status.item() == 0


def test_tree_attention_long_context_few_rows(native):
    """One sequence's chain over a long context: the keys are shared out over the whole GPU and joined."""
    t = make_tree(1, 4, 2, 1, 128, 16, [20000], [4], 3, parents=[[-1, 0, 1, 2]])
    want, tol = tree_oracle(*t, 128 ** -0.5)
    check_close(tree(native, *t), want, tol, "long")


def test_tree_attention_many_sequences(native):
    rng = np.random.default_rng(0)
    ctxs, counts = rng.integers(0, 400, 70), rng.integers(0, 7, 70)
    t = make_tree(70, 6, 4, 2, 64, 16, list(ctxs), list(counts), 5)
    want, tol = tree_oracle(*t, 0.125)
    check_close(tree(native, *t, scale=0.125), want, tol, "many")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_draft_does_not_notice_other_branches(native, bad, D):
    """Two branches behind the context; what one of them left in the cache is not finite."""
    d, ctx, bs = 6, 50, 16
    parents = [[-1, -1, 0, 1, 2, 3]]
    t = list(make_tree(1, d, 4, 2, D, bs, [ctx], [d], 6, parents=parents))
    want, tol = tree_oracle(*t, D ** -0.5)
    for p in (t[1], t[2]):
        for i in (1, 3, 5):
            p[t[3][0, (ctx + i) // bs], :, (ctx + i) % bs] = bad
    got = tree(native, *t)
    check_close(got[:, ::2], want[:, ::2], tol[:, ::2], "the other branch")
    assert not np.isfinite(got[:, 1::2]).any()


@pytest.mark.parametrize("D,ctx", [(64, 10), (128, 5000), (128, 127), (256, 60)])
def test_a_draft_notices_its_own_branch(native, D, ctx):
    """A value that is not finite in the cache row of draft 1 reaches its column of the drafts below it; one of the context reaches all."""
    t = list(make_tree(2, 5, 4, 2, D, 16, [ctx, ctx // 2], [5, 4], 6, parents=[[-1, -1, 1, 0, 2]] * 2))
    for s, n in enumerate((ctx, ctx // 2)):
        at = n + 1
        t[2][t[3][s, at // 16], 1, at % 16, 3] = np.inf
        t[2][t[3][s, (n - 1) // 16], 0, (n - 1) % 16, 9] = np.nan
    want, tol = tree_oracle(*t, D ** -0.5)
    got = tree(native, *t)
    check_close(got, want, tol, "own branch")
    assert not np.isfinite(want).all() and np.isfinite(want).mean() > 0.9


@pytest.mark.parametrize("D", [128, 256])
def test_tree_numbers_outside_are_reported(native, D):
    good = make_tree(2, 4, 4, 2, D, 16, [40, 30], [4, 4], 7)
    want, tol = tree_oracle(*good, D ** -0.5)
    pages = good[1].shape[0]

    def changed(which, where, value):
        t = [x.copy() for x in good]
        t[which][where] = value
        status = i32([0])
        got = tree(native, *t, status=status)
        assert status.item() == 4, (which, value)
        check_close(got[1], want[1], tol[1], "the other sequence")
        return got

    for value in (pages, -1, 2 ** 31 - 1, -2 ** 31):
        changed(3, (0, 1), value)                 # block id
    for value in (-1, 45, 2 ** 31 - 1):
        assert (changed(4, 0, value)[0] == 0).all()      # context
    for value in (-1, 5, 2 ** 31 - 1):
        assert (changed(5, 0, value)[0] == 0).all()      # count
    for value in (1, 2, -2, 2 ** 31 - 1):
        changed(6, (0, 1), value)                 # parent


# ------------------------------------------------------------------------------------------------ accepted drafts
@pytest.mark.parametrize("layers,seqs,drafts,Gr,D,bs", [(1, 1, 1, 1, 8, 1), (2, 3, 8, 2, 64, 16), (3, 5, 64, 8, 128, 16), (2, 2, 13, 3, 72, 8), (1, 4, 20, 1, 512, 32), (4, 1, 64, 12, 256, 4)])
def test_cache_keep(native, layers, seqs, drafts, Gr, D, bs):
    rng = np.random.default_rng(drafts)
    ctx = rng.integers(0, 40, seqs).astype(np.int32)
    mb = -(-(int(ctx.max()) + drafts) // bs)
    tables = rng.permutation(seqs * mb).reshape(seqs, mb).astype(np.int32)
    counts = rng.integers(0, drafts + 1, seqs).astype(np.int32)
    counts[0] = drafts if seqs == 1 else counts[0]
    path = np.full((seqs, drafts), -9, np.int32)
    for s in range(seqs):
        path[s, :counts[s]] = np.sort(rng.permutation(drafts)[:counts[s]])
    pools = randn((layers, 2, seqs * mb, Gr, bs, D), 12)
    want = pools.cpu().numpy().copy()
    for s in range(seqs):
        src = [(tables[s, (ctx[s] + p) // bs], (ctx[s] + p) % bs) for p in path[s, :counts[s]]]
        rows = [want[:, :, a, :, b].copy() for a, b in src]
        for j, r in enumerate(rows):
            to = ctx[s] + j
            want[:, :, tables[s, to // bs], :, to % bs] = r
    status = i32([0])
    ops.cache_keep(native, pools[:, 0], pools[:, 1], i32(tables), i32(ctx), i32(path), i32(counts), status=status, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(pools.cpu().numpy(), want) and status.item() == 0


@pytest.mark.parametrize("path,counts,ctx,table", [
    ([0, 2, 2, 3], 4, 5, None), ([3, 2, 5, 6], 4, 5, None), ([0, 1, 2, 8], 4, 5, None), ([-1, 1, 2, 3], 4, 5, None), ([1, 2, 3, 4], 5, 5, None), ([1, 2, 3, 4], -1, 5, None),
    ([1, 2, 3, 4], 4, 30, None), ([1, 2, 3, 4], 4, -1, None), ([1, 2, 3, 4], 4, 2 ** 31 - 1, None), ([1, 2, 3, 4], 4, 5, 4), ([1, 2, 3, 4], 4, 5, -1)])
def test_cache_keep_leaves_a_sequence_with_bad_numbers(native, path, counts, ctx, table):
    tables = np.array([[0, 1], [2, 3]], np.int32)
    if table is not None:
        tables[0, 0] = table
    pools = randn((2, 2, 4, 2, 16, 64), 13)
    before = pools.clone()
    status = i32([0])
    ops.cache_keep(native, pools[:, 0], pools[:, 1], i32(tables), i32([ctx, 3]), i32([path, [1, 3, 0, 0]]), i32([counts, 2]), status=status, stream=stream())
    torch.cuda.synchronize()
    assert status.item() == 4
    want = before.clone()
    want[:, :, 2, :, 3] = before[:, :, 2, :, 4]
    want[:, :, 2, :, 4] = before[:, :, 2, :, 6]
    assert torch.equal(pools, want)


# ------------------------------------------------------------------------------------------------ scores of tokens
def logprobs(native, logits, tokens, top, status=None):
    rows = logits.shape[0]
    o = [torch.full((rows,), 55.0, device="cuda"), torch.full((rows,), 55.0, device="cuda"), torch.full((rows, top), 55, dtype=torch.int32, device="cuda"),
         torch.full((rows, top), 55.0, device="cuda")]
    ws = room(ops.token_logprobs_workspace(native, logits, top))
    ops.token_logprobs(native, logits, tokens, *o, workspace=ws, status=status, stream=stream())
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in o]


def logprobs_oracle(x, tokens, top):
    rows, vocab = x.shape
    lp, ent = np.zeros(rows), np.zeros(rows)
    ids, tlp = np.full((rows, top), -1), np.full((rows, top), -np.inf)
    for r in range(rows):
        live = x[r] > -np.inf
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            ent[r], tlp[r] = np.nan, np.nan
            lp[r] = np.nan if tokens[r] >= 0 else 0
            continue
        if not live.any():
            lp[r] = -np.inf if tokens[r] >= 0 else 0
            continue
        d = x[r] - x[r][live].max()      # not the logits minus a log-sum: next to -3e38 a sum's logarithm is lost in 64 bits too
        log_s = np.log(np.exp(d[live]).sum())
        lp[r] = d[tokens[r]] - log_s if tokens[r] >= 0 else 0
        ent[r] = -(np.exp(d[live] - log_s) * (d[live] - log_s)).sum()
        order = np.argsort(-x[r], kind="stable")[:min(top, int(live.sum()))]
        ids[r, :len(order)], tlp[r, :len(order)] = order, d[order] - log_s
    return lp, ent, ids, tlp


def check_logprobs(got, want, x):
    """f32: a term's exponent is off by |x - m| 2^-24 in each of two roundings, exp2 by 2^-22, and a thread adds up to 2^10 terms before trees join
    the sums: 2^-14 of a sum at the very most, were every rounding to one side; the results are sums and differences of such and of logits."""
    biggest = np.abs(np.where(np.isfinite(x), x, 0)).max() if x.size else 0
    tol = 2.0 ** -14 + 3 * 2.0 ** -23 * (biggest + 1)
    for name, g, w in zip(("logprob", "entropy", "ids", "top"), got, want):
        if name == "ids":
            assert np.array_equal(g, w), name
            continue
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isinf(g), np.isinf(w)), name
        fine = np.isfinite(w)
        assert not fine.any() or np.abs(g[fine] - w[fine]).max() <= tol, (name, np.abs(g[fine] - w[fine]).max(), tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 5), (2, 31, 31), (5, 127, 20), (1, 129, 32), (4, 1000, 0), (7, 4097, 1), (2, 32001, 20), (1, 128256, 20), (40, 5003, 8), (2, 300007, 32), (1, 1300001, 32)])
def test_token_logprobs(native, dtype, rows, vocab, top):
    """Odd vocabularies put the rows of 16-bit logits off 16 bytes; bf16 has many equal logits."""
    x = randn((rows, vocab), rows + vocab, torch.float32)
    x = (x * 4).to(dtype)
    rng = np.random.default_rng(vocab)
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    if rows > 2:
        tokens[1] = -1
    got = logprobs(native, x, i32(tokens), top)
    check_logprobs(got, logprobs_oracle(f64(x), tokens, top), f64(x))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_token_logprobs_of_odd_rows(native, dtype):
    n, top = 3000, 6
    x = randn((12, n), 3, torch.float32).to(dtype)
    ninf, inf, nan = -float("inf"), float("inf"), float("nan")
    x[0] = ninf                                   # nothing is left
    x[1] = ninf
    x[1, 17] = 2.0                                # one token
    x[2, 100:] = ninf
    x[2, :97] = ninf                              # three
    x[3, 2999] = nan
    x[4, 5] = inf
    x[5] = 1.25                                   # all equal: the lowest ids
    x[6] = torch.arange(n, device="cuda") * 0.001      # rising (with ties in f16)
    x[7] = -torch.arange(n, device="cuda") * 0.001
    x[8] = torch.finfo(dtype).min                 # masks by the lowest value
    x[8, 1234] = 0.0
    x[9] = torch.finfo(dtype).min
    x[10] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.0, -0.0)     # two zeros, one value
    x[11, 64:128] = 30.0                          # ties across what a warp reads at once
    tokens = np.array([4, 17, 3, 1, 1, 7, 2999, 0, 1234, 3, 9, 64], np.int32)
    got = logprobs(native, x, i32(tokens), top)
    xs = f64(x)
    check_logprobs(got, logprobs_oracle(xs, tokens, top), np.where(np.abs(xs) > 1e4, 0, xs))


def test_token_logprobs_many_rows_strided_and_bad_tokens(native):
    rows, n = 70001, 9
    wide = randn((rows, n + 4), 4, torch.float32)
    x = wide[:, 3:3 + n]                          # rows 52 bytes apart, off 16 bytes
    tokens = np.random.default_rng(1).integers(0, n, rows).astype(np.int32)
    status = i32([0])
    got = logprobs(native, x, i32(tokens), 2, status)
    check_logprobs(got, logprobs_oracle(f64(x), tokens, 2), f64(x))
    assert status.item() == 0
    for bad in (n, -2, 2 ** 31 - 1):
        tokens[3] = bad
        status = i32([0])
        again = logprobs(native, x, i32(tokens), 2, status)
        assert status.item() == 4 and np.isnan(again[0][3])
        assert np.array_equal(np.delete(again[0], 3), np.delete(got[0], 3)) and all(np.array_equal(a, b) for a, b in zip(again[1:], got[1:]))


def test_token_logprobs_parts_may_be_left_out(native):
    x = randn((4, 500), 6, torch.float32)
    full = logprobs(native, x, i32([1, 2, 3, 4]), 3)
    ws, lp, ent = room(ops.token_logprobs_workspace(native, x, 0)), torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    ops.token_logprobs(native, x, i32([1, 2, 3, 4]), lp, workspace=ws, stream=stream())
    ops.token_logprobs(native, x, None, None, ent, workspace=ws, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(lp.cpu().numpy(), full[0]) and np.array_equal(ent.cpu().numpy(), full[1])


# ------------------------------------------------------------------------------------------------ streams, graphs, the library's own memory
def test_calls_are_captured_and_replayed(native):
    """Two graphs with a workspace each, replayed on inputs that changed, the second on a stream of its own; a call between them."""
    H, Gr, D, n = 4, 2, 128, 300

    def made(s):
        q, k, v = randn((n, H, D), 20 + s), randn((n, Gr, D), 30 + s), randn((n, Gr, D), 40 + s)
        t = [torch.tensor(x).cuda() for x in make_tree(2, 5, H, Gr, D, 16, [300, 40], [5, 3], 50 + s)]
        at, out, tout = i32([0, 100, n]), torch.zeros_like(q), torch.zeros((2, 5, H, D), dtype=torch.float16, device="cuda")
        x, tok, lp = randn((3, 5000), 60 + s, torch.float32), i32([1, 2, 3]), torch.zeros(3, device="cuda")
        ids, tlp = torch.zeros((3, 4), dtype=torch.int32, device="cuda"), torch.zeros((3, 4), device="cuda")
        w = [room(b) for b in (ops.packed_attention_workspace(native, q, k, 2), ops.tree_attention_workspace(native, t[0], t[1], t[3]), ops.token_logprobs_workspace(native, x, 4))]

        def go():
            ops.packed_attention(native, q, k, v, at, out, workspace=w[0], stream=torch.cuda.current_stream())
            ops.tree_attention(native, *t, tout, workspace=w[1], stream=torch.cuda.current_stream())
            ops.token_logprobs(native, x, tok, lp, None, ids, tlp, workspace=w[2], stream=torch.cuda.current_stream())

        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            go()
        return g, go, (q, t[0], x), (out, tout, lp, ids, tlp)

    graphs = [made(s) for s in range(2)]
    for g, go, ins, outs in graphs:
        for a in ins:
            a.copy_(torch.flip(a, [0]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    got = [[o.clone() for o in outs] for _, _, _, outs in graphs]
    for i, (g, go, ins, outs) in enumerate(graphs):
        for o in outs:
            o.zero_()
        go()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[i], outs)) and all(o.abs().sum() > 0 for o in outs)


def test_library_stream_and_memory(native):
    """Pools of a state block, the library's own stream, the same answer."""
    t = make_tree(2, 4, 4, 2, 128, 16, [100, 37], [4, 2], 8)
    want = tree(native, *t)
    model = Native.load([])
    model.alloc_states([t[1].nbytes, t[2].nbytes])
    pools = []
    for off, p in zip(model.state_offsets, (t[1], t[2])):
        model.state.write(off, p)
        pools.append(ops.DeviceArray(model.state.device_ptr + off, p.shape, "<f2", owner=model.state))
    q, tables, ctx, cnt, par = (torch.tensor(t[i]).cuda() for i in (0, 3, 4, 5, 6))
    out = torch.zeros(t[0].shape, dtype=torch.float16, device="cuda")
    ws = room(ops.tree_attention_workspace(model, q, pools[0], tables))
    torch.cuda.synchronize()
    ops.tree_attention(model, q, *pools, tables, ctx, cnt, par, out, workspace=ws)
    model.sync()
    assert np.array_equal(f64(out), want)
    model.close()


def test_results_do_not_change_from_run_to_run(native):
    q, k = randn((600, 8, 128), 1), randn((600, 2, 128), 2)
    t = make_tree(3, 8, 8, 2, 128, 16, [900, 10, 400], [8, 8, 5], 3)
    x = randn((5, 40000), 9, torch.float32)
    first = None
    for _ in range(5):
        out = torch.zeros_like(q)
        packed(native, q, k, k, [0, 50, 600], out)
        now = [f64(out), tree(native, *t)] + logprobs(native, x, i32([0] * 5), 10)
        first = first or now
        assert all(np.array_equal(a, b) for a, b in zip(first, now))


# ------------------------------------------------------------------------------------------------ nodes
def run_graph(g, out, inputs, states=()):
    native = Native.load([])
    native.alloc_states([s.nbytes for s in states])
    for off, s in zip(native.state_offsets, states):
        native.state.write(off, s)
    prog = NativeProgram.compile(native, g)
    for i, x in enumerate(inputs):
        prog.set_input(i, x)
    prog.run()
    prog.run()          # the captured sequence
    y = prog.read(out).copy()
    prog.free()
    native.close()
    return y


def test_packed_attention_node(native):
    H, Gr, D, q_at, kv_at = 4, 2, 128, [0, 30, 30, 170], [0, 400, 401, 600]
    q, k, v = randn((170, H, D), 1), randn((600, Gr, D), 2), randn((600, Gr, D), 3)
    out = torch.zeros_like(q)
    packed(native, q, k, v, q_at, out, kv_at, scale=0.1)
    g = G.Graph()
    tq, tk, tv = g.input(G.F16, [D, H, 170], "q"), g.input(G.F16, [D, Gr, 600], "k"), g.input(G.F16, [D, Gr, 600], "v")
    y = g.output(g.cast(g.packed_attention(tq, tk, tv, g.input(G.I32, [4], "qo"), 0.1, g.input(G.I32, [4], "ko")), G.F32))
    got = run_graph(g, y, [x.cpu().numpy() for x in (q, k, v)] + [np.array(a, np.int32) for a in (q_at, kv_at)])
    assert np.array_equal(got.reshape(170, H, D), out.float().cpu().numpy())


def test_tree_attention_and_logprobs_nodes(native):
    t = make_tree(3, 6, 4, 2, 64, 16, [100, 0, 333], [6, 1, 4], 9)
    want = tree(native, *t)
    g = G.Graph()
    kc, vc = g.state(G.F16, [t[1].size], "k"), g.state(G.F16, [t[2].size], "v")
    tq = g.input(G.F16, [64, 4, 6, 3], "q")
    tt, tc, tn, tp = g.input(G.I32, [t[3].shape[1], 3], "tables"), g.input(G.I32, [3], "context"), g.input(G.I32, [3], "counts"), g.input(G.I32, [6, 3], "parents")
    y = g.output(g.cast(g.paged_tree_attention(tq, kc, vc, tt, tc, tn, tp, 16, 0.125, 2), G.F32))
    got = run_graph(g, y, [t[0], t[3], t[4], t[5], t[6]], [t[1], t[2]])
    assert np.array_equal(got.reshape(want.shape), want)
    x = randn((5, 3001), 3, torch.float32)
    tok = np.array([5, -1, 3000, 0, 7], np.int32)
    lp, ent, ids, tlp = logprobs(native, x, i32(tok), 4)
    g = G.Graph()
    y = g.output(g.token_logprobs(g.input(G.F32, [3001, 5], "x"), g.input(G.I32, [5], "tok"), 4))
    got = run_graph(g, y, [x.cpu().numpy(), tok])
    assert np.array_equal(got, np.concatenate([lp[:, None], ent[:, None], ids.astype(np.float32), tlp], 1))


def test_nodes_report_numbers_outside(native):
    t = make_tree(1, 4, 4, 2, 128, 16, [40], [4], 7)
    g = G.Graph()
    kc, vc = g.state(G.F16, [t[1].size], "k"), g.state(G.F16, [t[2].size], "v")
    tq = g.input(G.F16, [128, 4, 4, 1], "q")
    ins = [g.input(G.I32, [t[3].shape[1], 1], "tables"), g.input(G.I32, [1], "context"), g.input(G.I32, [1], "counts"), g.input(G.I32, [4, 1], "parents")]
    g.output(g.paged_tree_attention(tq, kc, vc, *ins, 16, 0.1, 2))
    t[3][0, 1] = 99
    with pytest.raises(TlbError) as e:
        run_graph(g, 0, [t[0], t[3], t[4], t[5], t[6]], [t[1], t[2]])
    assert e.value.kind == "Execution" and "out of range" in str(e.value)


def test_nodes_refuse_what_they_do_not_take():
    n = Native.load([])

    def refused(build, word):
        g = G.Graph()
        g.output(build(g))
        with pytest.raises(TlbError) as e:
            NativeProgram.compile(n, g)
        assert e.value.kind == "Unsupported" and word in str(e.value), str(e.value)

    at = lambda g: g.input(G.I32, [3], "at")  # noqa: E731
    rows = lambda g, ty, h, d=64, r=10: g.input(ty, [d, h, r], "x")  # noqa: E731
    refused(lambda g: g.packed_attention(rows(g, G.F32, 4), rows(g, G.F32, 2), rows(g, G.F32, 2), at(g), 0.1), "f16 or all bf16")
    refused(lambda g: g.packed_attention(rows(g, G.F16, 4), rows(g, G.BF16, 2), rows(g, G.BF16, 2), at(g), 0.1), "f16 or all bf16")
    refused(lambda g: g.packed_attention(rows(g, G.F16, 4, 12), rows(g, G.F16, 2, 12), rows(g, G.F16, 2, 12), at(g), 0.1), "multiple of")
    refused(lambda g: g.packed_attention(rows(g, G.F16, 4, 520), rows(g, G.F16, 2, 520), rows(g, G.F16, 2, 520), at(g), 0.1), "head size")
    refused(lambda g: g.packed_attention(rows(g, G.F16, 4), rows(g, G.F16, 2, 64, 9), rows(g, G.F16, 2, 64, 9), at(g), 0.1), "offsets of their own")
    refused(lambda g: g.token_logprobs(g.input(G.F32, [100, 2], "x"), None, 33), "32")
    refused(lambda g: g.token_logprobs(g.input(G.I32, [100, 2], "x"), None, 3), "f32, f16 or bf16")
    n.close()


def test_nodes_refuse_views_between_two_values():
    n = Native.load([])

    def refused(build, word):
        g = G.Graph()
        g.output(build(g))
        with pytest.raises(TlbError) as e:
            NativeProgram.compile(n, g)
        assert e.value.kind == "Unsupported" and word in str(e.value), str(e.value)

    numbers = lambda g, off: g.view(g.input(G.I32, [16], "at"), [3], offset=off)  # noqa: E731
    rows = lambda g, h, off=0: g.view(g.input(G.F16, [64 * h * 11], "x"), [64, h, 10], 128, 128 * h, offset=off)  # noqa: E731
    refused(lambda g: g.packed_attention(rows(g, 4, 2), rows(g, 2), rows(g, 2), numbers(g, 0), 0.1), "")
    refused(lambda g: g.packed_attention(rows(g, 4), rows(g, 2), rows(g, 2, 8), numbers(g, 0), 0.1), "")
    refused(lambda g: g.packed_attention(rows(g, 4), rows(g, 2), rows(g, 2), numbers(g, 2), 0.1), "4-byte")
    refused(lambda g: g.packed_attention(rows(g, 4), rows(g, 2), rows(g, 2), numbers(g, 0), 0.1, numbers(g, 6)), "4-byte")
    refused(lambda g: g.token_logprobs(g.view(g.input(G.F32, [202], "x"), [100, 2], 400, offset=2), None, 3), "aligned")
    refused(lambda g: g.token_logprobs(g.input(G.F32, [100, 3], "x"), numbers(g, 3), 3), "aligned")
    n.close()


# ------------------------------------------------------------------------------------------------ far away
@pytest.mark.parametrize("D", [64, 128, 256])
def test_packed_attention_behind_four_gigabytes(native, D):
    H, Gr, rows = 4, 2, 1_200_000
    q_at, kv_at = offsets([30, 70]), offsets([100, 200], rows - 300)
    wide_q, wide_o = (torch.empty((100, 1 << 25), dtype=torch.float16, device="cuda") for _ in range(2))     # rows 64 MB apart
    q, out = (x[:, :H * D].view(100, H, D) for x in (wide_q, wide_o))
    both = torch.empty((rows, 2, 1024), dtype=torch.float16, device="cuda")                                    # 4 KB apart
    k, v = both[:, 0, :Gr * D].unflatten(1, (Gr, D)), both[:, 1, :Gr * D].unflatten(1, (Gr, D))
    q.copy_(randn((100, H, D), 41))
    k[-300:], v[-300:] = randn((300, Gr, D), 42), randn((300, Gr, D), 43)
    packed(native, q, k, v, q_at, out, kv_at)
    near = [c - (rows - 300) for c in kv_at]
    want, tol = packed_oracle(f64(q), f64(k[-300:]), f64(v[-300:]), q_at, near, D ** -0.5, U[torch.float16])
    check_close(f64(out), want, tol, "far rows")


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32), (128, 4)])
def test_pages_behind_four_gigabytes(native, D, bs):
    drafts, H, Gr, pages = 6, 4, 2, (5 << 30) // (2 * bs * D * 2)
    t = list(make_tree(2, drafts, H, Gr, D, bs, [130, 5], [6, 4], seed=44))
    want, tol = tree_oracle(*t, D ** -0.5)
    n = t[1].shape[0]
    pools = torch.empty((2, pages, Gr, bs, D), dtype=torch.float16, device="cuda")
    for i in range(2):
        pools[i, -n:] = torch.tensor(t[1 + i]).cuda()
    tables = i32(t[3] + (pages - n))
    q, ctx, counts, parents = torch.tensor(t[0]).cuda(), i32(t[4]), i32(t[5]), i32(t[6])
    out, status = torch.full(t[0].shape, 77.0, dtype=torch.float16, device="cuda"), i32([0])
    ws = room(ops.tree_attention_workspace(native, q, pools[0], tables))
    ops.tree_attention(native, q, pools[0], pools[1], tables, ctx, counts, parents, out, workspace=ws, status=status, stream=stream())
    before = pools[:, -n:].clone()
    path = i32([[0, 2, 5, 0, 0, 0], [1, 3, 0, 0, 0, 0]])
    ops.cache_keep(native, pools[None, 0], pools[None, 1], tables, ctx, path, i32([3, 2]), status=status, stream=stream())
    torch.cuda.synchronize()
    check_close(f64(out), want, tol, "far pages")
    for s, keep in enumerate(([0, 2, 5], [1, 3])):
        src = [before[:, t[3][s, (t[4][s] + p) // bs], :, (t[4][s] + p) % bs].clone() for p in keep]
        for j, r in enumerate(src):
            to = t[4][s] + j
            before[:, t[3][s, to // bs], :, to % bs] = r
    assert torch.equal(pools[:, -n:].view(torch.int16), before.view(torch.int16)) and status.item() == 0


def test_logits_behind_four_gigabytes(native):
    wide = torch.empty((130, 1 << 24), device="cuda")      # 64 MB apart
    x = wide[:, 5:1005]
    x.copy_(randn((130, 1000), 45, torch.float32))
    tok = np.arange(130, dtype=np.int32) * 7
    check_logprobs(logprobs(native, x, i32(tok), 3), logprobs_oracle(f64(x), tok, 3), f64(x))


def test_two_streams_at_once(native):
    """Calls of two streams with a workspace each, long and short ones by turns, give what they give alone."""
    H, Gr, D = 8, 2, 64
    a, b = [300, 5, 700], [1, 2, 150]
    q, k, v = randn((1005, H, D), 51), randn((1005, Gr, D), 52), randn((1005, Gr, D), 53)
    t = [torch.tensor(x).cuda() for x in make_tree(5, 16, H, Gr, 128, 16, [2000, 3, 900, 0, 64], [16, 1, 9, 16, 0], seed=54)]
    alone = [torch.full_like(q, 77.0), torch.full_like(q, 77.0), torch.full_like(t[0], 77.0)]
    packed(native, q, k, v, offsets(a), alone[0])
    packed(native, q, k, v, offsets(b), alone[1])
    ws = [room(ops.packed_attention_workspace(native, q, k, 3)), room(ops.tree_attention_workspace(native, t[0], t[1], t[3]))]
    ops.tree_attention(native, *t, alone[2], workspace=ws[1], stream=stream())
    at = [i32(offsets(a)), i32(offsets(b))]
    together = [[torch.full_like(x, 55.0) for x in alone] for _ in range(20)]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for o in together:
        ops.packed_attention(native, q, k, v, at[0], o[0], workspace=ws[0], stream=one)
        ops.tree_attention(native, *t, o[2], workspace=ws[1], stream=two)
        ops.packed_attention(native, q, k, v, at[1], o[1], workspace=ws[0], stream=one)
    torch.cuda.synchronize()
    for o in together:
        assert torch.equal(o[0], alone[0]) and torch.equal(o[2], alone[2])
        assert torch.equal(o[1][:153], alone[1][:153]) and (o[1][153:] == 55).all()
