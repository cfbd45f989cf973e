"""The serving operators together, as a server uses them: prompts of different lengths in one packed pass, drafted tokens verified as a tree, the
accepted ones moved into place, tokens scored. Against the padded prompt pass and the one-token decode loop of the same decoder.

f16 weights: no 8-bit activations, so two attention kernels that round differently leave logits that differ by roundings only. A layer's f16
roundings (queries, keys, values, P, result: 2^-11 each, of values of like size) reach the residual stream scaled by the projections; two layers of five
such roundings on either side stay below 20 x 2^-11 = 1e-2 of the largest logit. Embeddings and output are tied and large beside the layers, so that
the best token has a margin far above that."""
import numpy as np
import pytest

from tensorlisp_b200 import device_ops as ops
from tensorlisp_b200 import graph as G
from tensorlisp_b200.native import Native, NativeProgram
from tensorlisp_b200.programs import (DecodeLoop, DecoderConfig, TreeDecodeLoop, decoder_weights, packed_prefill_step, prefill_step)

pytestmark = pytest.mark.gpu
TOL = 1e-2


def config(**kw):
    return DecoderConfig(**{**dict(n_layers=2, d_model=512, n_heads=8, n_kv_heads=2, head_dim=64, d_ffn=1024, vocab=777, wtype=G.F16, etype=G.F16), **kw})


def weights(cfg, seed=0):
    rng = np.random.default_rng(seed)
    embedding = (rng.standard_normal((cfg.vocab, cfg.d_model)) * 3).astype(np.float16)
    out = []
    for s in decoder_weights(cfg):
        if len(s.ne) == 1:
            out.append((1 + 0.1 * rng.standard_normal(s.ne[0])).astype(np.float32))
        elif s.name in ("token_embd", "output"):
            out.append(embedding if s.name == "token_embd" else np.roll(embedding, 1, 0))     # token t is mostly followed by t + 1: a decoder with something to say
        else:
            out.append((rng.standard_normal((s.ne[1], s.ne[0])) * 0.02).astype(np.float16))
    return out


def prefill(native, cfg, prompts, tables, pool_blocks, extra=0):
    """The packed pass over `prompts`, with `extra` rows behind them; logits of the last tokens."""
    lens = [len(p) for p in prompts]
    T = sum(lens) + extra
    dg = packed_prefill_step(cfg, len(prompts), T, pool_blocks)
    if not native.state_offsets:
        native.alloc_states(dg.state_bytes)
    prog = NativeProgram.compile(native, dg.graph)
    ids, pos, slots = np.zeros(T, np.int32), np.zeros(T, np.int32), np.full(T, -1, np.int64)
    at = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    for b, p in enumerate(prompts):
        t = np.arange(lens[b])
        ids[at[b]:at[b + 1]], pos[at[b]:at[b + 1]] = p, t
        slots[at[b]:at[b + 1]] = tables[b, t // cfg.block_size].astype(np.int64) * cfg.block_size + t % cfg.block_size
    for name, a in dict(ids=ids, pos=pos, offsets=at, last=at[1:] - 1, slots=slots.view(np.int32)).items():
        prog.set_input(dg.inputs[name], a)
    prog.run()
    logits = prog.read(dg.logits).reshape(len(prompts), -1).copy()
    prog.free()
    return logits


def near(got, want):
    assert np.abs(got - want).max() <= TOL * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (4, 4, 128), (2, 1, 256)])
def test_packed_prompts_equal_padded_ones(heads, kvh, hd):
    """Each prompt of the packed pass against the padded pass of that prompt alone, logits and cached keys and values."""
    cfg = config(n_heads=heads, n_kv_heads=kvh, head_dim=hd)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab, n) for n in (130, 1, 47, 200)]
    mb = 13
    tables = rng.permutation(len(prompts) * mb).astype(np.int32).reshape(len(prompts), mb)
    w = weights(cfg)
    native = Native.load(w)
    got = prefill(native, cfg, prompts, tables, len(prompts) * mb, extra=5)
    pool = len(prompts) * mb * kvh * cfg.block_size * hd * 2
    k, v = native.state.gather_kv(native.state_offsets[2], native.state_offsets[3], len(prompts) * mb, kvh, hd, cfg.block_size, tables, [len(p) for p in prompts])
    native.close()
    at = 0
    for b, p in enumerate(prompts):
        n = len(p)
        dg = prefill_step(cfg, 1, n)
        one = Native.load(w)
        one.alloc_states(dg.state_bytes)
        prog = NativeProgram.compile(one, dg.graph)
        slots = np.arange(n, dtype=np.int64)
        mask = np.triu(np.full((n, n), -np.inf, np.float16), 1)
        for name, a in dict(ids=p.astype(np.int32), pos=np.arange(n, dtype=np.int32), mask=mask, last=np.array([n - 1], np.int32), slots=slots.view(np.int32)).items():
            prog.set_input(dg.inputs[name], a)
        prog.run()
        near(got[b], prog.read(dg.logits).reshape(-1))
        pages = -(-n // cfg.block_size)
        k1, v1 = one.state.gather_kv(one.state_offsets[2], one.state_offsets[3], pages, kvh, hd, cfg.block_size, np.arange(pages, dtype=np.int32)[None], [n])
        near(k[at:at + n].astype(np.float64), k1.astype(np.float64))
        near(v[at:at + n].astype(np.float64), v1.astype(np.float64))
        at += n
        prog.free()
        one.close()
    assert pool > 0


@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 4, 1), (256, 2, 2)])
def test_tree_decode_gives_the_tokens_of_the_plain_loop(hd, heads, kvh):
    """Prompts packed into the cache, then drafts of which some are right, some are not and some branch: the tokens of the one-token loop, in fewer
    steps, and its logits at the accepted rows."""
    cfg = config(n_heads=heads, n_kv_heads=kvh, head_dim=hd)
    rng = np.random.default_rng(2)
    B, D, max_ctx, mb = 3, 6, 96, 6
    prompts = [rng.integers(0, cfg.vocab, n) for n in (33, 1, 15)]
    tables = rng.permutation(B * mb).astype(np.int32).reshape(B, mb)
    w = weights(cfg, 3)
    native = Native.load(w)
    first = prefill(native, cfg, prompts, tables, B * mb).argmax(1)
    plain = DecodeLoop(native, cfg, B, max_ctx, tables)
    cached = np.array([len(p) for p in prompts], np.int32)
    plain.begin(first, cached)
    want, logits = [[] for _ in range(B)], [[] for _ in range(B)]
    for _ in range(24):
        plain.step()
        for b in range(B):
            want[b].append(int(plain.tokens()[b]))
            logits[b].append(plain.logits()[b].copy())
    plain.free()
    margin = min((np.sort(x)[-1] - np.sort(x)[-2]) / np.abs(x).max() for l in logits for x in l)
    assert margin > 2 * TOL, margin       # the comparison of tokens below has a meaning

    native.reset_state()
    assert np.array_equal(prefill(native, cfg, prompts, tables, B * mb).argmax(1), first)
    tree = TreeDecodeLoop(native, cfg, B, D, max_ctx, tables, top=3)
    tree.begin(first, cached)
    got = [[] for _ in range(B)]
    while min(len(x) for x in got) < 16:
        drafted = []
        for b in range(B):
            truth, n = want[b][len(got[b]):], int(rng.integers(0, D))
            d, good = [], -1        # right tokens in a chain, wrong ones beside them
            for i in range(n):
                if rng.random() < 0.6 and sum(t[2] for t in d) < len(truth):
                    d.append((truth[sum(t[2] for t in d)], good, 1))
                    good = i
                else:
                    d.append((int(rng.integers(0, cfg.vocab)), int(rng.integers(-1, i)) if i else -1, 0))
            drafted.append([t[:2] for t in d])
        before = [len(x) for x in got]
        for b, new in enumerate(tree.step(drafted)):
            got[b] += new
            near(tree.logits()[b, 0], logits[b][before[b]])
            s = tree.scores()[b]
            x = tree.logits()[b, 0].astype(np.float64)
            d = x - x.max()
            assert s[0, 2] == want[b][before[b]] == np.argmax(x) and abs(s[0, 5] + np.log(np.exp(d).sum())) < 1e-4
            if drafted[b]:
                follow = next(t for t, parent in drafted[b] if parent == -1)
                assert abs(s[0, 0] - (d[follow] - np.log(np.exp(d).sum()))) < 1e-3
            else:
                assert s[0, 0] == 0
    for b in range(B):
        n = min(len(got[b]), len(want[b]))
        assert got[b][:n] == want[b][:n]
    assert tree.steps < max(len(x) for x in got)       # drafts were accepted
    tree.free()
    native.close()


def test_tree_decode_reports_a_page_outside():
    cfg = config(n_layers=1)
    native = Native.load(weights(cfg))
    tables = np.array([[0, 1]], np.int32)
    tree = TreeDecodeLoop(native, cfg, 1, 4, 32, tables)
    tree.begin(np.array([5]), np.array([0]))
    assert tree.step([[(6, -1)]])[0][0] >= 0
    tree.room.write(0, np.array([[0, 99]], np.int32))       # what cache_keep sees
    tree.context[:] = 16
    with pytest.raises(RuntimeError):
        tree.step([[]])
    tree.free()
    native.close()
