"""What is timed of the serving operators on device arrays: attention over packed prompts, attention for a tree of drafted
tokens over the paged cache, moving the accepted drafts into place in the cache, and log probabilities with entropy and
top alternatives.

``run`` computes each in its plain form (elementary torch operations in 32 bits, rounded once) or, where ``own`` is set, with
the calls of ``tensorlisp_b200.device_ops``. Prompts and contexts of a batch are spread evenly over their range and come in an
order that the seed gives, so that a case's work is its own; cache pages lie in a random order.
"""
import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16      # tokens of a cache page


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    llama = dict(heads=32, kv_heads=8, hs=128)
    return [
        # one user's short chat turn: latency
        dict(name="packed_1x37", kind="packed", type="f16", seqs=1, low=37, high=37, behind=0, fused=False, **llama),
        # prompts of a batch that are admitted together, none padded; keys and values are columns of one projection's result
        dict(name="packed_bf16_24x1000", kind="packed", type="bf16", seqs=24, low=3, high=1000, behind=0, fused=True, heads=16, kv_heads=4, hs=64),
        # chunks of new tokens behind what the cache holds of their conversations
        dict(name="packed_chunk_8x200", kind="packed", type="f16", seqs=8, low=33, high=201, behind=4000, fused=False, **llama),
        # one long document
        dict(name="packed_1x8192", kind="packed", type="f16", seqs=1, low=8192, high=8192, behind=0, fused=False, **llama),
        # one user's chat with a short chain of drafts
        dict(name="tree_1x8_1000", kind="tree", seqs=1, drafts=8, chain=True, low=1000, high=1000, **llama),
        # a serving batch with small trees at the context of the decode benchmark
        dict(name="tree_32x16_2048", kind="tree", seqs=32, drafts=16, chain=False, low=2048, high=2048, **llama),
        # larger trees over very different contexts
        dict(name="tree_48x32_8192", kind="tree", seqs=48, drafts=32, chain=False, low=128, high=8192, **llama),
        # the accepted drafts of one user, all layers of the decoder
        dict(name="keep_1x8", kind="keep", layers=32, seqs=1, drafts=8, ctx=200, kv_heads=8, hs=128),
        # and of a serving batch
        dict(name="keep_32x16", kind="keep", layers=32, seqs=32, drafts=16, ctx=100, kv_heads=8, hs=128),
        # one sampled token with the alternatives that an API returns
        dict(name="logprobs_1x128256", kind="logprobs", type="f32", rows=1, vocab=128256, top=20, banned=0.0),
        # a batch of drafts that is verified: 32 sequences with 16 drafts each
        dict(name="logprobs_512x128256", kind="logprobs", type="f32", rows=512, vocab=128256, top=5, banned=0.0),
        # scoring a prompt under a grammar that bans a part of the vocabulary, logits in half precision
        dict(name="logprobs_bf16_333x32000", kind="logprobs", type="bf16", rows=333, vocab=32000, top=8, banned=0.3),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform in the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [dict(heads=32, kv_heads=8, hs=128), dict(heads=16, kv_heads=4, hs=64), dict(heads=8, kv_heads=8, hs=128), dict(heads=16, kv_heads=2, hs=128),
         dict(heads=28, kv_heads=4, hs=128), dict(heads=12, kv_heads=12, hs=64)]


def draw(rng):
    kind = rng.choice(["packed", "packed", "tree", "tree", "keep", "logprobs", "logprobs"])
    if kind == "packed":
        high = _log(rng, 1, 4000)
        # padded, the plain form's scores stay below those of the longest listed prompt
        seqs = _log(rng, 1, max(1, min(32, 60_000_000 // (high * (high + 4000)))))
        return dict(kind=kind, type=rng.choice(["f16", "bf16"]), seqs=seqs, low=_log(rng, 1, high), high=high, behind=rng.choice([0, 0, _log(rng, 1, 4000)]),
                    fused=rng.random() < 0.5, **rng.choice(HEADS))
    if kind == "tree":
        high = _log(rng, 17, 8192)
        return dict(kind=kind, seqs=_log(rng, 1, min(48, max(1, 160_000 // high))), drafts=_log(rng, 1, 32), chain=rng.random() < 0.3, low=_log(rng, 1, high), high=high,
                    **rng.choice(HEADS))
    if kind == "keep":
        h = rng.choice(HEADS)
        return dict(kind=kind, layers=_log(rng, 1, 32), seqs=_log(rng, 1, 32), drafts=_log(rng, 1, 16), ctx=_log(rng, 1, 100), kv_heads=h["kv_heads"], hs=h["hs"])
    vocab = _log(rng, 1000, 200000)
    return dict(kind=kind, type=rng.choice(["f32", "f32", "f16", "bf16"]), rows=_log(rng, 1, min(512, 60_000_000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                banned=rng.choice([0.0, 0.5]))


def _spread(case):
    """Lengths of the sequences: from the lowest to the highest in even steps."""
    n = case["seqs"]
    return [case["high"] if n == 1 else case["low"] + (case["high"] - case["low"]) * i // (n - 1) for i in range(n)]


def _cached(case):
    """How many keys lie in front of each prompt's own, before the order is shuffled."""
    n = case["seqs"]
    return [case["behind"] * (i + 1) // n for i in range(n)]


# ------------------------------------------------------------------------------------------------ prepare
@functools.lru_cache(maxsize=None)
def _device():
    """The framework's calls and its handle of the device, opened once by a process."""
    from tensorlisp_b200 import device_ops
    from tensorlisp_b200.native import Native
    return device_ops, Native(torch.cuda.current_device())


def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + salt)
    return g


def _order(seed, n):
    return torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _room(state, need):
    """What a program that serves keeps beside its buffers: the handle, and scratch memory of the size the framework asks for."""
    if own:
        state["ops"], state["native"] = _device()
        state["workspace"] = torch.empty(max(need(state["ops"], state["native"]), 16), dtype=torch.uint8, device="cuda")
    return state


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _prepare_packed(case, seed):
    order = _order(seed, case["seqs"])
    lens = [_spread(case)[i] for i in order]
    keys = [_spread(case)[i] + _cached(case)[i] for i in order]
    H, G, D, ty = case["heads"], case["kv_heads"], case["hs"], DTYPES[case["type"]]
    rows, kv_rows = sum(lens), sum(keys)
    gen = _generator(seed, 1)
    q = torch.randn((rows, H, D), generator=gen, device="cuda", dtype=ty)
    if case["fused"]:
        both = torch.randn((kv_rows, 2, G, D), generator=gen, device="cuda", dtype=ty)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.randn((kv_rows, G, D), generator=gen, device="cuda", dtype=ty) for _ in range(2))
    at = lambda n: _i32([sum(n[:i]) for i in range(len(n) + 1)])  # noqa: E731
    return _room(dict(kind="packed", q=q, k=k, v=v, q_offsets=at(lens), kv_offsets=at(keys) if case["behind"] else None, longest=max(lens),
                      most_keys=max(keys), scale=1.0 / math.sqrt(D), out=torch.empty_like(q)),
                 lambda ops, native: ops.packed_attention_workspace(native, q, k, case["seqs"]))


def _tables(lens, seed):
    """Pages of the sequences in a random order, [seqs, pages of the longest], and the number of pages."""
    need = [-(-n // BLOCK) for n in lens]
    pages = torch.randperm(sum(need), generator=_generator(seed, 2), device="cuda").to(torch.int32)
    tables = torch.zeros((len(lens), max(need)), dtype=torch.int32, device="cuda")
    owned = torch.arange(max(need), device="cuda") < torch.tensor(need, device="cuda")[:, None]
    tables[owned] = pages
    return tables, sum(need)


def _prepare_tree(case, seed):
    n, d, G, D = case["seqs"], case["drafts"], case["kv_heads"], case["hs"]
    lens = [_spread(case)[i] for i in _order(seed, n)]
    tables, pages = _tables([c + d for c in lens], seed)
    gen = _generator(seed, 3)
    q = torch.randn((n, d, case["heads"], D), generator=gen, device="cuda", dtype=torch.float16)
    pools = torch.randn((2, pages, G, BLOCK, D), generator=gen, device="cuda", dtype=torch.float16)
    # a token's parent is one of those before it (or the context); some sequences have drafted fewer tokens
    steps = torch.arange(d, device="cuda")
    parents = (steps - 1).expand(n, d) if case["chain"] else (torch.rand((n, d), generator=gen, device="cuda") * (steps + 1)).long() - 1
    counts = d - (torch.rand(n, generator=gen, device="cuda") * ((d + 3) // 4)).long()
    return _room(dict(kind="tree", q=q, k_pool=pools[0], v_pool=pools[1], tables=tables, context=_i32(lens), counts=counts.to(torch.int32),
                      parents=parents.to(torch.int32).contiguous(), scale=1.0 / math.sqrt(D), out=torch.empty_like(q)),
                 lambda ops, native: ops.tree_attention_workspace(native, q, pools[0], tables))


def _prepare_keep(case, seed):
    n, d = case["seqs"], case["drafts"]
    lens = [case["ctx"]] * n
    tables, pages = _tables([c + d for c in lens], seed)
    gen = _generator(seed, 4)
    pools = torch.randn((case["layers"], 2, pages, case["kv_heads"], BLOCK, case["hs"]), generator=gen, device="cuda", dtype=torch.float16)
    # the accepted path: half of the drafts of the listed cases, at rising places
    counts = _kept(case)
    path = torch.rand((n, d), generator=gen, device="cuda").argsort(1)
    path = torch.where(torch.arange(d, device="cuda") < counts, path, d).sort(1).values.to(torch.int32)
    return _room(dict(kind="keep", pools=pools, tables=tables, context=_i32(lens), path=path, counts=_i32([counts] * n)), lambda ops, native: 0)


def _kept(case):
    return (case["drafts"] + 1) // 2


def _prepare_logprobs(case, seed):
    rows, vocab, gen = case["rows"], case["vocab"], _generator(seed, 5)
    x = torch.randn((rows, vocab), generator=gen, device="cuda") * 3
    x[torch.rand((rows, vocab), generator=gen, device="cuda") < case["banned"]] = -math.inf
    x[:, :64] = torch.randn((rows, 64), generator=gen, device="cuda")       # a row keeps tokens, more than are asked for
    logits = x.to(DTYPES[case["type"]])
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    tokens = torch.where(torch.isfinite(logits.gather(1, tokens[:, None])[:, 0].float()), tokens, tokens % 64).to(torch.int32)
    top = case["top"]
    return _room(dict(kind="logprobs", logits=logits, tokens=tokens, top=top, logprob=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                      top_ids=torch.empty((rows, top), dtype=torch.int32, device="cuda"), top_logprobs=torch.empty((rows, top), device="cuda")),
                 lambda ops, native: ops.token_logprobs_workspace(native, logits, top))


# ------------------------------------------------------------------------------------------------ run
def run(state):
    if own:
        return globals()["_own_" + state["kind"]](state, state["ops"], torch.cuda.current_stream().cuda_stream)
    return globals()["_plain_" + state["kind"]](state)


def _own_packed(s, ops, stream):
    ops.packed_attention(s["native"], s["q"], s["k"], s["v"], s["q_offsets"], s["out"], s["scale"], kv_offsets=s["kv_offsets"], workspace=s["workspace"], stream=stream)
    return {"attention": s["out"]}


def _own_tree(s, ops, stream):
    ops.tree_attention(s["native"], s["q"], s["k_pool"], s["v_pool"], s["tables"], s["context"], s["counts"], s["parents"], s["out"], s["scale"],
                       workspace=s["workspace"], stream=stream)
    return {"attention": s["out"]}


def _own_keep(s, ops, stream):
    ops.cache_keep(s["native"], s["pools"][:, 0], s["pools"][:, 1], s["tables"], s["context"], s["path"], s["counts"], stream=stream)
    return {"pools": s["pools"]}


def _own_logprobs(s, ops, stream):
    ops.token_logprobs(s["native"], s["logits"], s["tokens"], s["logprob"], s["entropy"], s["top_ids"], s["top_logprobs"], workspace=s["workspace"], stream=stream)
    return {"logprob": s["logprob"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top_logprobs": s["top_logprobs"]}


def _softmax_times(scores, visible, v):
    """softmax over the visible scores times v; rows that see nothing are zero. The scores are overwritten."""
    scores.masked_fill_(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_packed(s):
    q_at, kv_at = s["q_offsets"].long(), (s["q_offsets"] if s["kv_offsets"] is None else s["kv_offsets"]).long()
    rows, H, D = s["q"].shape
    G = s["k"].shape[1]
    nq, nk = q_at.diff(), kv_at.diff()
    i, j = torch.arange(s["longest"], device="cuda"), torch.arange(s["most_keys"], device="cuda")
    q_row, kv_row = q_at[:-1, None] + i, (kv_at[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][q_row.clamp(max=rows - 1)].float().view(-1, i.numel(), G, H // G, D).permute(0, 2, 3, 1, 4)
    k, v = (s[x][kv_row].float().transpose(1, 2).unsqueeze(2) for x in ("k", "v"))
    # the last query sees all keys of its sequence, the one before it one less
    visible = (j <= i[:, None] + (nk - nq)[:, None, None])[:, None, None]
    o = _softmax_times(q @ k.transpose(-1, -2) * s["scale"], visible, v)
    out = torch.zeros((rows + 1, H, D), dtype=s["q"].dtype, device="cuda")
    out[torch.where(i < nq[:, None], q_row, rows)] = o.permute(0, 3, 1, 2, 4).reshape(-1, i.numel(), H, D).to(out.dtype)
    return {"attention": out[:rows]}


def _plain_tree(s):
    n, d, H, D = s["q"].shape
    G = s["k_pool"].shape[1]
    k, v = (s[x][s["tables"].long()].transpose(1, 2).reshape(n, G, -1, D).float().unsqueeze(2) for x in ("k_pool", "v_pool"))
    i, j = torch.arange(d, device="cuda"), torch.arange(k.shape[3], device="cuda")
    live = i < s["counts"][:, None]
    # a token sees itself and its ancestors: the paths of any length along the parents
    eye = torch.eye(d, dtype=torch.float64, device="cuda")
    up = torch.linalg.matrix_power(eye + (s["parents"][:, :, None] == i), d) > 0
    at = j - s["context"][:, None]
    drafted = up.gather(2, at.clamp(0, d - 1)[:, None, :].expand(n, d, -1)) & ((at >= 0) & (at < d))[:, None, :]
    visible = ((at < 0)[:, None, :] | drafted) & live[:, :, None]
    q = s["q"].float().view(n, d, G, H // G, D).permute(0, 2, 3, 1, 4)
    o = _softmax_times(q @ k.transpose(-1, -2) * s["scale"], visible[:, None, None], v)
    return {"attention": o.permute(0, 3, 1, 2, 4).reshape(n, d, H, D).half()}


def _plain_keep(s):
    n, d = s["path"].shape
    j = torch.arange(d, device="cuda")
    to = s["context"][:, None].long() + j
    # what is not kept stays where it is
    src = torch.where(j < s["counts"][:, None], s["context"][:, None] + s["path"], to)
    page = lambda t: s["tables"].long().gather(1, t // BLOCK)  # noqa: E731
    s["pools"][:, :, page(to), :, to % BLOCK] = s["pools"][:, :, page(src), :, src % BLOCK]
    return {"pools": s["pools"]}


def _plain_logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    z = x - top
    p = z.exp()
    total = p.sum(-1)
    log_total = total.log()
    entropy = log_total - torch.where(p > 0, p * z, 0).sum(-1) / total
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    return {"logprob": z.gather(1, s["tokens"].long()[:, None])[:, 0] - log_total, "entropy": entropy, "top_ids": ids.to(torch.int32),
            "top_logprobs": z.gather(1, ids) - log_total[:, None]}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: what the operator reads and writes once. FLOPs: two products of every visible (query, key) pair and head."""
    kind, elem = case["kind"], {"f32": 4}.get(case.get("type"), 2)
    if kind == "logprobs":
        return {"bytes": case["rows"] * (case["vocab"] * elem + 12 + 8 * case["top"]), "flops": 4 * case["rows"] * case["vocab"]}
    if kind == "keep":
        # keys and values of the kept drafts that are not in place already, read and written
        return {"bytes": case["seqs"] * (_kept(case) * case["layers"] * case["kv_heads"] * case["hs"] * 2 * 2 * 2 + 8 * case["drafts"]), "flops": 0}
    H, G, D = case["heads"], case["kv_heads"], case["hs"]
    if kind == "tree":
        d, total = case["drafts"], sum(_spread(case))
        return {"bytes": 4 * G * D * (total + case["seqs"] * d) + 4 * case["seqs"] * d * H * D, "flops": 4 * H * D * d * (total + case["seqs"] * (d + 1) // 2)}
    lens, cached = _spread(case), _cached(case)
    pairs = sum(n * (n + 1) // 2 + n * c for n, c in zip(lens, cached))
    return {"bytes": 4 * H * D * sum(lens) + 4 * G * D * (sum(lens) + sum(cached)), "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


def _attend(q, k, v, scale, seen):
    """One sequence and one KV head: q [heads of the group, rows, D], k and v [keys, D], seen [rows, keys], all in f64."""
    w = torch.exp(torch.einsum("hid,jd->hij", q, k) * scale) * seen
    return torch.einsum("hij,jd->hid", w, v) / w.sum(2, keepdim=True)


def _exact_packed(s):
    q_at = s["q_offsets"].tolist()
    kv_at = q_at if s["kv_offsets"] is None else s["kv_offsets"].tolist()
    G = s["k"].shape[1]
    group = s["q"].shape[1] // G
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for a, b, c, e in zip(q_at, q_at[1:], kv_at, kv_at[1:]):
        for g in range(G):
            h = slice(g * group, (g + 1) * group)
            k, v = s["k"][c:e, g].double(), s["v"][c:e, g].double()
            for r in range(a, b, 1024):     # so many queries at a time
                rows = torch.arange(r, min(r + 1024, b), device="cuda")
                seen = torch.arange(e - c, device="cuda") <= (rows - b + e - c)[:, None]
                out[rows, h] = _attend(s["q"][rows, h].double().transpose(0, 1), k, v, s["scale"], seen).transpose(0, 1)
    return {"attention": out}


def _exact_tree(s):
    n, d, H, D = s["q"].shape
    G, context, counts, parents = s["k_pool"].shape[1], s["context"].tolist(), s["counts"].tolist(), s["parents"].tolist()
    out = torch.zeros((n, d, H, D), dtype=torch.float64, device="cuda")
    for b in range(n):
        c, m = context[b], counts[b]
        seen = torch.zeros((m, c + m), dtype=torch.bool)
        seen[:, :c] = True
        for i in range(m):
            a = i
            while a >= 0:
                seen[i, c + a] = True
                a = parents[b][a]
        token = torch.arange(c + m, device="cuda")
        page = s["tables"][b].long()[token // BLOCK]
        for g in range(G):
            h = slice(g * (H // G), (g + 1) * (H // G))
            k, v = (s[x][page, g, token % BLOCK].double() for x in ("k_pool", "v_pool"))
            out[b, :m, h] = _attend(s["q"][b, :m, h].double().transpose(0, 1), k, v, s["scale"], seen.cuda()).transpose(0, 1)
    return {"attention": out}


def _exact_keep(s):
    pools = s["pools"].double()
    tables, context, path, counts = (s[x].tolist() for x in ("tables", "context", "path", "counts"))
    moves = [(b, context[b] + path[b][j], context[b] + j) for b in range(len(counts)) for j in range(counts[b])]
    taken = [s["pools"][:, :, tables[b][a // BLOCK], :, a % BLOCK].double() for b, a, _ in moves]
    for (b, _, to), rows in zip(moves, taken):
        pools[:, :, tables[b][to // BLOCK], :, to % BLOCK] = rows
    return {"pools": pools}


def _exact_logprobs(s):
    x = s["logits"].double()
    w = torch.exp(x)
    log_total = torch.log(w.sum(1))
    lp = x - log_total[:, None]
    entropy = -torch.nan_to_num(w / w.sum(1, keepdim=True) * lp, nan=0.0).sum(1)
    ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :s["top"]]
    rows = torch.arange(x.shape[0], device="cuda")
    return {"logprob": lp[rows, s["tokens"].long()], "entropy": entropy, "top_ids": None, "top_logprobs": lp.gather(1, ids)}
