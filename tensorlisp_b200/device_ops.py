"""The serving operators of include/tlb200.h on arrays that lie in device memory: attention over packed prompts, attention of
drafted tokens over the paged cache, moving accepted drafts into place, log probabilities of tokens. ``Graph`` has the same
operators as nodes (``packed_attention``, ``paged_tree_attention``, ``token_logprobs``).

An array is anything with ``__cuda_array_interface__``, or with the ``data_ptr() / dtype / shape / stride()`` of a torch tensor (which is
how bf16 gets here); ``DeviceArray`` describes memory of the library itself, a pool of a state block for instance. A call enqueues and
returns. ``stream`` is a CUDA stream handle or an object with ``cuda_stream`` (0: the legacy default stream), None the library's own
(``Native.stream``): arrays written on another stream are the caller's to order, and memory that a caching allocator gave out has
to stay allocated until the call has run. ``workspace`` is scratch memory of at least the bytes that the ``_workspace`` function
says, without initial content; calls that may overlap in time, two captured graphs among them, need one each. ``status`` (i32, one value,
zero) becomes 4 when a number in device memory pointed outside and was not followed.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib
from ._lib import TLB_INVALID, TlbError, check
from .graph import BF16, F16, F32, I8, I16, I32, I64

__all__ = ["DeviceArray", "cache_keep", "packed_attention", "packed_attention_workspace", "token_logprobs", "token_logprobs_workspace",
           "tree_attention", "tree_attention_workspace"]

_CODES = {"float32": F32, "float16": F16, "bfloat16": BF16, "int32": I32, "int64": I64, "int16": I16, "int8": I8, "uint8": I8,
          "<f4": F32, "<f2": F16, "<i4": I32, "<i8": I64, "<i2": I16, "|i1": I8, "|u1": I8}
_SIZE = {F32: 4, F16: 2, BF16: 2, I32: 4, I64: 8, I16: 2, I8: 1}
_NAMES = {F32: "f32", F16: "f16", BF16: "bf16", I32: "i32"}
_dtypes: dict = {}      # a dtype object as seen before -> ggml type


class DeviceArray:
    """Device memory at `ptr` as an array; `strides` in bytes (None: dense). `owner` is kept alive with it."""

    def __init__(self, ptr: int, shape, typestr: str, strides=None, owner=None) -> None:
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False), "version": 3,
                                         "strides": None if strides is None else tuple(strides)}


def _invalid(message: str):
    raise TlbError(TLB_INVALID, message)


def _code(dtype) -> int:
    code = _dtypes.get(dtype)
    if code is None:
        code = _dtypes[dtype] = _CODES.get(str(dtype).rsplit(".", 1)[-1], -1)
    return code


def _view(native, x, name: str, types, ndim: int):
    """(address, ggml type, shape, strides in bytes) of an array of one of `types` with `ndim` dimensions on the handle's device."""
    if hasattr(x, "data_ptr"):
        code, shape = _code(x.dtype), x.shape
        if x.get_device() != native.ordinal:
            _invalid("%s lies on another device than the handle's (GPU %d)" % (name, native.ordinal))
        size = _SIZE.get(code, 1)
        strides = [s * size for s in x.stride()]
        ptr = x.data_ptr()
    else:
        face = getattr(x, "__cuda_array_interface__", None)
        if face is None:
            _invalid("%s is not an array in device memory" % name)
        code, shape, ptr, strides = _code(face["typestr"]), face["shape"], face["data"][0], face.get("strides")
        if strides is None:
            strides, n = [0] * len(shape), _SIZE.get(code, 1)
            for i in range(len(shape) - 1, -1, -1):
                strides[i] = n
                n *= shape[i]
    if code not in types:
        _invalid("%s must be %s" % (name, " or ".join(_NAMES[t] for t in types)))
    if len(shape) != ndim:
        _invalid("%s must have %d dimensions, got %d" % (name, ndim, len(shape)))
    return ptr, code, shape, strides


def _dense(view, name: str, first: int = 0) -> None:
    """Dimensions from `first` on are dense."""
    _, code, shape, strides = view
    if 0 in shape:
        return
    n = _SIZE[code]
    for i in range(len(shape) - 1, first - 1, -1):
        if strides[i] != n and shape[i] > 1:
            _invalid("%s must be dense" % name if first == 0 else "%s must be dense from dimension %d on" % (name, first))
        n *= shape[i]


def _numbers(native, x, name: str, shape) -> int:
    v = _view(native, x, name, (I32,), len(shape))
    if tuple(v[2]) != shape:
        _invalid("%s must have the shape %s, got %s" % (name, shape, tuple(v[2])))
    _dense(v, name)
    return v[0]


def _optional(native, x, name: str, shape) -> int | None:
    return None if x is None else _numbers(native, x, name, shape)


def _step(view) -> int:
    """Bytes from row to row; those of a dense row where there are not two."""
    _, code, shape, strides = view
    if shape[0] > 1:
        return strides[0]
    n = _SIZE[code]
    for d in shape[1:]:
        n *= d
    return n


def _room(native, workspace) -> tuple:
    if workspace is None:
        return None, 0
    ptr, code, shape, _ = v = _view(native, workspace, "workspace", tuple(_SIZE), 1)
    _dense(v, "workspace")
    return ptr, shape[0] * _SIZE[code]


def _stream(stream):
    if stream is None:
        return None
    stream = getattr(stream, "cuda_stream", stream)
    return 1 if stream == 0 else stream      # cudaStreamLegacy: NULL is the library's own


# ------------------------------------------------------------------------------------------------ packed sequences
def _packed_args(native, q, k, seqs, scale, workspace=(None, 0), v=None, out=None, q_offsets=None, kv_offsets=None, status=None):
    Q, K = _view(native, q, "q", (F16, BF16), 3), _view(native, k, "k", (F16, BF16), 3)
    types = (Q[1],)
    V = K if v is None else _view(native, v, "v", types, 3)
    O = Q if out is None else _view(native, out, "out", types, 3)
    if K[1] != Q[1]:
        _invalid("k must have the type of q")
    if tuple(V[2]) != tuple(K[2]) or tuple(O[2]) != tuple(Q[2]) or K[2][2] != Q[2][2]:
        _invalid("q and out are [rows, heads, head size], k and v [rows, kv heads, head size]")
    for view, name in ((Q, "q"), (K, "k"), (V, "v"), (O, "out")):
        _dense(view, name, 1)
    return _lib.tlb_packed_attention_args(
        Q[1], seqs, Q[2][1], K[2][1], Q[2][2], scale if scale is not None else 1.0 / math.sqrt(max(Q[2][2], 1)), Q[2][0], K[2][0], Q[0], K[0], V[0], O[0],
        _step(Q), _step(K), _step(V), _step(O), q_offsets, kv_offsets, workspace[0], workspace[1], status)


def packed_attention_workspace(native, q, k, seqs: int) -> int:
    """Bytes of workspace for ``packed_attention`` of arrays of these shapes and `seqs` sequences."""
    a = _packed_args(native, q, k, seqs, None)
    return int(native.L.tlb_packed_attention_workspace(native.dev, C.byref(a)))


def packed_attention(native, q, k, v, q_offsets, out, scale: float | None = None, *, kv_offsets=None, workspace=None, status=None, stream=None) -> None:
    """Causal attention of packed sequences into `out`: q and out [rows, heads, head size], k and v [rows, kv heads, head size] (f16 or
    bf16; rows may be strided), q_offsets and kv_offsets i32 [sequences + 1]. Sequence s has the query rows q_offsets[s]:q_offsets[s + 1] and the
    keys kv_offsets[s]:kv_offsets[s + 1] (None: the same rows); its last query sees all of its keys, the one before it one less, and so
    on. Rows of no sequence are left as they were. `scale` defaults to 1 / sqrt(head size)."""
    at = _view(native, q_offsets, "q_offsets", (I32,), 1)
    _dense(at, "q_offsets")
    seqs = at[2][0] - 1
    if seqs < 0:
        _invalid("q_offsets holds sequences + 1 numbers")
    a = _packed_args(native, q, k, seqs, scale, _room(native, workspace), v, out, at[0], _optional(native, kv_offsets, "kv_offsets", (seqs + 1,)),
                     _optional(native, status, "status", (1,)))
    check(native.L.tlb_packed_attention(native.dev, C.byref(a), _stream(stream)))


# ------------------------------------------------------------------------------------------------ drafted tokens
def _tree_args(native, q, k_pool, tables, scale, v_pool=None, out=None, context=None, counts=None, parents=None, workspace=(None, 0), status=None):
    Q, K, T = _view(native, q, "q", (F16,), 4), _view(native, k_pool, "k_pool", (F16,), 4), _view(native, tables, "tables", (I32,), 2)
    V = K if v_pool is None else _view(native, v_pool, "v_pool", (F16,), 4)
    O = Q if out is None else _view(native, out, "out", (F16,), 4)
    if tuple(V[2]) != tuple(K[2]) or tuple(O[2]) != tuple(Q[2]) or K[2][3] != Q[2][3]:
        _invalid("q and out are [sequences, drafts, heads, head size], the pools [pages, kv heads, block size, head size]")
    if T[2][0] != Q[2][0]:
        _invalid("one block-table row per sequence")
    for view, name in ((Q, "q"), (K, "k_pool"), (V, "v_pool"), (O, "out"), (T, "tables")):
        _dense(view, name)
    return _lib.tlb_tree_attention_args(
        Q[2][0], Q[2][1], Q[2][2], K[2][1], Q[2][3], K[2][2], T[2][1], scale if scale is not None else 1.0 / math.sqrt(max(Q[2][3], 1)), K[2][0], Q[0], K[0], V[0], O[0],
        T[0], context, counts, parents, workspace[0], workspace[1], status)


def tree_attention_workspace(native, q, k_pool, tables) -> int:
    """Bytes of workspace for ``tree_attention`` of arrays of these shapes."""
    a = _tree_args(native, q, k_pool, tables, None)
    return int(native.L.tlb_tree_attention_workspace(native.dev, C.byref(a)))


def tree_attention(native, q, k_pool, v_pool, tables, context, counts, parents, out, scale: float | None = None, *, workspace=None, status=None, stream=None) -> None:
    """Attention of drafted tokens over the paged cache into `out` (f16): q and out [sequences, drafts, heads, head size], the pools
    [pages, kv heads, block size, head size], tables i32 [sequences, pages of a sequence], context and counts i32 [sequences], parents
    i32 [sequences, drafts]. Draft i of a sequence lies at position context + i of its cache and sees the context, itself and its ancestors:
    parents[i] is an earlier draft, or -1. Rows from counts on are padding and become zero."""
    shape = tuple(getattr(q, "shape", None) or q.__cuda_array_interface__["shape"])
    if len(shape) != 4:
        _invalid("q must have 4 dimensions, got %d" % len(shape))
    a = _tree_args(native, q, k_pool, tables, scale, v_pool, out, _numbers(native, context, "context", shape[:1]), _numbers(native, counts, "counts", shape[:1]),
                   _numbers(native, parents, "parents", shape[:2]), _room(native, workspace), _optional(native, status, "status", (1,)))
    check(native.L.tlb_tree_attention(native.dev, C.byref(a), _stream(stream)))


def cache_keep(native, k_pools, v_pools, tables, context, path, counts, *, status=None, stream=None) -> None:
    """Moves accepted drafts into place: k_pools and v_pools f16 [layers, pages, kv heads, block size, head size] (layers may be strided), tables
    i32 [sequences, pages of a sequence], context and counts i32 [sequences], path i32 [sequences, drafts]. For j < counts[s], position
    context[s] + path[s, j] of sequence s goes to position context[s] + j; a row of path rises."""
    K, V = _view(native, k_pools, "k_pools", (F16,), 5), _view(native, v_pools, "v_pools", (F16,), 5)
    T, P = _view(native, tables, "tables", (I32,), 2), _view(native, path, "path", (I32,), 2)
    if tuple(V[2]) != tuple(K[2]):
        _invalid("the pools are [layers, pages, kv heads, block size, head size]")
    n = T[2][0]
    if P[2][0] != n:
        _invalid("one path per sequence")
    _dense(K, "k_pools", 1)
    _dense(V, "v_pools", 1)
    _dense(T, "tables")
    _dense(P, "path")
    a = _lib.tlb_cache_keep_args(K[2][0], n, P[2][1], K[2][2], K[2][4], K[2][3], T[2][1], K[2][1], K[0], V[0], _step(K), _step(V), T[0],
                                 _numbers(native, context, "context", (n,)), _numbers(native, counts, "counts", (n,)), P[0], _optional(native, status, "status", (1,)))
    check(native.L.tlb_cache_keep(native.dev, C.byref(a), _stream(stream)))


# ------------------------------------------------------------------------------------------------ scores of tokens
def token_logprobs_workspace(native, logits, top: int) -> int:
    """Bytes of workspace for ``token_logprobs`` of logits of this shape with `top` alternatives."""
    L = _view(native, logits, "logits", (F32, F16, BF16), 2)
    a = _lib.tlb_token_logprobs_args(L[1], top, L[2][0], L[2][1])
    return int(native.L.tlb_token_logprobs_workspace(native.dev, C.byref(a)))


def token_logprobs(native, logits, tokens, logprob, entropy=None, top_ids=None, top_logprobs=None, *, workspace=None, status=None, stream=None) -> None:
    """Of each row of logits [rows, vocabulary] (f32, f16 or bf16; rows may be strided): the log probability of tokens[row] (i32 [rows], -1: none,
    0 is written) into `logprob` (f32 [rows]), the entropy in nats into `entropy`, and the most likely tokens, equal logits by rising id, into
    `top_ids` (i32 [rows, top], top up to 32) and `top_logprobs` (f32). tokens and logprob, entropy, and both top arrays may be None."""
    L = _view(native, logits, "logits", (F32, F16, BF16), 2)
    _dense(L, "logits", 1)
    rows, vocab = L[2]

    def floats(x, name, shape):
        if x is None:
            return None
        v = _view(native, x, name, (F32,), len(shape))
        if tuple(v[2]) != shape:
            _invalid("%s must have the shape %s, got %s" % (name, shape, tuple(v[2])))
        _dense(v, name)
        return v[0]

    top, ids = 0, None
    if (top_ids is None) != (top_logprobs is None):
        _invalid("top_ids and top_logprobs come together")
    if top_ids is not None:
        I = _view(native, top_ids, "top_ids", (I32,), 2)
        top, ids = I[2][1], I[0]
        if I[2][0] != rows:
            _invalid("top_ids must have a row for each row of the logits")
        _dense(I, "top_ids")
    room = _room(native, workspace)
    a = _lib.tlb_token_logprobs_args(L[1], top, rows, vocab, L[0], _step(L), _optional(native, tokens, "tokens", (rows,)), floats(logprob, "logprob", (rows,)),
                                     floats(entropy, "entropy", (rows,)), ids, floats(top_logprobs, "top_logprobs", (rows, top)), room[0], room[1],
                                     _optional(native, status, "status", (1,)))
    check(native.L.tlb_token_logprobs(native.dev, C.byref(a), _stream(stream)))
