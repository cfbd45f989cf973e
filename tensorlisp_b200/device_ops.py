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
import struct

from . import _lib
from ._lib import TLB_INVALID, TlbError, check
from .graph import BF16, F16, F32, I8, I16, I32, I64

__all__ = ["DeviceArray", "cache_keep", "packed_attention", "packed_attention_workspace", "token_logprobs", "token_logprobs_workspace",
           "tree_attention", "tree_attention_workspace"]

_CODES = {"float32": F32, "float16": F16, "bfloat16": BF16, "int32": I32, "int64": I64, "int16": I16, "int8": I8, "uint8": I8,
          "<f4": F32, "<f2": F16, "<i4": I32, "<i8": I64, "<i2": I16, "|i1": I8, "|u1": I8}
_SIZE = {F32: 4, F16: 2, BF16: 2, I32: 4, I64: 8, I16: 2, I8: 1}
_NAMES = {F32: "f32", F16: "f16", BF16: "bf16", I32: "i32"}
_HALVES, _HALF, _INTS, _FLOATS, _ROOM = (F16, BF16), (F16,), (I32,), (F32, F16, BF16), tuple(_SIZE)
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
    """(address, ggml type, shape, strides in elements or None where they are dense, dense) of an array of one of `types` with `ndim` dimensions on the
    handle's device."""
    try:        # a torch tensor whose type has been seen
        code, shape, dense = _dtypes[x.dtype], x.shape, x.is_contiguous()
        if code in types and len(shape) == ndim and x.get_device() == native.ordinal:
            return x.data_ptr(), code, shape, None if dense else x.stride(), dense
    except (AttributeError, KeyError):
        pass
    if hasattr(x, "data_ptr"):
        code, shape, strides, ptr = _code(x.dtype), x.shape, x.stride(), x.data_ptr()
        if x.get_device() != native.ordinal:
            _invalid("%s lies on another device than the handle's (GPU %d)" % (name, native.ordinal))
    else:
        face = getattr(x, "__cuda_array_interface__", None)
        if face is None:
            _invalid("%s is not an array in device memory" % name)
        code, shape, ptr, strides = _code(face["typestr"]), face["shape"], face["data"][0], face.get("strides")
        size = _SIZE.get(code, 1)
        if strides is not None:
            if any(b % size for b in strides):
                _invalid("%s has strides that are no whole elements" % name)
            strides = [b // size for b in strides]
    if code not in types:
        _invalid("%s must be %s" % (name, " or ".join(_NAMES[t] for t in types)))
    if len(shape) != ndim:
        _invalid("%s must have %d dimensions, got %d" % (name, ndim, len(shape)))
    return ptr, code, shape, strides, strides is None


def _dense(view, name: str, first: int = 0) -> None:
    """Dimensions from `first` on are dense."""
    if view[4]:
        return
    _, _, shape, strides, _ = view
    if 0 in shape:
        return
    n = 1
    for i in range(len(shape) - 1, first - 1, -1):
        if strides[i] != n and shape[i] > 1:
            _invalid("%s must be dense" % name if first == 0 else "%s must be dense from dimension %d on" % (name, first))
        n *= shape[i]


def _array(native, x, name: str, code: int, shape: tuple) -> int:
    """The address of a dense array of one type and shape, 0 for None."""
    if x is None:
        return 0
    try:
        if x.shape == shape and _dtypes[x.dtype] == code and x.is_contiguous() and x.get_device() == native.ordinal:
            return x.data_ptr()
    except (AttributeError, KeyError):
        pass
    v = _view(native, x, name, (code,), len(shape))
    if tuple(v[2]) != shape:
        _invalid("%s must have the shape %s, got %s" % (name, shape, tuple(v[2])))
    _dense(v, name)
    return v[0]


def _given(x, name: str):
    if x is None:
        _invalid("%s is not an array in device memory" % name)
    return x


def _step(view, row: int) -> int:
    """Bytes from row to row, for rows of `row` bytes."""
    return row if view[4] or view[2][0] < 2 else view[3][0] * _SIZE[view[1]]


def _room(native, workspace) -> tuple:
    if workspace is None:
        return 0, 0
    ptr, code, shape, _, _ = v = _view(native, workspace, "workspace", _ROOM, 1)
    _dense(v, "workspace")
    return ptr, shape[0] * _SIZE[code]


def _stream(stream):
    if stream is None:
        return None
    stream = getattr(stream, "cuda_stream", stream)
    return 1 if stream == 0 else stream      # cudaStreamLegacy: NULL is the library's own


def _layout(args) -> struct.Struct:
    """A structure of the header as struct.pack fills it: a call makes its arguments in one go (a ctypes structure takes them one by one)."""
    return struct.Struct("@" + "".join({C.c_uint32: "I", C.c_uint64: "Q", C.c_float: "f", C.c_void_p: "P"}[t] for _, t in args._fields_) + "0P")


def _pack(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except (struct.error, OverflowError) as e:
        _invalid("an argument is out of range: %s" % e)


_PACKED, _TREE = _layout(_lib.tlb_packed_attention_args), _layout(_lib.tlb_tree_attention_args)
_KEEP, _SCORES = _layout(_lib.tlb_cache_keep_args), _layout(_lib.tlb_token_logprobs_args)


# ------------------------------------------------------------------------------------------------ packed sequences
def _packed_args(native, q, k, seqs, scale, v=None, out=None, q_offsets=0, kv_offsets=0, workspace=None, status=None):
    Q, K = _view(native, q, "q", _HALVES, 3), _view(native, k, "k", _HALVES, 3)
    types = (Q[1],)
    V = K if v is None else _view(native, v, "v", types, 3)
    O = Q if out is None else _view(native, out, "out", types, 3)
    if K[1] != Q[1]:
        _invalid("k must have the type of q")
    (rows, heads, size), (kv_rows, kv_heads, kv_size) = Q[2], K[2]
    row, kv_row = heads * size * 2, kv_heads * size * 2
    if V[2] != K[2] or O[2] != Q[2] or kv_size != size:
        _invalid("q and out are [rows, heads, head size], k and v [rows, kv heads, head size]")
    _dense(Q, "q", 1)
    _dense(K, "k", 1)
    _dense(V, "v", 1)
    _dense(O, "out", 1)
    room, room_bytes = _room(native, workspace)
    return _pack(_PACKED, Q[1], seqs, heads, kv_heads, size, 1.0 / math.sqrt(max(size, 1)) if scale is None else scale, rows, kv_rows, Q[0], K[0], V[0], O[0],
                        _step(Q, row), _step(K, kv_row), _step(V, kv_row), _step(O, row), q_offsets, kv_offsets, room, room_bytes, _array(native, status, "status", I32, (1,)))


def packed_attention_workspace(native, q, k, seqs: int) -> int:
    """Bytes of workspace for ``packed_attention`` of arrays of these shapes and `seqs` sequences."""
    return int(native.L.tlb_packed_attention_workspace(native.dev, _packed_args(native, q, k, seqs, None)))


def packed_attention(native, q, k, v, q_offsets, out, scale: float | None = None, *, kv_offsets=None, workspace=None, status=None, stream=None) -> None:
    """Causal attention of packed sequences into `out`: q and out [rows, heads, head size], k and v [rows, kv heads, head size] (f16 or
    bf16; rows may be strided), q_offsets and kv_offsets i32 [sequences + 1]. Sequence s has the query rows q_offsets[s]:q_offsets[s + 1] and the
    keys kv_offsets[s]:kv_offsets[s + 1] (None: the same rows); its last query sees all of its keys, the one before it one less, and so
    on. Rows of no sequence are left as they were. `scale` defaults to 1 / sqrt(head size)."""
    at = _view(native, q_offsets, "q_offsets", _INTS, 1)
    _dense(at, "q_offsets")
    seqs = at[2][0] - 1
    if seqs < 0:
        _invalid("q_offsets holds sequences + 1 numbers")
    a = _packed_args(native, q, k, seqs, scale, _given(v, "v"), _given(out, "out"), at[0], _array(native, kv_offsets, "kv_offsets", I32, (seqs + 1,)), workspace, status)
    check(native.L.tlb_packed_attention(native.dev, a, _stream(stream)))


# ------------------------------------------------------------------------------------------------ drafted tokens
def _tree_args(native, q, k_pool, tables, scale, v_pool=None, out=None, context=None, counts=None, parents=None, workspace=None, status=None):
    Q, K, T = _view(native, q, "q", _HALF, 4), _view(native, k_pool, "k_pool", _HALF, 4), _view(native, tables, "tables", _INTS, 2)
    V = K if v_pool is None else _view(native, v_pool, "v_pool", _HALF, 4)
    O = Q if out is None else _view(native, out, "out", _HALF, 4)
    (seqs, drafts, heads, size), (pages, kv_heads, block_size, kv_size) = Q[2], K[2]
    if V[2] != K[2] or O[2] != Q[2] or kv_size != size:
        _invalid("q and out are [sequences, drafts, heads, head size], the pools [pages, kv heads, block size, head size]")
    if T[2][0] != seqs:
        _invalid("one block-table row per sequence")
    _dense(Q, "q")
    _dense(K, "k_pool")
    _dense(V, "v_pool")
    _dense(O, "out")
    _dense(T, "tables")
    room, room_bytes = _room(native, workspace)
    return _pack(_TREE, seqs, drafts, heads, kv_heads, size, block_size, T[2][1], 1.0 / math.sqrt(max(size, 1)) if scale is None else scale, pages, Q[0], K[0], V[0], O[0],
                      T[0], _array(native, context, "context", I32, (seqs,)), _array(native, counts, "counts", I32, (seqs,)),
                      _array(native, parents, "parents", I32, (seqs, drafts)), room, room_bytes, _array(native, status, "status", I32, (1,)))


def tree_attention_workspace(native, q, k_pool, tables) -> int:
    """Bytes of workspace for ``tree_attention`` of arrays of these shapes."""
    return int(native.L.tlb_tree_attention_workspace(native.dev, _tree_args(native, q, k_pool, tables, None)))


def tree_attention(native, q, k_pool, v_pool, tables, context, counts, parents, out, scale: float | None = None, *, workspace=None, status=None, stream=None) -> None:
    """Attention of drafted tokens over the paged cache into `out` (f16): q and out [sequences, drafts, heads, head size], the pools
    [pages, kv heads, block size, head size], tables i32 [sequences, pages of a sequence], context and counts i32 [sequences], parents
    i32 [sequences, drafts]. Draft i of a sequence lies at position context + i of its cache and sees the context, itself and its ancestors:
    parents[i] is an earlier draft, or -1. Rows from counts on are padding and become zero."""
    a = _tree_args(native, q, k_pool, tables, scale, _given(v_pool, "v_pool"), _given(out, "out"), _given(context, "context"), _given(counts, "counts"),
                   _given(parents, "parents"), workspace, status)
    check(native.L.tlb_tree_attention(native.dev, a, _stream(stream)))


def cache_keep(native, k_pools, v_pools, tables, context, path, counts, *, status=None, stream=None) -> None:
    """Moves accepted drafts into place: k_pools and v_pools f16 [layers, pages, kv heads, block size, head size] (layers may be strided), tables
    i32 [sequences, pages of a sequence], context and counts i32 [sequences], path i32 [sequences, drafts]. For j < counts[s], position
    context[s] + path[s, j] of sequence s goes to position context[s] + j; a row of path rises."""
    K, V = _view(native, k_pools, "k_pools", _HALF, 5), _view(native, v_pools, "v_pools", _HALF, 5)
    T, P = _view(native, tables, "tables", _INTS, 2), _view(native, path, "path", _INTS, 2)
    if V[2] != K[2]:
        _invalid("the pools are [layers, pages, kv heads, block size, head size]")
    layers, pages, kv_heads, block_size, size = K[2]
    n, drafts = P[2]
    if T[2][0] != n:
        _invalid("one path per sequence")
    _dense(K, "k_pools", 1)
    _dense(V, "v_pools", 1)
    _dense(T, "tables")
    _dense(P, "path")
    pool = pages * kv_heads * block_size * size * 2
    a = _pack(_KEEP, layers, n, drafts, kv_heads, size, block_size, T[2][1], pages, K[0], V[0], _step(K, pool), _step(V, pool), T[0],
                   _array(native, _given(context, "context"), "context", I32, (n,)), _array(native, _given(counts, "counts"), "counts", I32, (n,)), P[0],
                   _array(native, status, "status", I32, (1,)))
    check(native.L.tlb_cache_keep(native.dev, a, _stream(stream)))


# ------------------------------------------------------------------------------------------------ scores of tokens
def token_logprobs_workspace(native, logits, top: int) -> int:
    """Bytes of workspace for ``token_logprobs`` of logits of this shape with `top` alternatives."""
    L = _view(native, logits, "logits", _FLOATS, 2)
    return int(native.L.tlb_token_logprobs_workspace(native.dev, _pack(_SCORES, L[1], top, L[2][0], L[2][1], 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)))


def token_logprobs(native, logits, tokens, logprob, entropy=None, top_ids=None, top_logprobs=None, *, workspace=None, status=None, stream=None) -> None:
    """Of each row of logits [rows, vocabulary] (f32, f16 or bf16; rows may be strided): the log probability of tokens[row] (i32 [rows], -1: none,
    0 is written) into `logprob` (f32 [rows]), the entropy in nats into `entropy`, and the most likely tokens, equal logits by rising id, into
    `top_ids` (i32 [rows, top], top up to 32) and `top_logprobs` (f32). tokens and logprob, entropy, and both top arrays may be None."""
    L = _view(native, logits, "logits", _FLOATS, 2)
    _dense(L, "logits", 1)
    rows, vocab = L[2]
    top = 0
    if (top_ids is None) != (top_logprobs is None):
        _invalid("top_ids and top_logprobs come together")
    if top_ids is not None:
        I = _view(native, top_ids, "top_ids", _INTS, 2)
        if I[2][0] != rows:
            _invalid("top_ids must have a row for each row of the logits")
        top = I[2][1]
    room, room_bytes = _room(native, workspace)
    a = _pack(_SCORES, L[1], top, rows, vocab, L[0], _step(L, vocab * _SIZE[L[1]]), _array(native, tokens, "tokens", I32, (rows,)), _array(native, logprob, "logprob", F32, (rows,)),
                     _array(native, entropy, "entropy", F32, (rows,)), _array(native, top_ids, "top_ids", I32, (rows, top)),
                     _array(native, top_logprobs, "top_logprobs", F32, (rows, top)), room, room_bytes, _array(native, status, "status", I32, (1,)))
    check(native.L.tlb_token_logprobs(native.dev, a, _stream(stream)))
