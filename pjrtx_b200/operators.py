"""Operators on device memory: a paged key-value cache, attention of packed prompts and the scoring of a decoder's logits.

Bindings of the `pjrtx_b200_paged_cache_*`, `pjrtx_b200_prompt_attention` and `pjrtx_b200_token_log_probs*` entry points of
include/pjrtx_b200.h, reached through `Backend.paged_cache`, `Backend.prompt_attention`, `Backend.token_log_probs` and
`Backend.token_log_probs_backward`. Arrays are `DeviceBuffer`s or any device tensors with `data_ptr()`, `shape`, `stride()` and
`dtype` (torch's). Types, shapes and the device that an array says it is on (`get_device()` or `device`) are checked here, the rest
behind the C ABI; nothing is copied, cast or kept. Calls enqueue on `stream`, a `cudaStream_t` as an integer (0: the default stream).

`stream=None` is the stream on which the backend's buffers and executables work. It does not wait for the default stream or for a
tensor library's, nor they for it: tensors need the stream that they are worked on given, or events. Buffers are filled and freed
on the backend's stream: a call that gets one on another stream has to be ordered behind its upload, and the buffer kept until the
backend's stream is ordered behind the call.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional, Tuple

from . import plan as P

_P, _I32, _I64, _U64, _F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float


class PagedCacheConfig(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("track", _I32), ("batch", _I64), ("heads", _I64), ("kv_heads", _I64),
                ("head_dim", _I64), ("page_size", _I64), ("max_pages", _I64), ("tree_nodes", _I64)]


class PagedView(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("k_pages", _P), ("v_pages", _P), ("num_pages", _I64), ("page_stride", _I64),
                ("row_stride", _I64), ("head_stride", _I64), ("page_table", _P), ("table_stride", _I64), ("lengths", _P),
                ("batch", _I64), ("tokens", _P), ("weights", _P), ("positions", _P)]


class PagedAppendArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("k_new", _P), ("v_new", _P), ("rows", _I64), ("batch_stride", _I64), ("row_stride", _I64),
                ("head_stride", _I64), ("counts", _P)]


class PagedAttendArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("q", _P), ("q_batch_stride", _I64), ("q_head_stride", _I64), ("out", _P),
                ("out_batch_stride", _I64), ("out_head_stride", _I64), ("lse", _P), ("k_new", _P), ("v_new", _P),
                ("new_batch_stride", _I64), ("new_head_stride", _I64), ("scale", _F32)]


class PagedEvictArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("keep", _I64), ("recent", _I64), ("sinks", _I64), ("lengths_out", _P), ("weights_out", _P),
                ("positions_out", _P)]


class PagedTreeArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("q", _P), ("q_batch_stride", _I64), ("q_node_stride", _I64), ("q_head_stride", _I64), ("out", _P),
                ("out_batch_stride", _I64), ("out_node_stride", _I64), ("out_head_stride", _I64), ("lse", _P), ("k_new", _P), ("v_new", _P),
                ("new_batch_stride", _I64), ("new_node_stride", _I64), ("new_head_stride", _I64), ("parents", _P), ("counts", _P),
                ("nodes", _I64), ("scale", _F32)]


class PagedStoreArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("k_new", _P), ("v_new", _P), ("rows", _I64), ("row_stride", _I64), ("head_stride", _I64), ("slots", _P)]


class PagedAssignArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("batch", _I64), ("lengths", _P), ("held", _P), ("page_table", _P), ("table_stride", _I64),
                ("free_pages", _P), ("free_count", _P), ("num_pages", _I64), ("held_out", _P), ("page_table_out", _P),
                ("table_out_stride", _I64), ("free_pages_out", _P), ("free_count_out", _P), ("starts", _P), ("slots", _P), ("tokens", _I64)]


class PagedPathArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("batch", _I64), ("nodes", _I64), ("page_table", _P), ("table_stride", _I64), ("lengths", _P),
                ("parents", _P), ("leaves", _P), ("slots", _P), ("lengths_out", _P)]


class PromptAttentionArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("scale", _F32), ("q", _P), ("k", _P), ("v", _P), ("out", _P), ("lse", _P),
                ("tokens", _I64), ("heads", _I64), ("kv_heads", _I64), ("head_dim", _I64), ("q_stride", _I64), ("q_head_stride", _I64),
                ("k_stride", _I64), ("k_head_stride", _I64), ("v_stride", _I64), ("v_head_stride", _I64), ("out_stride", _I64),
                ("out_head_stride", _I64), ("starts", _P), ("sequences", _I64)]


class TokenLogProbsArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("top", _I32), ("logits", _P), ("rows", _I64), ("vocab", _I64),
                ("row_stride", _I64), ("tokens", _P), ("scale", _F32), ("log_probs", _P), ("entropy", _P), ("lse", _P),
                ("top_ids", _P), ("top_log_probs", _P)]


class TokenLogProbsBackwardArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("scale", _F32), ("logits", _P), ("grad_logits", _P), ("rows", _I64),
                ("vocab", _I64), ("row_stride", _I64), ("grad_row_stride", _I64), ("tokens", _P), ("lse", _P), ("entropy", _P),
                ("grad_log_probs", _P), ("grad_entropy", _P)]


# Every symbol of the operator section of include/pjrtx_b200.h: name -> (restype, argtypes).
# Argument structs go in as bytes or by reference.
SYMBOLS = {
    "pjrtx_b200_device_stream": (_P, [ctypes.c_int]),
    "pjrtx_b200_buffer_device_pointer": (_P, [_P]),
    "pjrtx_b200_paged_cache_create": (_P, [ctypes.c_int, ctypes.POINTER(PagedCacheConfig)]),
    "pjrtx_b200_paged_cache_destroy": (None, [_P]),
    "pjrtx_b200_paged_cache_append": (ctypes.c_int, [_P, _P, _P, _P]),
    "pjrtx_b200_paged_cache_attend": (ctypes.c_int, [_P, _P, _P, _P]),
    "pjrtx_b200_paged_cache_evict": (ctypes.c_int, [_P, _P, _P, _P]),
    "pjrtx_b200_paged_cache_attend_tree": (ctypes.c_int, [_P, _P, _P, _P]),
    "pjrtx_b200_paged_cache_store": (ctypes.c_int, [_P, _P, _P, _P]),
    "pjrtx_b200_paged_cache_assign": (ctypes.c_int, [_P, _P, _P]),
    "pjrtx_b200_paged_cache_path_slots": (ctypes.c_int, [_P, _P, _P]),
    "pjrtx_b200_prompt_attention": (ctypes.c_int, [ctypes.c_int, _P, _P]),
    "pjrtx_b200_token_log_probs": (ctypes.c_int, [ctypes.c_int, _P, _P]),
    "pjrtx_b200_token_log_probs_backward": (ctypes.c_int, [ctypes.c_int, _P, _P]),
    "pjrtx_b200_operators_status": (ctypes.c_int, [ctypes.c_int, _P]),
}

# Argument structs are packed in one step: filling a ctypes structure field by field takes twice as long as the call itself.
_FORMAT = {_U64: "Q", _I64: "q", _I32: "i", _F32: "f", _P: "P"}


def _packer(cls):
    """pack(*fields behind struct_size) -> the struct as bytes."""
    layout = struct.Struct("@" + "".join(_FORMAT[t] for _, t in cls._fields_) + "0Q")
    assert layout.size == ctypes.sizeof(cls)
    return functools.partial(layout.pack, layout.size)


_pack_view, _pack_append, _pack_attend, _pack_evict, _pack_score, _pack_score_grad = map(
    _packer, (PagedView, PagedAppendArgs, PagedAttendArgs, PagedEvictArgs, TokenLogProbsArgs, TokenLogProbsBackwardArgs))
_pack_tree, _pack_store, _pack_assign, _pack_path, _pack_prompt = map(
    _packer, (PagedTreeArgs, PagedStoreArgs, PagedAssignArgs, PagedPathArgs, PromptAttentionArgs))

_FLOATS = frozenset((P.F32, P.F16, P.BF16_CODE))
_TENSOR_TYPES = {"float32": P.F32, "float16": P.F16, "bfloat16": P.BF16_CODE, "int32": P.S32}
_codes: dict = {}  # a tensor library's dtype object -> element-type code, 0 for the others
_types: dict = {}  # element-type code -> the dtype object seen last


def _error(message: str):
    from .backend import BackendError

    return BackendError("InvalidArgument", message)


def _dims(x) -> Tuple[int, ...]:
    try:
        return x.shape
    except AttributeError:
        return x.dims


def _code(x) -> int:
    dtype = x.dtype
    if isinstance(dtype, int):
        return dtype
    code = _codes.get(dtype)
    if code is None:
        code = _codes[dtype] = _TENSOR_TYPES.get(str(dtype).split(".")[-1], 0)
        if code:
            _types[code] = dtype
    return code


def _place(x):
    """Device address and strides (elements)."""
    try:
        return x.data_ptr(), x.stride()
    except AttributeError:
        strides, step = [], 1
        for d in reversed(x.dims):
            strides.insert(0, step)
            step *= d
        return x.device_pointer or 0, tuple(strides)


def _device(x) -> Optional[int]:
    """Ordinal of the device an array is on, -1 for the host, None where it does not say."""
    try:
        return x.get_device()
    except AttributeError:
        at = getattr(x, "device", None)
    if at is None or isinstance(at, int):
        return at
    return (at.index or 0) if at.type == "cuda" else -1


def _check(x, name: str, dtype: int, shape: Tuple[int, ...], device: int) -> None:
    if _code(x) != dtype:
        raise _error(f"{name} has element type {P.DTYPE_NAMES.get(_code(x), 'other')}, {P.DTYPE_NAMES.get(dtype, dtype)} is needed")
    if _dims(x) != shape:
        raise _error(f"{name} has shape {tuple(_dims(x))}, {shape} is needed")
    at = _device(x)
    if at is not None and at != device:
        raise _error(f"{name} is on {'the host' if at < 0 else f'device {at}'}, device {device} is needed")


def _rows(x, name: str, dtype: int, shape: Tuple[int, ...], device: int):
    """Address and strides of an array whose innermost axis has to be dense."""
    try:  # a tensor that is as it has to be
        if x.shape == shape and _codes[x.dtype] == dtype and x.get_device() == device:
            strides = x.stride()
            if strides[-1] == 1:
                return x.data_ptr(), strides
    except (AttributeError, KeyError):
        pass
    _check(x, name, dtype, shape, device)
    place = _place(x)
    if place[1][-1] != 1 and shape[-1] != 1:
        raise _error(f"{name} has stride {place[1][-1]} along its last axis, which has to be dense")
    return place


def _twin(x, name: str, like: str, dtype: int, shape: Tuple[int, ...], strides, device: int) -> int:
    """Address of an array that has the type, shape and strides of another one."""
    try:
        if x.shape == shape and _codes[x.dtype] == dtype and x.stride() == strides and x.get_device() == device:
            return x.data_ptr()
    except (AttributeError, KeyError):
        pass
    if _code(x) != dtype or _dims(x) != shape:
        raise _error(f"{like} and {name} differ in type or shape")
    _check(x, name, dtype, shape, device)
    pointer, own = _place(x)
    if own != strides:
        raise _error(f"{like} and {name} differ in their strides")
    return pointer


def _dense(x, name: str, dtype: int, shape: Tuple[int, ...], device: int) -> int:
    """Address of an array that has to be dense; None is 0."""
    if x is None:
        return 0
    try:
        if x.shape == shape and _codes[x.dtype] == dtype and x.is_contiguous() and x.get_device() == device:
            return x.data_ptr()
    except (AttributeError, KeyError):
        pass
    _check(x, name, dtype, shape, device)
    pointer, strides = _place(x)
    step = 1
    for d, s in zip(reversed(shape), reversed(strides)):
        if s != step and d != 1 and 0 not in shape:
            raise _error(f"{name} has to be dense, its strides are {strides}")
        step *= d
    return pointer


# (library, handle) of caches that the collector found. Freeing one waits for the device, which would end a stream capture that is
# under way wherever the collector happens to run, so it is done where the caller waits for the device anyway.
_unreferenced: list = []


def free_unreferenced() -> None:
    try:
        while True:
            lib, handle = _unreferenced.pop()
            lib.pjrtx_b200_paged_cache_destroy(handle)
    except IndexError:  # empty, if only because another thread was faster
        pass


class PagedCache:
    """Geometry and workspaces of a paged key-value cache: one handle serves all layers of a shape, on one stream at a time.

    Pools are [pages, page_size, kv_heads, head_dim] in any layout that keeps the last axis dense and rows 16-byte aligned,
    the same for keys and values. Row t of sequence b is row t % page_size of page page_table[b, t // page_size]; `lengths[b]`
    counts the rows of a sequence, those that a call appends among them. With `track`, weights and positions are
    [batch, kv_heads, max_pages * page_size], and `tokens[b]` counts the tokens a sequence has seen. Calls go to `stream`, None: the
    backend's own, which is not ordered with any stream of a tensor library.

    `tree` is how many drafted tokens of a sequence `attend_tree` can take, up to 64; it sizes a workspace.

    `destroy` waits for the device and frees the workspaces; those of a cache that is only dropped are freed by the next `destroy`,
    `Backend.paged_cache` or `Backend.synchronize`.
    """

    def __init__(self, backend, dtype: int, batch: int, heads: int, kv_heads: int, head_dim: int, page_size: int, max_pages: int,
                 track: bool = False, device: int = 0, tree: int = 0):
        self._lib, self._err, self.device = backend.lib, backend._err, device
        self.dtype, self.batch, self.heads, self.kv_heads, self.head_dim = dtype, batch, heads, kv_heads, head_dim
        self.page_size, self.max_pages, self.track, self.capacity = page_size, max_pages, bool(track), page_size * max_pages
        self.handle = None
        free_unreferenced()
        config = PagedCacheConfig(ctypes.sizeof(PagedCacheConfig), dtype, int(bool(track)), batch, heads, kv_heads, head_dim, page_size,
                                  max_pages, tree)
        self.handle = self._lib.pjrtx_b200_paged_cache_create(device, ctypes.byref(config))
        if not self.handle:
            raise _error(self._err())
        self._stream = self._lib.pjrtx_b200_device_stream(device)
        self._page_dims = (page_size, kv_heads, head_dim)

    def _view(self, k_pages, v_pages, page_table, lengths, tokens, weights, positions) -> Tuple[int, bytes]:
        """The batch and the packed view."""
        try:  # tensors that are as they have to be, checked in one go; anything else takes the checks one by one
            kind, s32, here = _types[self.dtype], _types[P.S32], self.device
            dims, strides, (batch,) = k_pages.shape, k_pages.stride(), lengths.shape
            if (dims[1:] == self._page_dims and k_pages.dtype is kind and strides[3] == 1 and v_pages.shape == dims and v_pages.dtype is kind
                    and v_pages.stride() == strides and page_table.shape == (batch, self.max_pages) and page_table.dtype is s32
                    and page_table.is_contiguous() and lengths.dtype is s32 and lengths.is_contiguous() and k_pages.get_device() == here
                    and v_pages.get_device() == here and page_table.get_device() == here and lengths.get_device() == here):
                if weights is None and tokens is None and positions is None:
                    return batch, _pack_view(k_pages.data_ptr(), v_pages.data_ptr(), dims[0], strides[0], strides[1], strides[2],
                                             page_table.data_ptr(), self.max_pages, lengths.data_ptr(), batch, 0, 0, 0)
                tracked = (batch, self.kv_heads, self.capacity)
                return batch, _pack_view(k_pages.data_ptr(), v_pages.data_ptr(), dims[0], strides[0], strides[1], strides[2],
                                         page_table.data_ptr(), self.max_pages, lengths.data_ptr(), batch,
                                         _dense(tokens, "tokens", P.S32, (batch,), here), _dense(weights, "weights", P.F32, tracked, here),
                                         _dense(positions, "positions", P.S32, tracked, here))
        except (AttributeError, KeyError, ValueError, TypeError, IndexError):
            pass
        dims, batch_dims = _dims(k_pages), _dims(lengths)
        if len(dims) != 4 or dims[1:] != self._page_dims:
            raise _error(f"k_pages has shape {tuple(dims)}, (pages, {', '.join(map(str, self._page_dims))}) is needed")
        if len(batch_dims) != 1:
            raise _error(f"lengths has shape {tuple(batch_dims)}, (batch,) is needed")
        k, strides = _rows(k_pages, "k_pages", self.dtype, dims, self.device)
        v = _twin(v_pages, "v_pages", "k_pages", self.dtype, dims, strides, self.device)
        batch = batch_dims[0]
        table, table_strides = _rows(page_table, "page_table", P.S32, (batch, self.max_pages), self.device)
        tracked = (batch, self.kv_heads, self.capacity)
        return batch, _pack_view(k, v, dims[0], strides[0], strides[1], strides[2], table, table_strides[0],
                                 _dense(lengths, "lengths", P.S32, (batch,), self.device), batch,
                                 _dense(tokens, "tokens", P.S32, (batch,), self.device),
                                 _dense(weights, "weights", P.F32, tracked, self.device), _dense(positions, "positions", P.S32, tracked, self.device))

    def _call(self, fn, view, args, stream) -> None:
        if not self.handle:
            raise _error("the paged cache was destroyed")
        if not fn(self.handle, view, args, self._stream if stream is None else stream):
            raise _error(self._err())

    def _hand(self, fn, args, stream) -> None:
        """A call without a view."""
        if not self.handle:
            raise _error("the paged cache was destroyed")
        if not fn(self.handle, args, self._stream if stream is None else stream):
            raise _error(self._err())

    def append(self, k_pages, v_pages, page_table, lengths, k_new, v_new, counts=None, tokens=None, weights=None, positions=None,
               stream: Optional[int] = None) -> None:
        """Stores the first counts[b] of the rows k_new / v_new [batch, rows, kv_heads, head_dim] (None: all of them) as the
        last ones of the lengths[b] rows of each sequence; with tracking their weights become 0."""
        batch, view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        shape = _dims(k_new)
        if len(shape) != 4 or shape[0] != batch or shape[2] != self.kv_heads or shape[3] != self.head_dim:
            raise _error(f"k_new has shape {tuple(shape)}, ({batch}, rows, {self.kv_heads}, {self.head_dim}) is needed")
        k, strides = _rows(k_new, "k_new", self.dtype, shape, self.device)
        v = _twin(v_new, "v_new", "k_new", self.dtype, shape, strides, self.device)
        args = _pack_append(k, v, shape[1], strides[0], strides[1], strides[2], _dense(counts, "counts", P.S32, (batch,), self.device))
        self._call(self._lib.pjrtx_b200_paged_cache_append, view, args, stream)

    def attend(self, q, k_pages, v_pages, page_table, lengths, out, lse=None, k_new=None, v_new=None, tokens=None, weights=None,
               positions=None, scale: Optional[float] = None, stream: Optional[int] = None) -> None:
        """out [batch, heads, head_dim] = softmax(scale * q . k) v over each sequence's rows (`scale` None: 1 / sqrt(head_dim)),
        lse [batch, heads] its log-sum-exp. k_new / v_new [batch, kv_heads, head_dim] become row lengths[b] - 1 first. With
        tracking, weights[b, g, t] grows by what the query heads of KV head g give row t."""
        batch, view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        scale = self.head_dim ** -0.5 if scale is None else scale
        fn, stream = self._lib.pjrtx_b200_paged_cache_attend, self._stream if stream is None else stream
        shape, new_shape = (batch, self.heads, self.head_dim), (batch, self.kv_heads, self.head_dim)
        try:  # tensors that are as they have to be, as in _view
            kind, qs, os, here = _types[self.dtype], q.stride(), out.stride(), self.device
            if (q.shape == shape and q.dtype is kind and qs[2] == 1 and out.shape == shape and out.dtype is kind and os[2] == 1
                    and q.get_device() == here and out.get_device() == here
                    and (lse is None or lse.shape == shape[:2] and lse.dtype is _types[P.F32] and lse.is_contiguous() and lse.get_device() == here)):
                if k_new is None and v_new is None:
                    return self._call(fn, view, _pack_attend(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
                                                             0 if lse is None else lse.data_ptr(), 0, 0, 0, 0, scale), stream)
                ns = k_new.stride()
                if (k_new.shape == new_shape and k_new.dtype is kind and ns[2] == 1 and v_new.shape == new_shape and v_new.dtype is kind
                        and v_new.stride() == ns and k_new.get_device() == here and v_new.get_device() == here):
                    return self._call(fn, view, _pack_attend(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
                                                             0 if lse is None else lse.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), ns[0],
                                                             ns[1], scale), stream)
        except (AttributeError, KeyError, IndexError):
            pass
        q_at, q_strides = _rows(q, "q", self.dtype, shape, self.device)
        out_at, out_strides = _rows(out, "out", self.dtype, shape, self.device)
        k = v = 0
        new_strides = (0, 0)
        if k_new is not None and v_new is not None:
            k, new_strides = _rows(k_new, "k_new", self.dtype, new_shape, self.device)
            v = _twin(v_new, "v_new", "k_new", self.dtype, new_shape, new_strides, self.device)
        elif k_new is not None or v_new is not None:
            raise _error("a new key and a new value go together")
        args = _pack_attend(q_at, q_strides[0], q_strides[1], out_at, out_strides[0], out_strides[1],
                            _dense(lse, "lse", P.F32, (batch, self.heads), self.device), k, v, new_strides[0], new_strides[1], scale)
        return self._call(fn, view, args, stream)

    def attend_tree(self, q, k_pages, v_pages, page_table, lengths, out, k_new, v_new, parents, counts=None, lse=None,
                    scale: Optional[float] = None, stream: Optional[int] = None) -> None:
        """out [batch, nodes, heads, head_dim] = softmax(scale * q . k) v for a tree of drafted tokens per sequence: node i sees the
        lengths[b] cached rows, its ancestors by parents [batch, nodes] (a node before i, -1: a root) and itself, whose keys and
        values are k_new / v_new [batch, nodes, kv_heads, head_dim]. counts [batch]: nodes of each sequence (None: all), results
        behind them stay. lse [batch, nodes, heads]: log-sum-exp. Stores nothing and tracks no weights; a chain is a further piece of
        a prompt."""
        batch, view = self._view(k_pages, v_pages, page_table, lengths, None, None, None)
        dims = _dims(parents)
        if len(dims) != 2 or dims[0] != batch:
            raise _error(f"parents has shape {tuple(dims)}, ({batch}, nodes) is needed")
        nodes = dims[1]
        shape, new_shape = (batch, nodes, self.heads, self.head_dim), (batch, nodes, self.kv_heads, self.head_dim)
        q_at, qs = _rows(q, "q", self.dtype, shape, self.device)
        out_at, os = _rows(out, "out", self.dtype, shape, self.device)
        k, ns = _rows(k_new, "k_new", self.dtype, new_shape, self.device)
        v = _twin(v_new, "v_new", "k_new", self.dtype, new_shape, ns, self.device)
        args = _pack_tree(q_at, qs[0], qs[1], qs[2], out_at, os[0], os[1], os[2], _dense(lse, "lse", P.F32, shape[:3], self.device), k, v, ns[0],
                          ns[1], ns[2], _dense(parents, "parents", P.S32, dims, self.device), _dense(counts, "counts", P.S32, (batch,), self.device),
                          nodes, self.head_dim ** -0.5 if scale is None else scale)
        self._call(self._lib.pjrtx_b200_paged_cache_attend_tree, view, args, stream)

    def store(self, k_pages, v_pages, k_new, v_new, slots, stream: Optional[int] = None) -> None:
        """Stores rows k_new / v_new [rows, kv_heads, head_dim] at slots [rows] of the pools: a page times the page size plus a row in
        it, negative: nowhere. A slot must not come twice."""
        dims, shape = _dims(k_pages), _dims(k_new)
        if len(dims) != 4 or dims[1:] != self._page_dims:
            raise _error(f"k_pages has shape {tuple(dims)}, (pages, {', '.join(map(str, self._page_dims))}) is needed")
        if len(shape) != 3 or shape[1:] != self._page_dims[1:]:
            raise _error(f"k_new has shape {tuple(shape)}, (rows, {self.kv_heads}, {self.head_dim}) is needed")
        k_at, strides = _rows(k_pages, "k_pages", self.dtype, dims, self.device)
        v_at = _twin(v_pages, "v_pages", "k_pages", self.dtype, dims, strides, self.device)
        k, ns = _rows(k_new, "k_new", self.dtype, shape, self.device)
        v = _twin(v_new, "v_new", "k_new", self.dtype, shape, ns, self.device)
        view = _pack_view(k_at, v_at, dims[0], strides[0], strides[1], strides[2], 0, 0, 0, 0, 0, 0, 0)
        args = _pack_store(k, v, shape[0], ns[0], ns[1], _dense(slots, "slots", P.S32, shape[:1], self.device))
        self._call(self._lib.pjrtx_b200_paged_cache_store, view, args, stream)

    def assign_pages(self, lengths, held, page_table, free_pages, free_count, starts=None, slots=None, held_out=None, page_table_out=None,
                     free_pages_out=None, free_count_out=None, stream: Optional[int] = None) -> None:
        """Pages for lengths[b] rows of every sequence: those beyond them go back onto the stack of free_count[0] page ids in free_pages
        [pages of the pool], what sequences lack comes from its top, in order; the first that wants more than is left, and those
        behind it that want any, keep what they have. held [batch] counts pages. Results go to the `*_out` arrays, None: in place.
        slots [tokens] gets the slots of packed new tokens, those of sequence b from starts[b] to starts[b + 1] being its last rows;
        -1 where there is no page."""
        shape = _dims(lengths)
        if len(shape) != 1:
            raise _error(f"lengths has shape {tuple(shape)}, (batch,) is needed")
        pool, tokens = _dims(free_pages), () if slots is None else _dims(slots)
        if len(pool) != 1 or len(tokens) > 1:
            raise _error(f"{'free_pages' if len(pool) != 1 else 'slots'} has shape {tuple(pool if len(pool) != 1 else tokens)}, one axis is needed")
        here, tables = self.device, shape + (self.max_pages,)
        table, strides = _rows(page_table, "page_table", P.S32, tables, here)
        table_out, out_strides = (table, strides) if page_table_out is None else _rows(page_table_out, "page_table_out", P.S32, tables, here)
        args = _pack_assign(
            shape[0], _dense(lengths, "lengths", P.S32, shape, here), _dense(held, "held", P.S32, shape, here), table, strides[0],
            _dense(free_pages, "free_pages", P.S32, pool, here), _dense(free_count, "free_count", P.S32, (1,), here), pool[0],
            _dense(held if held_out is None else held_out, "held_out", P.S32, shape, here), table_out, out_strides[0],
            _dense(free_pages if free_pages_out is None else free_pages_out, "free_pages_out", P.S32, pool, here),
            _dense(free_count if free_count_out is None else free_count_out, "free_count_out", P.S32, (1,), here),
            _dense(starts, "starts", P.S32, (shape[0] + 1,), here), _dense(slots, "slots", P.S32, tokens, here), tokens[0] if tokens else 0)
        self._hand(self._lib.pjrtx_b200_paged_cache_assign, args, stream)

    def path_slots(self, page_table, lengths, parents, leaves, slots, lengths_out=None, stream: Optional[int] = None) -> None:
        """slots [batch, nodes] of the nodes on the way from leaves[b] to its root, as rows lengths[b], lengths[b] + 1, ... of each
        sequence; -1 for the others, and for all where the leaf is negative. lengths_out (None: in place) counts them."""
        dims = _dims(parents)
        if len(dims) != 2:
            raise _error(f"parents has shape {tuple(dims)}, (batch, nodes) is needed")
        here, batch = self.device, dims[:1]
        table, strides = _rows(page_table, "page_table", P.S32, batch + (self.max_pages,), here)
        args = _pack_path(batch[0], dims[1], table, strides[0], _dense(lengths, "lengths", P.S32, batch, here),
                          _dense(parents, "parents", P.S32, dims, here), _dense(leaves, "leaves", P.S32, batch, here),
                          _dense(slots, "slots", P.S32, dims, here),
                          _dense(lengths if lengths_out is None else lengths_out, "lengths_out", P.S32, batch, here))
        self._hand(self._lib.pjrtx_b200_paged_cache_path_slots, args, stream)

    def evict(self, k_pages, v_pages, page_table, lengths, tokens, weights, positions, keep: int, recent: int = 0, sinks: int = 0,
              lengths_out=None, weights_out=None, positions_out=None, stream: Optional[int] = None) -> None:
        """Cuts every sequence to `keep` rows by weight; tokens before `sinks` and the last `recent` ones stay. Results go to the
        `*_out` arrays, None: in place. Layers that share `lengths` need another array as `lengths_out`. Pages must not be shared
        between sequences."""
        batch, view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        tracked = (batch, self.kv_heads, self.capacity)
        args = _pack_evict(keep, recent, sinks, _dense(lengths if lengths_out is None else lengths_out, "lengths_out", P.S32, (batch,), self.device),
                           _dense(weights if weights_out is None else weights_out, "weights_out", P.F32, tracked, self.device),
                           _dense(positions if positions_out is None else positions_out, "positions_out", P.S32, tracked, self.device))
        self._call(self._lib.pjrtx_b200_paged_cache_evict, view, args, stream)

    def destroy(self) -> None:
        free_unreferenced()
        if self.handle:
            self._lib.pjrtx_b200_paged_cache_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self.handle:
                _unreferenced.append((self._lib, self.handle))
        except Exception:  # a half-made cache, or the interpreter's end
            pass


def prompt_attention(backend, q, k, v, starts, out, lse=None, scale: Optional[float] = None, stream: Optional[int] = None,
                     device: int = 0) -> None:
    shape, new_shape, code = _dims(q), _dims(k), _code(q)
    if code not in _FLOATS:
        raise _error(f"q has element type {P.DTYPE_NAMES.get(code, 'other')}; f32, f16 and bf16 are supported")
    if len(shape) != 3:
        raise _error(f"q has shape {tuple(shape)}, (tokens, heads, head_dim) is needed")
    if len(new_shape) != 3 or new_shape[0] != shape[0] or new_shape[2] != shape[2]:
        raise _error(f"k has shape {tuple(new_shape)}, ({shape[0]}, KV heads, {shape[2]}) is needed")
    ends = _dims(starts)
    if len(ends) != 1 or ends[0] < 1:
        raise _error(f"starts has shape {tuple(ends)}, (sequences + 1,) is needed")
    q_at, qs = _rows(q, "q", code, shape, device)
    k_at, ks = _rows(k, "k", code, new_shape, device)
    v_at, vs = _rows(v, "v", code, new_shape, device)
    out_at, os = _rows(out, "out", code, shape, device)
    args = _pack_prompt(code, shape[2] ** -0.5 if scale is None else scale, q_at, k_at, v_at, out_at, _dense(lse, "lse", P.F32, shape[:2], device),
                        shape[0], shape[1], new_shape[1], shape[2], qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
                        _dense(starts, "starts", P.S32, ends, device), ends[0] - 1)
    lib = backend.lib
    if not lib.pjrtx_b200_prompt_attention(device, args, lib.pjrtx_b200_device_stream(device) if stream is None else stream):
        raise _error(backend._err())


def _logits(x, device: int):
    """Element type, rows, vocabulary, address and row stride."""
    try:
        (rows, vocab), code, strides = x.shape, _codes[x.dtype], x.stride()
        if code in _FLOATS and strides[1] == 1 and x.get_device() == device:
            return code, rows, vocab, x.data_ptr(), strides[0]
    except (AttributeError, KeyError, ValueError):
        pass
    dims, code = _dims(x), _code(x)
    if len(dims) != 2:
        raise _error(f"logits has shape {tuple(dims)}, (rows, vocabulary) is needed")
    if code not in _FLOATS:
        raise _error(f"logits has element type {P.DTYPE_NAMES.get(code, 'other')}; f32, f16 and bf16 are supported")
    pointer, strides = _rows(x, "logits", code, dims, device)
    return code, dims[0], dims[1], pointer, strides[0]


def token_log_probs(backend, logits, tokens, log_probs, entropy=None, lse=None, top_ids=None, top_log_probs=None, scale: float = 1.0,
                    stream: Optional[int] = None, device: int = 0) -> None:
    dtype, rows, vocab, at, stride = _logits(logits, device)
    wide = top_ids if top_ids is not None else top_log_probs
    top = 0 if wide is None else _dims(wide)[-1]
    args = _pack_score(dtype, top, at, rows, vocab, stride, _dense(tokens, "tokens", P.S32, (rows,), device), scale,
                       _dense(log_probs, "log_probs", P.F32, (rows,), device), _dense(entropy, "entropy", P.F32, (rows,), device),
                       _dense(lse, "lse", P.F32, (rows,), device), _dense(top_ids, "top_ids", P.S32, (rows, top), device),
                       _dense(top_log_probs, "top_log_probs", P.F32, (rows, top), device))
    lib = backend.lib
    if not lib.pjrtx_b200_token_log_probs(device, args, lib.pjrtx_b200_device_stream(device) if stream is None else stream):
        raise _error(backend._err())


def token_log_probs_backward(backend, logits, tokens, lse, grad_logits, grad_log_probs=None, entropy=None, grad_entropy=None,
                             scale: float = 1.0, stream: Optional[int] = None, device: int = 0) -> None:
    dtype, rows, vocab, at, stride = _logits(logits, device)
    grad_at, grad_strides = _rows(grad_logits, "grad_logits", dtype, (rows, vocab), device)
    args = _pack_score_grad(dtype, scale, at, grad_at, rows, vocab, stride, grad_strides[0], _dense(tokens, "tokens", P.S32, (rows,), device),
                            _dense(lse, "lse", P.F32, (rows,), device), _dense(entropy, "entropy", P.F32, (rows,), device),
                            _dense(grad_log_probs, "grad_log_probs", P.F32, (rows,), device),
                            _dense(grad_entropy, "grad_entropy", P.F32, (rows,), device))
    lib = backend.lib
    if not lib.pjrtx_b200_token_log_probs_backward(device, args, lib.pjrtx_b200_device_stream(device) if stream is None else stream):
        raise _error(backend._err())
