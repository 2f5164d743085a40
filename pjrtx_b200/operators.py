"""Operators on device memory: a paged key-value cache and the scoring of a decoder's logits.

Bindings of the `pjrtx_b200_paged_cache_*` and `pjrtx_b200_token_log_probs*` entry points of include/pjrtx_b200.h, reached
through `Backend.paged_cache`, `Backend.token_log_probs` and `Backend.token_log_probs_backward`. Arrays are `DeviceBuffer`s
or any device tensors with `data_ptr()`, `shape`, `stride()` and `dtype` (torch's). Types and shapes are checked here, the
rest behind the C ABI; nothing is copied, cast or kept. Calls enqueue on `stream`, a `cudaStream_t` as an integer (0: the
default stream); None is the stream on which the backend's buffers and executables work.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

from . import plan as P

_P, _I32, _I64, _U64, _F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float


class PagedCacheConfig(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("track", _I32), ("batch", _I64), ("heads", _I64), ("kv_heads", _I64),
                ("head_dim", _I64), ("page_size", _I64), ("max_pages", _I64)]


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


class TokenLogProbsArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("top", _I32), ("logits", _P), ("rows", _I64), ("vocab", _I64),
                ("row_stride", _I64), ("tokens", _P), ("scale", _F32), ("log_probs", _P), ("entropy", _P), ("lse", _P),
                ("top_ids", _P), ("top_log_probs", _P)]


class TokenLogProbsBackwardArgs(ctypes.Structure):
    _fields_ = [("struct_size", _U64), ("dtype", _I32), ("scale", _F32), ("logits", _P), ("grad_logits", _P), ("rows", _I64),
                ("vocab", _I64), ("row_stride", _I64), ("grad_row_stride", _I64), ("tokens", _P), ("lse", _P), ("entropy", _P),
                ("grad_log_probs", _P), ("grad_entropy", _P)]


# Every symbol of the operator section of include/pjrtx_b200.h: name -> (restype, argtypes).
_CACHE_CALL = [_P, ctypes.POINTER(PagedView)]
SYMBOLS = {
    "pjrtx_b200_device_stream": (_P, [ctypes.c_int]),
    "pjrtx_b200_buffer_device_pointer": (_P, [_P]),
    "pjrtx_b200_paged_cache_create": (_P, [ctypes.c_int, ctypes.POINTER(PagedCacheConfig)]),
    "pjrtx_b200_paged_cache_destroy": (None, [_P]),
    "pjrtx_b200_paged_cache_append": (ctypes.c_int, _CACHE_CALL + [ctypes.POINTER(PagedAppendArgs), _P]),
    "pjrtx_b200_paged_cache_attend": (ctypes.c_int, _CACHE_CALL + [ctypes.POINTER(PagedAttendArgs), _P]),
    "pjrtx_b200_paged_cache_evict": (ctypes.c_int, _CACHE_CALL + [ctypes.POINTER(PagedEvictArgs), _P]),
    "pjrtx_b200_token_log_probs": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(TokenLogProbsArgs), _P]),
    "pjrtx_b200_token_log_probs_backward": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(TokenLogProbsBackwardArgs), _P]),
}

_TENSOR_TYPES = {"float32": P.F32, "float16": P.F16, "bfloat16": P.BF16_CODE, "int32": P.S32}
_codes: dict = {}  # a tensor library's dtype object -> element-type code


def _error(message: str):
    from .backend import BackendError

    return BackendError("InvalidArgument", message)


def _code(dtype) -> Optional[int]:
    code = _codes.get(dtype)
    if code is None:
        code = _TENSOR_TYPES.get(str(dtype).split(".")[-1])
        if code is not None:
            _codes[dtype] = code
    return code


def _array(x, name: str, dtype: int, shape: Sequence[int]) -> Tuple[Optional[int], Tuple[int, ...]]:
    """Device address and strides (elements) of an array that must have this type and shape (-1: any extent)."""
    if hasattr(x, "data_ptr"):
        code, dims, strides, pointer = _code(x.dtype), x.shape, x.stride(), x.data_ptr()
    else:
        code, dims, strides, pointer = x.dtype, x.dims, None, x.device_pointer
    if code != dtype:
        raise _error(f"{name} has element type {P.DTYPE_NAMES.get(code, 'other')}, {P.DTYPE_NAMES.get(dtype, dtype)} is needed")
    if tuple(dims) != shape and (len(dims) != len(shape) or any(want not in (-1, have) for have, want in zip(dims, shape))):
        raise _error(f"{name} has shape {tuple(dims)}, {tuple(shape)} is needed")
    if strides is None:
        strides, step = [], 1
        for d in reversed(dims):
            strides.insert(0, step)
            step *= d
    return pointer, strides


def _rows(x, name: str, dtype: int, shape: Sequence[int]):
    """The same for an array whose innermost axis has to be dense."""
    pointer, strides = _array(x, name, dtype, shape)
    if strides[-1] != 1 and shape[-1] != 1:
        raise _error(f"{name} has stride {strides[-1]} along its last axis, which has to be dense")
    return pointer, strides


def _dense(x, name: str, dtype: int, shape: Sequence[int]):
    """Address of an array that has to be dense; None stays None."""
    if x is None:
        return None
    pointer, strides = _array(x, name, dtype, shape)
    step = 1
    for d, s in zip(reversed(shape), reversed(strides)):
        if s != step and d != 1:
            raise _error(f"{name} has to be dense, its strides are {tuple(strides)}")
        step *= d
    return pointer


class PagedCache:
    """Geometry and workspaces of a paged key-value cache: one handle serves all layers of a shape, on one stream at a time.

    Pools are [pages, page_size, kv_heads, head_dim] in any layout that keeps the last axis dense and rows 16-byte aligned,
    the same for keys and values. Row t of sequence b is row t % page_size of page page_table[b, t // page_size]; `lengths[b]`
    counts the rows of a sequence, those that a call appends among them. With `track`, weights and positions are
    [batch, kv_heads, max_pages * page_size], and `tokens[b]` counts the tokens a sequence has seen.
    """

    def __init__(self, backend, dtype: int, batch: int, heads: int, kv_heads: int, head_dim: int, page_size: int, max_pages: int,
                 track: bool = False, device: int = 0):
        self._lib, self._err, self.device = backend.lib, backend._err, device
        self.dtype, self.batch, self.heads, self.kv_heads, self.head_dim = dtype, batch, heads, kv_heads, head_dim
        self.page_size, self.max_pages, self.track, self.capacity = page_size, max_pages, bool(track), page_size * max_pages
        self.handle = None
        config = PagedCacheConfig(ctypes.sizeof(PagedCacheConfig), dtype, int(bool(track)), batch, heads, kv_heads, head_dim, page_size, max_pages)
        self.handle = self._lib.pjrtx_b200_paged_cache_create(device, ctypes.byref(config))
        if not self.handle:
            raise _error(self._err())
        self._stream = self._lib.pjrtx_b200_device_stream(device)

    def _view(self, k_pages, v_pages, page_table, lengths, tokens=None, weights=None, positions=None) -> PagedView:
        dims = (-1, self.page_size, self.kv_heads, self.head_dim)
        k, strides = _rows(k_pages, "k_pages", self.dtype, dims)
        v, v_strides = _rows(v_pages, "v_pages", self.dtype, dims)
        shape = k_pages.shape if hasattr(k_pages, "shape") else k_pages.dims
        v_shape = v_pages.shape if hasattr(v_pages, "shape") else v_pages.dims
        if shape[0] != v_shape[0] or tuple(strides) != tuple(v_strides):
            raise _error("k_pages and v_pages differ in their number of pages or in their strides")
        batch = (lengths.shape if hasattr(lengths, "shape") else lengths.dims)[0]
        table, table_strides = _rows(page_table, "page_table", P.S32, (batch, self.max_pages))
        tracked = (batch, self.kv_heads, self.capacity)
        return PagedView(ctypes.sizeof(PagedView), k, v, shape[0], strides[0], strides[1], strides[2], table, table_strides[0],
                         _dense(lengths, "lengths", P.S32, (batch,)), batch, _dense(tokens, "tokens", P.S32, (batch,)),
                         _dense(weights, "weights", P.F32, tracked), _dense(positions, "positions", P.S32, tracked))

    def _call(self, fn, view, args, stream) -> None:
        if not self.handle:
            raise _error("the paged cache was destroyed")
        if not fn(self.handle, ctypes.byref(view), ctypes.byref(args), self._stream if stream is None else stream):
            raise _error(self._err())

    def append(self, k_pages, v_pages, page_table, lengths, k_new, v_new, counts=None, tokens=None, weights=None, positions=None,
               stream: Optional[int] = None) -> None:
        """Stores the first counts[b] of the rows k_new / v_new [batch, rows, kv_heads, head_dim] (None: all of them) as the
        last ones of the lengths[b] rows of each sequence; with tracking their weights become 0."""
        view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        shape = (view.batch, -1, self.kv_heads, self.head_dim)
        k, strides = _rows(k_new, "k_new", self.dtype, shape)
        v, v_strides = _rows(v_new, "v_new", self.dtype, shape)
        rows, v_rows = ((x.shape if hasattr(x, "shape") else x.dims)[1] for x in (k_new, v_new))
        if rows != v_rows or tuple(strides) != tuple(v_strides):
            raise _error("k_new and v_new differ in their number of rows or in their strides")
        args = PagedAppendArgs(ctypes.sizeof(PagedAppendArgs), k, v, rows, strides[0], strides[1], strides[2],
                               _dense(counts, "counts", P.S32, (view.batch,)))
        self._call(self._lib.pjrtx_b200_paged_cache_append, view, args, stream)

    def attend(self, q, k_pages, v_pages, page_table, lengths, out, lse=None, k_new=None, v_new=None, tokens=None, weights=None,
               positions=None, scale: Optional[float] = None, stream: Optional[int] = None) -> None:
        """out [batch, heads, head_dim] = softmax(scale * q . k) v over each sequence's rows (`scale` None: 1 / sqrt(head_dim)),
        lse [batch, heads] its log-sum-exp. k_new / v_new [batch, kv_heads, head_dim] become row lengths[b] - 1 first. With
        tracking, weights[b, g, t] grows by what the query heads of KV head g give row t."""
        view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        batch, shape = view.batch, (view.batch, self.heads, self.head_dim)
        q_at, q_strides = _rows(q, "q", self.dtype, shape)
        out_at, out_strides = _rows(out, "out", self.dtype, shape)
        k = v = None
        new_strides = (0, 0)
        if k_new is not None and v_new is not None:
            k, new_strides = _rows(k_new, "k_new", self.dtype, (batch, self.kv_heads, self.head_dim))
            v, v_strides = _rows(v_new, "v_new", self.dtype, (batch, self.kv_heads, self.head_dim))
            if tuple(new_strides) != tuple(v_strides):
                raise _error("k_new and v_new differ in their strides")
        elif k_new is not None or v_new is not None:
            raise _error("a new key and a new value go together")
        args = PagedAttendArgs(ctypes.sizeof(PagedAttendArgs), q_at, q_strides[0], q_strides[1], out_at, out_strides[0], out_strides[1],
                               _dense(lse, "lse", P.F32, (batch, self.heads)), k, v, new_strides[0], new_strides[1],
                               1.0 / math.sqrt(self.head_dim) if scale is None else scale)
        self._call(self._lib.pjrtx_b200_paged_cache_attend, view, args, stream)

    def evict(self, k_pages, v_pages, page_table, lengths, tokens, weights, positions, keep: int, recent: int = 0, sinks: int = 0,
              lengths_out=None, weights_out=None, positions_out=None, stream: Optional[int] = None) -> None:
        """Cuts every sequence to `keep` rows by weight; tokens before `sinks` and the last `recent` ones stay. Results go to the
        `*_out` arrays, None: in place. Pages must not be shared between sequences."""
        view = self._view(k_pages, v_pages, page_table, lengths, tokens, weights, positions)
        tracked = (view.batch, self.kv_heads, self.capacity)
        args = PagedEvictArgs(ctypes.sizeof(PagedEvictArgs), keep, recent, sinks,
                              _dense(lengths if lengths_out is None else lengths_out, "lengths_out", P.S32, (view.batch,)),
                              _dense(weights if weights_out is None else weights_out, "weights_out", P.F32, tracked),
                              _dense(positions if positions_out is None else positions_out, "positions_out", P.S32, tracked))
        self._call(self._lib.pjrtx_b200_paged_cache_evict, view, args, stream)

    def destroy(self) -> None:
        if self.handle:
            self._lib.pjrtx_b200_paged_cache_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def _logits(x, name: str):
    dims = x.shape if hasattr(x, "data_ptr") else x.dims
    if len(dims) != 2:
        raise _error(f"{name} has shape {tuple(dims)}, (rows, vocabulary) is needed")
    code = _code(x.dtype) if hasattr(x, "data_ptr") else x.dtype
    if code not in (P.F32, P.F16, P.BF16_CODE):
        raise _error(f"{name} has element type {P.DTYPE_NAMES.get(code, 'other')}; f32, f16 and bf16 are supported")
    pointer, strides = _rows(x, name, code, dims)
    return code, dims[0], dims[1], pointer, strides[0]


def token_log_probs(backend, logits, tokens, log_probs, entropy=None, lse=None, top_ids=None, top_log_probs=None, scale: float = 1.0,
                    stream: Optional[int] = None, device: int = 0) -> None:
    dtype, rows, vocab, at, stride = _logits(logits, "logits")
    top = 0
    for x in (top_ids, top_log_probs):
        if x is not None:
            top = (x.shape if hasattr(x, "shape") else x.dims)[-1]
    args = TokenLogProbsArgs(ctypes.sizeof(TokenLogProbsArgs), dtype, top, at, rows, vocab, stride, _dense(tokens, "tokens", P.S32, (rows,)), scale,
                             _dense(log_probs, "log_probs", P.F32, (rows,)), _dense(entropy, "entropy", P.F32, (rows,)),
                             _dense(lse, "lse", P.F32, (rows,)), _dense(top_ids, "top_ids", P.S32, (rows, top)),
                             _dense(top_log_probs, "top_log_probs", P.F32, (rows, top)))
    if not backend.lib.pjrtx_b200_token_log_probs(device, ctypes.byref(args), _stream_of(backend, device, stream)):
        raise _error(backend._err())


def token_log_probs_backward(backend, logits, tokens, lse, grad_logits, grad_log_probs=None, entropy=None, grad_entropy=None,
                             scale: float = 1.0, stream: Optional[int] = None, device: int = 0) -> None:
    dtype, rows, vocab, at, stride = _logits(logits, "logits")
    grad_at, grad_strides = _rows(grad_logits, "grad_logits", dtype, (rows, vocab))
    args = TokenLogProbsBackwardArgs(ctypes.sizeof(TokenLogProbsBackwardArgs), dtype, scale, at, grad_at, rows, vocab, stride, grad_strides[0],
                                     _dense(tokens, "tokens", P.S32, (rows,)), _dense(lse, "lse", P.F32, (rows,)),
                                     _dense(entropy, "entropy", P.F32, (rows,)), _dense(grad_log_probs, "grad_log_probs", P.F32, (rows,)),
                                     _dense(grad_entropy, "grad_entropy", P.F32, (rows,)))
    if not backend.lib.pjrtx_b200_token_log_probs_backward(device, ctypes.byref(args), _stream_of(backend, device, stream)):
        raise _error(backend._err())


def _stream_of(backend, device: int, stream: Optional[int]):
    return backend.lib.pjrtx_b200_device_stream(device) if stream is None else stream
