"""Operators on device memory against plain 64-bit forms: a paged key-value cache (append, attend, evict) and the scoring of
logits (log probabilities, entropy, likeliest tokens, gradient).

Tolerances follow from the arithmetic: a score is a sum of head_dim products in f32, so it is off by at most
(head_dim + 16) * 2^-24 * sum |q k| * scale; a probability by that factor twice (numerator and denominator) and 2^-17 for the
exponential and what a split of it into two 16-bit numbers leaves; the result is rounded once to its type.
"""
import ctypes
import gc
import math

import numpy as np
import pytest

from pjrtx_b200 import backend as be_mod
from pjrtx_b200 import operators as ops
from pjrtx_b200 import plan as P

CODE = {"f32": P.F32, "f16": P.F16, "bf16": P.BF16_CODE}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8.0 / 2}
FLOOR = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}  # half the spacing of subnormal numbers


def _torch_type(dtype):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def _stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def _within(got, want, bound, what):
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu() if hasattr(bound, "double") else bound
    same = (got == want) | (got.isnan() & want.isnan())
    ok = same | ((got - want).abs() <= bound)
    assert bool(ok.all()), (what, int((~ok).sum()), float((got - want).abs()[~ok].max()), got[~ok][:4], want[~ok][:4])


# ---- refusals (no device needed) -----------------------------------------------------------------------------------


class _Array:
    """A dense device tensor as the facade sees one; nothing ever reads its address."""

    class _Type:
        def __init__(self, name):
            self.name = name

        def __str__(self):
            return self.name

    _types = {}

    def __init__(self, name, *shape, pointer=1 << 20, strides=None):
        self.dtype = _Array._types.setdefault(name, _Array._Type("fake." + name))
        self.shape, self._pointer = shape, pointer
        self._strides = strides or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def data_ptr(self):
        return self._pointer

    def stride(self):
        return self._strides


@pytest.mark.parametrize("change,message", [
    (dict(dtype=P.S32), "element type"), (dict(batch=0), "batch 0"), (dict(batch=70000), "batch 70000"), (dict(heads=6), "6 query heads"),
    (dict(kv_heads=0), "0 KV heads"), (dict(head_dim=0), "head dimension 0"), (dict(head_dim=100), "head dimension 100"),
    (dict(head_dim=264), "head dimension 264"), (dict(page_size=0), "pages of 0 rows"), (dict(max_pages=0), "0 pages"),
    (dict(page_size=1 << 20, max_pages=1 << 20), "rows a sequence")])
def test_paged_cache_refuses_bad_geometry(backend, change, message):
    shape = dict(dtype=P.BF16_CODE, batch=2, heads=8, kv_heads=4, head_dim=64, page_size=16, max_pages=4)
    shape.update(change)
    with pytest.raises(be_mod.BackendError, match=message):
        backend.paged_cache(**shape)


@pytest.mark.parametrize("batch,heads,page_size", [(65535, 65535, 1 << 30), (50000, 30000, 993763988), (1 << 10, 1 << 10, (1 << 20) + 1)])
def test_paged_cache_refuses_workspaces_beyond_any_memory(backend, batch, heads, page_size):
    """Sizes of a tracked cache whose workspace would not fit 64 bits must not become those of a small one."""
    with pytest.raises(be_mod.BackendError, match="too many for a workspace"):
        backend.paged_cache(P.BF16_CODE, batch, heads, heads, 8, page_size, 1, track=True)


def test_operator_structs_without_size_and_null_handles_are_refused(backend):
    lib = backend.lib
    config = ops.PagedCacheConfig(0, P.F32, 0, 1, 1, 1, 64, 16, 1)
    assert not lib.pjrtx_b200_paged_cache_create(0, ctypes.byref(config)) and b"struct_size" in lib.pjrtx_b200_last_error()
    assert not lib.pjrtx_b200_paged_cache_create(0, None) and b"null argument" in lib.pjrtx_b200_last_error()
    view = ops.PagedView(ctypes.sizeof(ops.PagedView))
    assert not lib.pjrtx_b200_paged_cache_evict(None, ctypes.byref(view), None, None) and b"null paged cache" in lib.pjrtx_b200_last_error()
    assert not lib.pjrtx_b200_token_log_probs(0, None, None)
    assert not lib.pjrtx_b200_token_log_probs_backward(0, ctypes.byref(ops.TokenLogProbsBackwardArgs(8)), None)
    lib.pjrtx_b200_paged_cache_destroy(None)
    assert not lib.pjrtx_b200_buffer_device_pointer(None)


def _score_args(**change):
    a = dict(logits=_Array("bfloat16", 4, 100), tokens=_Array("int32", 4), log_probs=_Array("float32", 4))
    a.update(change)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(logits=_Array("int32", 4, 100)), "element type s32"), (dict(logits=_Array("bfloat16", 4, 100, 2)), "shape"),
    (dict(logits=_Array("bfloat16", 4, 100, strides=(200, 2))), "dense"), (dict(tokens=_Array("int64", 4)), "tokens has element type"),
    (dict(tokens=_Array("int32", 3)), "tokens has shape"), (dict(log_probs=_Array("float32", 5)), "log_probs has shape"),
    (dict(log_probs=None), "null result"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"), (dict(top_ids=_Array("int32", 4, 65)), "65 alternatives"),
    (dict(logits=_Array("float32", 4, 3), top_ids=_Array("int32", 4, 5)), "5 alternatives"),
    (dict(top_ids=_Array("int32", 4, 5), top_log_probs=_Array("float32", 4, 6)), "shape"),
    (dict(logits=_Array("bfloat16", 4, 100, pointer=1 << 20 | 1)), "misaligned"), (dict(logits=_Array("bfloat16", 4, 100, pointer=0)), "null"),
    (dict(logits=_Array("bfloat16", 4, 100, strides=(50, 1))), "50 apart"),
    (dict(logits=_Array("bfloat16", 4, (1 << 22) + 1)), "rows of")])
def test_token_log_probs_refuses(backend, change, message):
    with pytest.raises(be_mod.BackendError, match=message):
        backend.token_log_probs(**_score_args(**change), stream=0)


@pytest.mark.parametrize("change,message", [
    (dict(grad_log_probs=None), "no incoming gradient"), (dict(entropy=None, grad_entropy=_Array("float32", 4)), "null log-sum-exp or entropy"),
    (dict(lse=None), "null log-sum-exp"), (dict(grad_logits=_Array("float32", 4, 100)), "grad_logits has element type"),
    (dict(grad_logits=_Array("bfloat16", 4, 100, strides=(50, 1))), "overlapping"),
    (dict(grad_logits=_Array("bfloat16", 4, 100, strides=(128, 1))), "in place"), (dict(scale=0.0), "scale")])
def test_token_log_probs_backward_refuses(backend, change, message):
    a = dict(logits=_Array("bfloat16", 4, 100), tokens=_Array("int32", 4), lse=_Array("float32", 4), grad_logits=_Array("bfloat16", 4, 100),
             grad_log_probs=_Array("float32", 4))
    a.update(change)
    with pytest.raises(be_mod.BackendError, match=message):
        backend.token_log_probs_backward(**a, stream=0)


class _Placed(_Array):
    """A device tensor that says where it is, as torch does (`get_device`) or by its `device`."""

    def __init__(self, where, like, says):
        super().__init__(like.dtype.name[5:], *like.shape)
        if says == "get_device":
            self.get_device = lambda: where
        else:
            self.device = type("Device", (), dict(type="cuda" if where >= 0 else "cpu", index=where if where >= 0 else None))()

    def is_contiguous(self):
        return True


def test_a_dropped_cache_is_freed_where_the_caller_waits(backend):
    freed = []

    class Library:
        @staticmethod
        def pjrtx_b200_paged_cache_destroy(handle):
            freed.append(handle)

    caches = [ops.PagedCache.__new__(ops.PagedCache) for _ in range(3)]
    for i, c in enumerate(caches):
        c._lib, c.handle = Library, 100 + i
    del c
    last = caches.pop()
    caches.clear()
    assert freed == []  # wherever the collector runs, a capture may be under way
    last.destroy()
    last.destroy()
    assert sorted(freed) == [100, 101, 102] and last.handle is None
    del last
    ops.free_unreferenced()
    assert len(freed) == 3


class _Unreachable:
    """In the place of the library: no call with a refused argument may get there."""

    def __getattr__(self, name):
        def reached(*_):
            raise AssertionError(f"{name} was reached")

        return reached


def _host_cache():
    """A paged cache without a device: what the facade checks, and a library that must not be reached."""
    cache = ops.PagedCache.__new__(ops.PagedCache)
    cache.dtype, cache.batch, cache.heads, cache.kv_heads, cache.head_dim = P.BF16_CODE, 2, 8, 4, 64
    cache.page_size, cache.max_pages, cache.track, cache.capacity, cache.device = 16, 4, True, 64, 1
    cache._page_dims, cache._stream, cache._lib, cache.handle = (16, 4, 64), 0, _Unreachable(), 0
    return cache


@pytest.mark.parametrize("says", ["get_device", "device"])
@pytest.mark.parametrize("where,message", [(-1, "on the host, device 1"), (0, "on device 0, device 1")])
def test_arrays_of_the_host_and_of_other_devices_are_refused(backend, where, message, says):
    def check(call, good):
        place = lambda at, a: _Placed(at, a, says)
        for name in good:
            if isinstance(good[name], _Array):
                with pytest.raises(be_mod.BackendError, match=f"{name} is {message}"):
                    call(**{n: place(where if n == name else 1, a) if isinstance(a, _Array) else a for n, a in good.items()}, stream=0)

    cache = _host_cache()
    view = dict(k_pages=_Array("bfloat16", 9, 16, 4, 64), v_pages=_Array("bfloat16", 9, 16, 4, 64), page_table=_Array("int32", 2, 4),
                lengths=_Array("int32", 2), tokens=_Array("int32", 2), weights=_Array("float32", 2, 4, 64), positions=_Array("int32", 2, 4, 64))
    check(cache.append, dict(view, k_new=_Array("bfloat16", 2, 3, 4, 64), v_new=_Array("bfloat16", 2, 3, 4, 64), counts=_Array("int32", 2)))
    check(cache.attend, dict(view, q=_Array("bfloat16", 2, 8, 64), out=_Array("bfloat16", 2, 8, 64), lse=_Array("float32", 2, 8),
                             k_new=_Array("bfloat16", 2, 4, 64), v_new=_Array("bfloat16", 2, 4, 64)))
    check(cache.evict, dict(view, keep=8, lengths_out=_Array("int32", 2), weights_out=_Array("float32", 2, 4, 64),
                            positions_out=_Array("int32", 2, 4, 64)))
    row = _Array("float32", 4)
    scored = dict(logits=_Array("float16", 4, 100), tokens=_Array("int32", 4), entropy=row, lse=row, device=1)
    check(backend.token_log_probs, dict(scored, log_probs=row, top_ids=_Array("int32", 4, 3), top_log_probs=_Array("float32", 4, 3)))
    check(backend.token_log_probs_backward, dict(scored, grad_logits=_Array("float16", 4, 100), grad_log_probs=row, grad_entropy=row))


def test_tensors_in_host_memory_are_refused(backend):
    import torch

    cache = _host_cache()
    view = dict(k_pages=torch.zeros(9, 16, 4, 64).bfloat16(), v_pages=torch.zeros(9, 16, 4, 64).bfloat16(),
                page_table=torch.zeros(2, 4, dtype=torch.int32), lengths=torch.zeros(2, dtype=torch.int32))
    q = torch.zeros(2, 8, 64).bfloat16()
    for _ in range(2):  # types are known after the first call
        with pytest.raises(be_mod.BackendError, match="k_pages is on the host"):
            cache.attend(q, **view, out=torch.zeros_like(q), stream=0)
        with pytest.raises(be_mod.BackendError, match="logits is on the host"):
            backend.token_log_probs(torch.zeros(4, 100), torch.zeros(4, dtype=torch.int32), torch.zeros(4), stream=0)


@pytest.mark.gpu
def test_paged_cache_calls_refuse_bad_arguments(gpu_backend):
    """Everything here is refused on the host: the addresses are never used."""
    cache = gpu_backend.paged_cache(P.BF16_CODE, 2, 8, 4, 64, 16, 4, track=True)
    plain = gpu_backend.paged_cache(P.BF16_CODE, 2, 8, 4, 64, 16, 4)

    def base(batch=2):
        return dict(k_pages=_Array("bfloat16", 9, 16, 4, 64), v_pages=_Array("bfloat16", 9, 16, 4, 64), page_table=_Array("int32", batch, 4),
                    lengths=_Array("int32", batch))

    def refused(call, message, *changes, **arguments):
        for change in changes:
            arguments.update(change)
        with pytest.raises(be_mod.BackendError, match=message):
            call(**arguments, stream=0)

    q, out = _Array("bfloat16", 2, 8, 64), _Array("bfloat16", 2, 8, 64)
    attend = dict(base(), q=q, out=out)
    refused(cache.attend, "k_pages has shape", attend, dict(k_pages=_Array("bfloat16", 9, 8, 4, 64)))
    refused(cache.attend, "k_pages has element type", attend, dict(k_pages=_Array("float16", 9, 16, 4, 64)))
    refused(cache.attend, "differ", attend, dict(v_pages=_Array("bfloat16", 8, 16, 4, 64)))
    refused(cache.attend, "differ", attend, dict(v_pages=_Array("bfloat16", 9, 16, 4, 64, strides=(8192, 512, 64, 1))))
    refused(cache.attend, "last axis", attend, dict(k_pages=_Array("bfloat16", 9, 16, 4, 64, strides=(4096, 256, 1, 4))))
    refused(cache.attend, "16-byte aligned", attend, dict(k_pages=_Array("bfloat16", 9, 16, 4, 64, pointer=(1 << 20) + 8)))
    refused(cache.attend, "16-byte aligned", attend, dict(q=_Array("bfloat16", 2, 8, 64, strides=(515, 64, 1))))
    refused(cache.attend, "page_table has shape", attend, dict(page_table=_Array("int32", 2, 5)))
    refused(cache.attend, "a batch of 3", dict(base(3), q=_Array("bfloat16", 3, 8, 64), out=_Array("bfloat16", 3, 8, 64)))
    refused(cache.attend, "go together", attend, dict(k_new=_Array("bfloat16", 2, 4, 64)))
    refused(cache.attend, "not finite", attend, dict(scale=math.nan))
    refused(cache.attend, "weights and positions go together", attend, dict(weights=_Array("float32", 2, 4, 64)))
    refused(cache.attend, "lse has shape", attend, dict(lse=_Array("float32", 2, 4)))
    tracked = dict(weights=_Array("float32", 2, 4, 64), positions=_Array("int32", 2, 4, 64))
    refused(plain.attend, "made to track", attend, tracked)
    refused(cache.attend, "token counts", attend, tracked, dict(k_new=_Array("bfloat16", 2, 4, 64), v_new=_Array("bfloat16", 2, 4, 64)))
    append = dict(base(), k_new=_Array("bfloat16", 2, 3, 4, 64), v_new=_Array("bfloat16", 2, 3, 4, 64))
    refused(cache.append, "differ", append, dict(v_new=_Array("bfloat16", 2, 2, 4, 64)))
    refused(cache.append, "token counts", append, tracked)
    refused(cache.append, "counts has shape", append, dict(counts=_Array("int32", 3)))
    evict = dict(base(), tokens=_Array("int32", 2), keep=8, **tracked)
    refused(cache.evict, "rows to keep", evict, dict(keep=0))
    refused(cache.evict, "rows to keep", evict, dict(recent=5, sinks=4))
    refused(cache.evict, "rows to keep", evict, dict(recent=-1, sinks=0))
    refused(plain.evict, "made to track", evict, dict(recent=0))
    cache.destroy()
    refused(cache.evict, "destroyed", evict)


# ---- a paged cache and its plain forms -----------------------------------------------------------------------------


class _Case:
    """Pools, table and lengths in torch, with NaN in every place that nothing may read."""

    def __init__(self, dtype, heads, kv_heads, head_dim, page, lengths, seed=0, max_pages=None, layout="nhd", spare=2):
        import torch

        self.torch, self.dtype, self.heads, self.kv_heads, self.head_dim, self.page = torch, dtype, heads, kv_heads, head_dim, page
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths_list, batch = list(lengths), len(lengths)
        used = [-(-n // page) for n in lengths]
        self.max_pages = max_pages or max(1, max(used))
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=self.gen, device="cuda").tolist()
        table = torch.full((batch, self.max_pages), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table, self.lengths = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
        shape = (pages, page, kv_heads, head_dim) if layout == "nhd" else (pages, kv_heads, page, head_dim)
        self.k, self.v = (torch.full(shape, math.nan, dtype=_torch_type(dtype), device="cuda") for _ in range(2))
        if layout != "nhd":
            self.k, self.v = self.k.permute(0, 2, 1, 3), self.v.permute(0, 2, 1, 3)
        for b, n in enumerate(lengths):
            pg, row = self.places(b, n)
            self.k[pg, row], self.v[pg, row] = self.randn(n, kv_heads, head_dim), self.randn(n, kv_heads, head_dim)

    def randn(self, *shape, dtype=None):
        return self.torch.randn(shape, generator=self.gen, device="cuda").to(dtype or _torch_type(self.dtype))

    def places(self, b, n):
        t = self.torch.arange(n, device="cuda")
        return self.table[b].long()[t // self.page], t % self.page

    def tracking(self):
        torch, batch = self.torch, len(self.lengths_list)
        capacity = self.max_pages * self.page
        self.weights = torch.rand((batch, self.kv_heads, capacity), generator=self.gen, device="cuda")
        self.positions = torch.arange(capacity, device="cuda", dtype=torch.int32).expand(batch, self.kv_heads, -1).contiguous()
        self.tokens = self.lengths + 3
        return dict(tokens=self.tokens, weights=self.weights, positions=self.positions)

    def handle(self, be, batch=None, track=False):
        return be.paged_cache(CODE[self.dtype], batch or len(self.lengths_list), self.heads, self.kv_heads, self.head_dim, self.page,
                              self.max_pages, track=track)

    def attention(self, q, scale=None):
        """64-bit results of the cache as it is: out, lse, weights of every row, and the bounds of all three."""
        torch = self.torch
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        rep, batch = self.heads // self.kv_heads, len(self.lengths_list)
        out = torch.zeros((batch, self.heads, self.head_dim), dtype=torch.float64, device="cuda")
        lse = torch.full((batch, self.heads), -math.inf, dtype=torch.float64, device="cuda")
        p_sum = torch.zeros((batch, self.kv_heads, self.max_pages * self.page), dtype=torch.float64, device="cuda")
        out_bound, lse_bound, p_bound = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(p_sum)
        for b, n in enumerate(self.lengths_list):
            if not n:
                continue
            pg, row = self.places(b, n)
            for h in range(self.heads):
                k, v = self.k[pg, row, h // rep].double(), self.v[pg, row, h // rep].double()
                s = (k @ q[b, h].double()) * scale
                err = float((k.abs() @ q[b, h].double().abs()).max()) * abs(scale) * (self.head_dim + 16) * 2.0 ** -24
                p = torch.softmax(s, 0)
                out[b, h], lse[b, h] = p @ v, torch.logsumexp(s, 0)
                p_sum[b, h // rep, :n] += p
                off = 2 * err + 2.0 ** -17
                out_bound[b, h] = off * (p @ v.abs()) + HALF_ULP[self.dtype] * 2 * out[b, h].abs() + FLOOR[self.dtype]
                lse_bound[b, h] = err + 2.0 ** -20 * (1 + abs(float(lse[b, h])))
                p_bound[b, h // rep, :n] += off * p
        return out, lse, p_sum, out_bound, lse_bound, p_bound


GEOMETRY = [(32, 8, 128), (4, 2, 64), (8, 8, 64), (8, 1, 128), (12, 4, 96), (20, 1, 64), (40, 2, 128), (6, 3, 256), (5, 1, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", GEOMETRY)
def test_attend_over_lengths_and_heads(gpu_backend, dtype, heads, kv_heads, head_dim):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 300, 2]
    c = _Case(dtype, heads, kv_heads, head_dim, 16, lengths, seed=heads + head_dim)
    q = c.randn(len(lengths), heads, head_dim) * 2
    out, lse = c.torch.full_like(q, math.nan), c.torch.full((len(lengths), heads), math.nan, device="cuda")
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, lse=lse, stream=_stream())
    want, want_lse, _, bound, lse_bound, _ = c.attention(q)
    _within(out, want, bound, "out")
    _within(lse, want_lse, lse_bound, "lse")
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,layout", [(1, "nhd"), (5, "hnd"), (7, "nhd"), (48, "nhd"), (128, "hnd"), (1000, "nhd")])
def test_attend_pages_of_any_size_and_layout(gpu_backend, dtype, page, layout):
    c = _Case(dtype, 8, 2, 64, page, [257, 3, 1000, 999], seed=page, layout=layout)
    packed = c.randn(4, 8 + 4, 64)  # queries and new rows as one projection writes them
    q, out = packed[:, :8], c.torch.empty((4, 10, 64), dtype=packed.dtype, device="cuda")[:, 1:9]
    c.handle(gpu_backend, batch=6).attend(q, c.k, c.v, c.table, c.lengths, out, scale=0.3, stream=_stream())
    want, _, _, bound, _, _ = c.attention(q, 0.3)
    _within(out, want, bound, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths", [[2500], [5000, 0, 1, 777], [64] * 40])
def test_attend_appends_and_tracks(gpu_backend, dtype, lengths):
    c = _Case(dtype, 16, 4, 128, 16, lengths, seed=len(lengths))
    tracked = c.tracking()
    before = c.weights.clone()
    packed = c.randn(len(lengths), 24, 128)
    q, k_new, v_new = packed[:, :16], packed[:, 16:20], packed[:, 20:]
    last = [(b, n) for b, n in enumerate(lengths) if n]
    for b, n in last:  # what the call has to put there first
        pg, row = c.places(b, n)
        c.k[pg[-1], row[-1]] = math.nan
        c.v[pg[-1], row[-1]] = math.nan
    k_was, v_was = c.k.clone(), c.v.clone()
    out = c.torch.empty((len(lengths), 16, 128), dtype=packed.dtype, device="cuda")
    cache = c.handle(gpu_backend, track=True)
    cache.attend(q, c.k, c.v, c.table, c.lengths, out, k_new=k_new, v_new=v_new, stream=_stream(), **tracked)
    for b, n in last:
        pg, row = c.places(b, n)
        k_was[pg[-1], row[-1]], v_was[pg[-1], row[-1]] = k_new[b], v_new[b]
        before[b, :, n - 1] = 0
    same = lambda x, y: bool(((x == y) | (x.isnan() & y.isnan())).all())
    assert same(c.k, k_was) and same(c.v, v_was)
    want, _, p, bound, _, p_bound = c.attention(q)
    _within(out, want, bound, "out")
    _within(c.weights, before.double() + p, p_bound + 2.0 ** -23 * (before.double() + p), "weights")
    for b, n in enumerate(lengths):
        expect = c.torch.arange(c.max_pages * 16, device="cuda", dtype=c.torch.int32).expand(4, -1).clone()
        if n:
            expect[:, n - 1] = int(c.tokens[b]) - 1
        assert (c.positions[b] == expect).all()
    # the same call again: everything that was written is written again the same
    again = c.torch.empty_like(out)
    cache.attend(q, c.k, c.v, c.table, c.lengths, again, k_new=k_new, v_new=v_new, stream=_stream(), **tracked)
    assert c.torch.equal(out, again)


@pytest.mark.gpu
def test_attend_extreme_scores(gpu_backend):
    """Scores far apart, a row that takes everything, equal rows, infinities and NaN among what a sequence may see."""
    c = _Case("f32", 4, 2, 64, 16, [200, 33, 70, 50], seed=3)
    torch = c.torch
    q = c.randn(4, 4, 64) * 40
    pg, row = c.places(1, 33)
    c.k[pg, row] = c.k[pg[:1], row[:1]]  # equal scores
    pg, row = c.places(2, 70)
    c.v[pg[69], row[69], 0, 5] = math.inf
    c.k[pg[3], row[3], 1] = math.nan
    out, lse = torch.empty_like(q), torch.empty((4, 4), device="cuda")
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, lse=lse, stream=_stream())
    want, want_lse, _, bound, lse_bound, _ = c.attention(q)
    for b in (0, 1, 3):
        _within(out[b], want[b], bound[b], "out")
        _within(lse[b], want_lse[b], lse_bound[b], "lse")
    assert (out[2, :2, 5] == math.inf).all() or out[2, :2, 5].isnan().any()  # inf where its probability is not zero
    assert out[2, 2:].isnan().all() and lse[2, 2:].isnan().all()
    finite = [d for d in range(64) if d != 5]
    _within(out[2, :2][:, finite], want[2, :2][:, finite], bound[2, :2][:, finite], "beside the infinity")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (12, 1, 128), (4, 2, 64), (3, 1, 256)])
def test_attend_infinite_values_at_any_probability(gpu_backend, dtype, heads, kv_heads, head_dim):
    """An infinite value makes its dimension infinite however small its (f32) probability is, and nothing else."""
    c = _Case(dtype, heads, kv_heads, head_dim, 16, [300, 1, 40], seed=head_dim)
    torch = c.torch
    q = torch.zeros((3, heads, head_dim), dtype=_torch_type(dtype), device="cuda")
    q[:, :, 0] = 1
    pg, row = c.places(0, 300)
    c.k[pg, row, :, 1:] = 0
    c.k[pg, row, :, 0] = -c.torch.rand((300, kv_heads), generator=c.gen, device="cuda").to(q.dtype) * 60
    c.k[pg[17], row[17], :, 0] = 0.5  # the largest
    c.k[pg[40], row[40], :, 0] = -math.inf  # probability 0 with finite values: nothing
    for j, (t, score) in enumerate([(17, 0.5), (3, -5.0), (100, -17.0), (200, -30.0), (299, -60.0), (150, -80.0)]):
        c.k[pg[t], row[t], :, 0] = score
        c.v[pg[t], row[t], :, 2 * j] = math.inf
        c.v[pg[t], row[t], :, 2 * j + 1] = -math.inf
    c.v[pg[20], row[20], :, 0] = -math.inf  # both: NaN
    c.v[pg[8], row[8], :, 1] = math.nan
    pg, row = c.places(1, 1)
    c.v[pg[0], row[0], :, 3] = -math.inf
    out = torch.empty_like(q)
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, scale=1.0, stream=_stream())
    want, _, _, bound, _, _ = c.attention(q, 1.0)
    odd = ~want.isfinite()
    assert int(odd[0, 0].sum()) == 12 and int(odd[1, 0].sum()) == 1 and not odd[2].any()
    got = out.double()
    assert ((got == want) | (got.isnan() & want.isnan()))[odd].all(), (got[odd], want[odd])
    _within(out[~odd], want[~odd], bound[~odd], "beside the infinities")


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 2, 128), (2, 2, 68), (2, 1, 4), (9, 3, 100), (16, 2, 72), (11, 1, 256), (6, 2, 132)])
@pytest.mark.parametrize("track", [False, True])
def test_attend_f32_heads_and_widths(gpu_backend, heads, kv_heads, head_dim, track):
    """Every grouping of heads and width on the CUDA cores, with lengths around the rows of a warp and of a tile."""
    lengths = [0, 1, 7, 8, 9, 47, 48, 49, 95, 96, 97, 1500, 16, 17]
    c = _Case("f32", heads, kv_heads, head_dim, 7, lengths, seed=heads * head_dim)
    tracked = c.tracking() if track else {}
    before = c.weights.clone() if track else None
    q = c.randn(len(lengths), heads, head_dim)
    out, lse = c.torch.empty_like(q), c.torch.empty((len(lengths), heads), device="cuda")
    c.handle(gpu_backend, track=track).attend(q, c.k, c.v, c.table, c.lengths, out, lse=lse, stream=_stream(), **tracked)
    want, want_lse, p, bound, lse_bound, p_bound = c.attention(q)
    _within(out, want, bound, "out")
    _within(lse, want_lse, lse_bound, "lse")
    if track:
        _within(c.weights, before.double() + p, p_bound + 2.0 ** -23 * (before.double() + p), "weights")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("head_dim,score", [(64, -17.3), (128, -21.0), (256, -14.0)])
def test_attend_many_small_probabilities(gpu_backend, dtype, head_dim, score):
    """Thousands of rows that each weigh less than a 16-bit number can say, against one with all the rest and values of zero."""
    c = _Case(dtype, 4, 1, head_dim, 16, [6000], seed=7)
    q = c.torch.zeros((1, 4, head_dim), dtype=_torch_type(dtype), device="cuda")
    q[:, :, 0] = 1
    pg, row = c.places(0, 6000)
    c.k[pg, row, 0, 0] = score
    c.k[pg[1234], row[1234], 0, 0] = 0
    c.v[pg, row] = c.v[pg, row].abs() * 2000
    c.v[pg[1234], row[1234]] = 0
    out = c.torch.empty_like(q)
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, scale=1.0, stream=_stream())
    want, _, _, bound, _, _ = c.attention(q, 1.0)
    assert (want > 4 * bound).all()
    _within(out, want, bound, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 1, 64), (8, 2, 128), (12, 1, 128), (3, 1, 256)])
@pytest.mark.parametrize("score", [-math.inf, -400.0])
def test_attend_rows_of_probability_zero_add_nothing(gpu_backend, dtype, heads, kv_heads, head_dim, score):
    """Rows whose probability is zero, or too small for f32, with values as large as sums of them allow: what they add rounds to 0."""
    c = _Case(dtype, heads, kv_heads, head_dim, 16, [5000, 40], seed=11)
    torch = c.torch
    q = torch.zeros((2, heads, head_dim), dtype=_torch_type(dtype), device="cuda")
    q[:, :, 0] = 1
    for b, n in enumerate([5000, 40]):
        pg, row = c.places(b, n)
        c.k[pg, row] = 0
        c.k[pg, row, :, 0] = score
        c.v[pg, row] = min(torch.finfo(q.dtype).max, 2.0 ** 112)
        top = slice(n // 3, n // 3 + 2)  # two rows with all of the probability
        c.k[pg[top], row[top], :, 0] = 0
        c.v[pg[top], row[top]] = 0
        c.v[pg[top], row[top], :, ::2] = 0.5
    out = torch.full_like(q, math.nan)
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, scale=1.0, stream=_stream())
    want = torch.zeros_like(out)
    want[..., ::2] = 0.5
    assert torch.equal(out, want), (out - want).abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 1, 64), (16, 1, 64), (8, 2, 128), (12, 1, 128), (3, 1, 256)])
@pytest.mark.parametrize("score", [-14.0, -15.3, -22.0, -26.0, -30.0, -40.0, -60.0, None])
def test_attend_probabilities_of_any_size(gpu_backend, dtype, heads, kv_heads, head_dim, score):
    """Tens of thousands of rows of one sign against one row with all the rest and values of zero; None: scores from 0 to -60."""
    n = 40000
    c = _Case(dtype, heads, kv_heads, head_dim, 64, [n], seed=13)
    torch = c.torch
    q = torch.zeros((1, heads, head_dim), dtype=_torch_type(dtype), device="cuda")
    q[:, :, 0] = 1
    pg, row = c.places(0, n)
    c.k[pg, row, :, 0] = score if score else (-60 * torch.rand((n, kv_heads), generator=c.gen, device="cuda")).to(q.dtype)
    c.v[pg, row] = (c.v[pg, row].abs() * 15000).clamp(max=60000)
    c.k[pg[12345], row[12345], :, 0] = 0
    c.v[pg[12345], row[12345]] = 0
    out, lse = torch.empty_like(q), torch.empty((1, heads), device="cuda")
    c.handle(gpu_backend).attend(q, c.k, c.v, c.table, c.lengths, out, lse=lse, scale=1.0, stream=_stream())
    want, want_lse, _, bound, lse_bound, _ = c.attention(q, 1.0)
    _within(out, want, bound, "out")
    _within(lse, want_lse, lse_bound, "lse")


@pytest.mark.gpu
def test_attend_offsets_beyond_32_bits(gpu_backend):
    import torch

    stride = (1 << 30) + 64
    flat = [torch.empty(2 * stride + 16 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pools = [f.as_strided((3, 16, 1, 64), (stride, 64, 64, 1)) for f in flat]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for p in pools:
        p.copy_(torch.randn(p.shape, generator=gen, device="cuda"))
    q = torch.randn((1, 4, 64), generator=gen, device="cuda").bfloat16()
    table, lengths = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([45], dtype=torch.int32, device="cuda")
    new = [torch.randn((1, 1, 64), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    out = torch.empty_like(q)
    cache = gpu_backend.paged_cache(P.BF16_CODE, 1, 4, 1, 64, 16, 3)
    cache.append(*pools, table, torch.tensor([3], dtype=torch.int32, device="cuda"), new[0][:, None], new[1][:, None], stream=_stream())
    assert torch.equal(pools[0][2, 2], new[0][0]) and torch.equal(pools[1][2, 2], new[1][0])
    cache.attend(q, *pools, table, lengths, out, stream=_stream())
    k, v = (torch.cat([p[2], p[0], p[1]])[:45, 0].double() for p in pools)
    p = torch.softmax((q[0].double() @ k.T) / 8, 1)
    _within(out[0], p @ v, 2.0 ** -7 * (p @ v.abs()), "out")


@pytest.mark.gpu
def test_out_of_range_pages_and_lengths_are_reported_and_not_followed(gpu_backend):
    c = _Case("bf16", 4, 2, 64, 16, [40, 40, 40], seed=9)
    q, out = c.randn(3, 4, 64), c.torch.empty((3, 4, 64), dtype=c.torch.bfloat16, device="cuda")
    cache = c.handle(gpu_backend)
    want, _, _, bound, _, _ = c.attention(q)
    for entry in (-1, 10 ** 6):
        table = c.table.clone()
        table[1, 1] = entry
        cache.attend(q, c.k, c.v, table, c.lengths, out, stream=_stream())
        c.torch.cuda.synchronize()
        with pytest.raises(be_mod.BackendError, match="outside the pool"):
            gpu_backend.synchronize()
        _within(out[::2], want[::2], bound[::2], "the other sequences")
    for n in (-5, 49):
        lengths = c.lengths.clone()
        lengths[1] = n
        table = c.table.clone()
        table[1, 2] = 0
        cache.attend(q, c.k, c.v, table, lengths, out, stream=_stream())
        c.torch.cuda.synchronize()
        with pytest.raises(be_mod.BackendError, match="outside the page table"):
            gpu_backend.synchronize()
        _within(out[::2], want[::2], bound[::2], "the other sequences")
    gpu_backend.synchronize()  # reported once


@pytest.mark.gpu
def test_status_waits_for_the_callers_stream(gpu_backend):
    """A bad argument of a call that a stream has not come to yet is known when its status is."""
    c = _Case("bf16", 4, 2, 64, 16, [40, 40], seed=10)
    torch, cache = c.torch, c.handle(gpu_backend)
    q, table = c.randn(2, 4, 64), c.table.clone()
    table[1, 1] = 10 ** 6
    out, x = torch.empty_like(q), torch.zeros((3, 100), device="cuda")
    tokens, score = torch.tensor([5, 100, 7], dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # 0.1 s
    cache.attend(q, c.k, c.v, table, c.lengths, out, stream=side.cuda_stream)
    gpu_backend.synchronize()  # of the backend's stream, where nothing happened
    with pytest.raises(be_mod.BackendError, match="outside the pool of pages .code 40.;"):
        gpu_backend.operators_status(stream=side.cuda_stream)
    gpu_backend.operators_status(stream=side.cuda_stream)  # reported once
    # several of them, from several calls
    cache.attend(q, c.k, c.v, table, c.lengths, out, stream=side.cuda_stream)
    gpu_backend.token_log_probs(x, tokens, score, stream=side.cuda_stream)
    with pytest.raises(be_mod.BackendError, match="code 40.*code 42"):
        gpu_backend.operators_status(stream=side.cuda_stream)
    gpu_backend.operators_status()
    gpu_backend.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("wait_first", [True, False])
def test_an_operators_report_does_not_replace_that_of_a_wait(gpu_backend, wait_first):
    import torch

    x, score = torch.zeros((3, 100), device="cuda"), torch.empty(3, device="cuda")
    tokens = torch.tensor([5, 100, 7], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for wait in (wait_first, not wait_first):
        if wait:
            gpu_backend.bounded_wait_probe(0, timeout_ms=20)
        else:
            gpu_backend.token_log_probs(x, tokens, score)
    torch.cuda.synchronize()
    reports = []
    for _ in range(2):
        with pytest.raises(be_mod.BackendError) as e:
            gpu_backend.synchronize()
        reports.append(str(e.value))
    assert "bounded wait" in reports[0] and "outside the vocabulary" in reports[1]
    gpu_backend.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv_heads,head_dim,page", [("bf16", 8, 128, 16), ("f32", 2, 64, 5), ("f16", 1, 8, 3), ("f32", 3, 4, 64)])
@pytest.mark.parametrize("track", [False, True])
def test_append(gpu_backend, dtype, kv_heads, head_dim, page, track):
    import torch

    lengths, counts = [7, 40, 1, 0, 33], [7, 13, 1, 0, 0]
    c = _Case(dtype, kv_heads, kv_heads, head_dim, page, lengths, seed=page)
    tracked = c.tracking() if track else {}
    new = c.randn(5, 14, 2, kv_heads, head_dim)
    k_new, v_new = new[:, :, 0], new[:, :, 1]
    k, v = c.k.clone(), c.v.clone()
    weights, positions = (c.weights.clone(), c.positions.clone()) if track else (None, None)
    for b, (n, m) in enumerate(zip(lengths, counts)):
        pg, row = (x[n - m:] for x in c.places(b, n))
        k[pg, row], v[pg, row] = k_new[b, :m], v_new[b, :m]
        if track:
            weights[b, :, n - m:n] = 0
            positions[b, :, n - m:n] = torch.arange(m, device="cuda", dtype=torch.int32) + (c.tokens[b] - m)
    cache = c.handle(gpu_backend, track=track)
    cache.append(c.k, c.v, c.table, c.lengths, k_new, v_new, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), stream=_stream(), **tracked)
    same = lambda x, y: bool(((x == y) | (x.isnan() & y.isnan())).all())
    assert same(c.k, k) and same(c.v, v)
    if track:
        assert torch.equal(c.weights, weights) and torch.equal(c.positions, positions)
    cache.append(c.k, c.v, c.table, c.lengths, k_new[:, :0], v_new[:, :0], stream=_stream())
    assert same(c.k, k)
    # more rows than a sequence has: reported, the rows that fit its length are the first ones
    cache.append(c.k, c.v, c.table, c.lengths, k_new[:, :2], v_new[:, :2], stream=_stream())
    torch.cuda.synchronize()
    with pytest.raises(be_mod.BackendError, match="count beyond its length"):
        gpu_backend.synchronize()


def _evicted(lengths, tokens, weights, positions, keep, recent, sinks):
    """Per (sequence, head): which row each place holds afterwards, as lists."""
    out = []
    for b, n in enumerate(lengths):
        heads = []
        for w, p in zip(weights[b], positions[b]):
            protected = [p[t] < sinks or p[t] >= tokens[b] - recent for t in range(n)]
            value = lambda t: math.inf if w[t] != w[t] else w[t]
            rank = sorted(range(n), key=lambda t: (not protected[t], not w[t] != w[t], -value(t), t))
            kept = set(rank[:keep])
            place, moved = list(range(min(n, keep))), iter(t for t in range(keep, n) if t in kept)
            heads.append([t if t in kept else next(moved) for t in place])
        out.append(heads)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,page,keep,recent,sinks,kind", [
    ([100, 0, 1, 65, 64, 63], 16, 64, 8, 4, "spread"), ([2049], 16, 2048, 256, 4, "spread"), ([3000, 2999, 10], 8, 1000, 100, 0, "spread"),
    ([500, 400], 20, 100, 0, 0, "ties"), ([500], 16, 100, 60, 40, "zero"), ([1500, 1499], 16, 1, 0, 0, "spread"), ([700], 16, 600, 0, 0, "odd values"),
    ([1000], 16, 300, 0, 0, "ascending"), ([1000], 16, 300, 0, 0, "descending"), ([50], 16, 60, 60, 0, "spread")])
def test_evict(gpu_backend, lengths, page, keep, recent, sinks, kind, in_place):
    import torch

    c = _Case("bf16", 4, 2, 16, page, lengths, seed=keep)
    t = c.tracking()
    w = c.weights
    if kind == "ties":
        w.copy_((w * 4).floor())
    elif kind == "zero":
        w.copy_(torch.where(w < 0.5, 0.0, -0.0))
    elif kind == "odd values":
        w[..., ::7] = math.nan
        w[..., 1::7] = math.inf
        w[..., 2::7] = -math.inf
        w[..., 3::7] = -1.0
        w[..., 4::7] = 1e-42
    elif kind == "ascending":
        w.copy_(torch.arange(w.shape[-1], device="cuda").float().expand(w.shape))
    elif kind == "descending":
        w.copy_(-torch.arange(w.shape[-1], device="cuda").float().expand(w.shape))
    perm = torch.rand(w.shape, generator=c.gen, device="cuda").argsort(-1).int()
    c.positions.copy_(perm)
    c.tokens.fill_(w.shape[-1])
    place = _evicted(lengths, c.tokens.tolist(), w.cpu().tolist(), c.positions.cpu().tolist(), keep, recent, sinks)
    k, v = c.k.clone(), c.v.clone()
    want_w, want_p = torch.zeros_like(w), torch.full_like(c.positions, -1)
    for b, n in enumerate(lengths):
        pg, row = c.places(b, n)
        for g in range(2):
            at = torch.tensor(place[b][g], dtype=torch.long, device="cuda")
            left = len(at)
            k[pg[:left], row[:left], g], v[pg[:left], row[:left], g] = c.k[pg[at], row[at], g], c.v[pg[at], row[at], g]
            want_w[b, g, :left], want_p[b, g, :left] = w[b, g, at], c.positions[b, g, at]
    outs = {} if in_place else dict(lengths_out=torch.empty_like(c.lengths), weights_out=torch.empty_like(w), positions_out=torch.empty_like(c.positions))
    was = [x.clone() for x in (c.lengths, w, c.positions)]
    cache = c.handle(gpu_backend, track=True)
    cache.evict(c.k, c.v, c.table, c.lengths, c.tokens, w, c.positions, keep, recent=recent, sinks=sinks, stream=_stream(), **outs)
    got = (c.lengths, w, c.positions) if in_place else (outs["lengths_out"], outs["weights_out"], outs["positions_out"])
    same = lambda x, y: bool(((x == y) | (x.isnan() & y.isnan())).all()) if x.is_floating_point() else torch.equal(x, y)
    assert got[0].tolist() == [min(n, keep) for n in lengths]
    assert same(got[1], want_w) and same(got[2], want_p) and same(c.k, k) and same(c.v, v)
    if not in_place:
        assert all(same(x, y) for x, y in zip((c.lengths, w, c.positions), was))
        # a second pass over the same rows moves the same ones again
        cache.evict(c.k, c.v, c.table, c.lengths, c.tokens, w, c.positions, keep, recent=recent, sinks=sinks, stream=_stream(), **outs)
        assert same(outs["weights_out"], want_w) and same(c.k, k) and same(c.v, v)


@pytest.mark.gpu
def test_evict_of_a_cache_too_long_for_shared_memory(gpu_backend):
    import torch

    n, keep = 70001, 40000
    c = _Case("f16", 1, 1, 8, 128, [n], seed=2)
    t = c.tracking()
    w = c.weights[0, 0, :n].double().cpu().numpy()
    kept = np.zeros(n, bool)
    protected = np.arange(n) >= int(c.tokens[0]) - 50
    order = np.lexsort((np.arange(n), -w, ~protected))
    kept[order[:keep]] = True
    place = np.arange(keep)
    place[~kept[:keep]] = keep + np.flatnonzero(kept[keep:])
    at = torch.from_numpy(place).cuda()
    pg, row = c.places(0, n)
    k, want_w = c.k[pg[at], row[at]].clone(), c.weights[0, 0, at].clone()
    c.handle(gpu_backend, track=True).evict(c.k, c.v, c.table, c.lengths, c.tokens, c.weights, c.positions, keep, recent=50, stream=_stream())
    assert torch.equal(c.k[pg[:keep], row[:keep]], k) and torch.equal(c.weights[0, 0, :keep], want_w)
    assert int(c.lengths[0]) == keep and (c.positions[0, 0, keep:] == -1).all() and (c.positions[0, 0, :keep] == at).all()


@pytest.mark.gpu
@pytest.mark.parametrize("track", [False, True])
def test_a_batch_of_no_sequences(gpu_backend, track):
    """Empty tensors have no address; such a call does nothing and is not an error, but its other arguments are looked at."""
    import torch

    cache = gpu_backend.paged_cache(P.BF16_CODE, 2, 4, 2, 64, 16, 3, track=track)
    pools = [torch.zeros((9, 16, 2, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    empty = lambda *d, t=torch.int32: torch.empty(d, dtype=t, device="cuda")
    view = dict(k_pages=pools[0], v_pages=pools[1], page_table=empty(0, 3), lengths=empty(0), stream=_stream())
    if track:
        view.update(tokens=empty(0), weights=empty(0, 2, 48, t=torch.float32), positions=empty(0, 2, 48))
    rows = lambda *d: empty(0, *d, t=torch.bfloat16)
    cache.append(k_new=rows(5, 2, 64), v_new=rows(5, 2, 64), counts=empty(0), **view)
    cache.attend(rows(4, 64), out=rows(4, 64), lse=empty(0, 4, t=torch.float32), k_new=rows(2, 64), v_new=rows(2, 64), **view)
    if track:
        cache.evict(keep=10, **view)
        with pytest.raises(be_mod.BackendError, match="rows to keep"):
            cache.evict(keep=0, **view)
    gpu_backend.operators_status(stream=_stream())
    assert not pools[0].any() and not pools[1].any()


@pytest.mark.gpu
def test_one_handle_serves_batches_of_different_sizes(gpu_backend):
    """Workspaces hold counters that every call leaves at zero, whatever the batch was before."""
    torch = None
    cache = None
    for turn, lengths in enumerate([[900], [500] * 90, [700, 0, 300], [100] * 90, [2000]]):
        c = _Case("bf16", 8, 2, 64, 16, lengths, seed=turn, max_pages=125)
        torch = c.torch
        cache = cache or c.handle(gpu_backend, batch=100, track=True)
        c.tracking()
        q = c.randn(len(lengths), 8, 64)
        out = torch.empty_like(q)
        cache.attend(q, c.k, c.v, c.table, c.lengths, out, stream=_stream())
        want, _, _, bound, _, _ = c.attention(q)
        _within(out, want, bound, lengths)
        keep = 80
        place = _evicted(lengths, c.tokens.tolist(), c.weights.cpu().tolist(), c.positions.cpu().tolist(), keep, 5, 2)
        cache.evict(c.k, c.v, c.table, c.lengths, c.tokens, c.weights, c.positions, keep, recent=5, sinks=2, stream=_stream())
        assert c.lengths.tolist() == [min(n, keep) for n in lengths]
        for b, heads in enumerate(place):
            for g, at in enumerate(heads):
                assert c.positions[b, g, :len(at)].tolist() == at, (turn, b, g)


# ---- scoring -------------------------------------------------------------------------------------------------------


def _score(be, logits, tokens, top, scale=1.0, stream=None):
    import torch

    rows = logits.shape[0]
    f = lambda *s: torch.full(s, 12345.0, device="cuda")
    out = dict(log_probs=f(rows), entropy=f(rows), lse=f(rows))
    if top:
        out.update(top_ids=torch.full((rows, top), -9, dtype=torch.int32, device="cuda"), top_log_probs=f(rows, top))
    be.token_log_probs(logits, tokens, **out, scale=scale, stream=_stream() if stream is None else stream)
    return out


def _check_score(out, logits, tokens, top, scale):
    import torch

    x = logits.double() * scale
    vocab = x.shape[1]
    lse = torch.logsumexp(x, 1)
    p = torch.softmax(x, 1)
    entropy = -torch.special.xlogy(p, p).sum(1)
    largest = torch.where(x.isinf(), 0.0, x).abs().amax(1)
    # an exponent is off by 2^-22 of the largest logit, a sum of n terms in one thread by n 2^-24
    off = 2.0 ** -22 * largest + (vocab / 512 + 64) * 2.0 ** -23
    _within(out["lse"], lse, off, "lse")
    _within(out["entropy"], entropy, off * (4 + 2 * math.log(vocab)), "entropy")
    given = torch.where(tokens < 0, 0.0, x.gather(1, tokens.long().clamp(min=0)[:, None])[:, 0] - lse)
    _within(out["log_probs"], given, 2 * off, "log_probs")
    if top:
        order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(out["top_ids"].long(), order), "top_ids"
        _within(out["top_log_probs"], x.gather(1, order) - lse[:, None], 2 * off[:, None], "top_log_probs")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,top,stride,scale", [
    (3, 1, 1, 1, 1.0), (5, 2, 2, 3, 2.5), (4, 7, 7, 7, 1.0), (9, 40, 32, 41, 0.7), (2, 255, 64, 255, 1.0), (1, 257, 3, 257, 1.0),
    (33, 1024, 20, 1024, 1.0), (3, 4099, 64, 4100, 1.0), (2, 32001, 20, 32001, 0.5), (1, 128256, 5, 128256, 1.0), (300, 32000, 5, 32000, 1.0),
    (7, 8192, 0, 8200, 1.0), (1, 200003, 64, 200003, 3.0)])
def test_token_log_probs(gpu_backend, dtype, rows, vocab, top, stride, scale):
    import torch

    scale = float(np.float32(scale))  # an f32 argument
    gen = torch.Generator(device="cuda").manual_seed(vocab + rows)
    store = torch.full((rows * stride + 1,), math.nan, dtype=_torch_type(dtype), device="cuda")
    logits = store[1:].as_strided((rows, vocab), (stride, 1), storage_offset=1)  # no row starts on a 16-byte boundary by itself
    logits.copy_(torch.randn((rows, vocab), generator=gen, device="cuda") * 3)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[rows // 2] = -1
    out = _score(gpu_backend, logits, tokens, top, scale)
    _check_score(out, logits, tokens, top, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [12, 700])
def test_token_log_probs_of_masked_and_tied_rows(gpu_backend, dtype, rows):
    import torch

    lowest = torch.finfo(_torch_type(dtype)).min
    gen = torch.Generator(device="cuda").manual_seed(rows)
    vocab, top = 20011, 48
    x = torch.randn((rows, vocab), generator=gen, device="cuda")
    x[0] = -math.inf
    x[1] = lowest
    x[2, ::3] = -math.inf
    x[3, 5:] = lowest
    x[4] = 0.25                                     # all equal
    x[5] = (x[5] * 2).round()                       # long ties
    x[6, :] = -math.inf
    x[6, 19999] = 1.0                               # one left
    x[7, 4000:4600] = 9.0 + x[7, 4000:4600].abs()   # the likeliest side by side
    x[8, 300:] = -2.0                               # a tie at the last places
    x[9, ::2] = -0.0
    x[9, 1::2] = 0.0
    logits = x.to(_torch_type(dtype))
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[6] = 19999
    out = _score(gpu_backend, logits, tokens, top)
    keep = [i for i in range(rows) if i != 0]
    _check_score({n: v[keep] for n, v in out.items()}, logits[keep], tokens[keep], top, 1.0)
    assert out["lse"][0] == -math.inf and out["entropy"][0] == 0 and out["log_probs"][0] == -math.inf
    assert out["top_ids"][0].tolist() == list(range(top)) and (out["top_log_probs"][0] == -math.inf).all()
    assert out["log_probs"][6] == 0 and out["entropy"][6] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,top,stride", [
    (700, 1024, 5, 1024), (5, 1024, 64, 1027), (650, 131, 33, 133), (601, 4000, 20, 4001), (600, 6137, 8, 6137), (1300, 3, 3, 3),
    (84, 30011, 5, 30011), (98, 40000, 3, 40001), (118, 33001, 20, 33001), (197, 9000, 1, 9000), (296, 130000, 2, 130000)])
def test_token_log_probs_by_warps_and_by_any_number_of_blocks(gpu_backend, dtype, rows, vocab, top, stride):
    """Rows of a few batches and clusters of each size, with masked logits, ties and empty rows among them."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.empty((rows, stride), device="cuda")
    x[:, :vocab] = torch.randn((rows, vocab), generator=gen, device="cuda") * 3
    x[1::3, :vocab].masked_fill_(torch.rand((len(range(1, rows, 3)), vocab), generator=gen, device="cuda") < 0.9, -math.inf)
    x[1::3, vocab - 1] = 0.5
    x[2::3] = x[2::3].round()
    x[3] = -math.inf
    logits = x.to(_torch_type(dtype))[:, :vocab]
    tokens = torch.randint(-1, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    out = _score(gpu_backend, logits, tokens, top)
    keep = [i for i in range(rows) if i != 3]
    _check_score({n: v[keep] for n, v in out.items()}, logits[keep], tokens[keep], top, 1.0)
    assert out["lse"][3] == -math.inf and out["top_ids"][3].tolist() == list(range(top))


@pytest.mark.gpu
def test_token_log_probs_of_nan_and_infinity(gpu_backend):
    import torch

    x = torch.zeros((4, 5000), device="cuda")
    x[0, 4321] = math.nan
    x[1, 77] = math.inf
    x[2, 3] = -math.inf
    out = _score(gpu_backend, x, torch.zeros(4, dtype=torch.int32, device="cuda"), 3)
    for i in (0, 1):
        assert out["lse"][i].isnan() and out["entropy"][i].isnan() and out["log_probs"][i].isnan()
    assert out["top_ids"].tolist() == [[4321, 0, 1], [77, 0, 1], [0, 1, 2], [0, 1, 2]]
    assert abs(float(out["lse"][2]) - math.log(4999)) < 1e-5 and abs(float(out["lse"][3]) - math.log(5000)) < 1e-5


@pytest.mark.gpu
def test_token_ids_beyond_the_vocabulary_are_reported(gpu_backend):
    import torch

    x = torch.zeros((3, 100), device="cuda")
    tokens = torch.tensor([5, 100, 7], dtype=torch.int32, device="cuda")
    out = _score(gpu_backend, x, tokens, 0)
    torch.cuda.synchronize()
    with pytest.raises(be_mod.BackendError, match="outside the vocabulary"):
        gpu_backend.synchronize()
    assert out["log_probs"][1].isnan() and abs(float(out["log_probs"][2]) + math.log(100)) < 1e-5
    grad = torch.empty_like(x)
    gpu_backend.token_log_probs_backward(x, tokens, out["lse"], grad, grad_log_probs=torch.ones(3, device="cuda"), stream=_stream())
    torch.cuda.synchronize()
    with pytest.raises(be_mod.BackendError, match="outside the vocabulary"):
        gpu_backend.synchronize()
    gpu_backend.synchronize()


def _loss64(x, tokens, g, h):
    """sum g log p[token] + h entropy, in 64 bits on the host, of scaled logits x."""
    m = x.max(1, keepdims=True)
    log_p = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
    p = np.exp(log_p)
    given = np.array([log_p[r, t] if t >= 0 else 0.0 for r, t in enumerate(tokens)])
    entropy = -(p * np.where(p > 0, log_p, 0.0)).sum(1)
    return float((g * given + h * entropy).sum())


@pytest.mark.gpu
def test_gradient_against_differences(gpu_backend):
    import torch

    rng = np.random.default_rng(4)
    rows, vocab, scale = 5, 13, 1.7
    x, tokens = rng.standard_normal((rows, vocab)) * 2, np.array([3, 0, 12, -1, 7])
    g, h = rng.standard_normal(rows), rng.standard_normal(rows)
    cuda = lambda a, t=torch.float32: torch.tensor(a, dtype=t, device="cuda")
    x32 = cuda(x)
    fw = _score(gpu_backend, x32, cuda(tokens, torch.int32), 0, scale)
    grad = torch.empty_like(x32)
    gpu_backend.token_log_probs_backward(x32, cuda(tokens, torch.int32), fw["lse"], grad, grad_log_probs=cuda(g), entropy=fw["entropy"],
                                         grad_entropy=cuda(h), scale=scale, stream=_stream())
    x, step = x32.double().cpu().numpy(), 1e-5
    for r in range(rows):
        for j in range(vocab):
            hi, lo = x.copy(), x.copy()
            hi[r, j] += step
            lo[r, j] -= step
            slope = (_loss64(hi * scale, tokens, g, h) - _loss64(lo * scale, tokens, g, h)) / (2 * step)
            assert abs(slope - float(grad[r, j])) < 2e-6 * (1 + abs(slope)), (r, j)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,stride,grad_stride,which,scale", [
    (3, 1, 1, 1, "both", 1.0), (4, 7, 9, 7, "both", 0.5), (5, 1000, 1000, 1000, "log_probs", 1.0), (97, 32001, 32001, 32001, "both", 0.8),
    (2, 128256, 128256, 128256, "entropy", 1.0), (6, 5003, 5003, 5008, "both", 2.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_token_log_probs_backward(gpu_backend, dtype, rows, vocab, stride, grad_stride, which, scale, in_place):
    import torch

    scale = float(np.float32(scale))  # an f32 argument
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    make = lambda s: torch.full((rows * s + 3,), 7.0, dtype=_torch_type(dtype), device="cuda").as_strided((rows, vocab), (s, 1), storage_offset=3)
    logits = make(stride)
    logits.copy_(torch.randn((rows, vocab), generator=gen, device="cuda") * 3)
    if vocab > 100:
        logits[0, ::2] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[rows - 1] = -1
    if vocab > 100:
        tokens[0] = 2  # ruled out, and given all the same
    g, h = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    fw = _score(gpu_backend, logits, tokens, 0, scale)
    log_p = logits.double() * scale - fw["lse"].double()[:, None]
    p = torch.exp(log_p)
    given = torch.where(tokens < 0, 0.0, g.double())[:, None] if which != "entropy" else torch.zeros((rows, 1), dtype=torch.float64, device="cuda")
    term = torch.where(p > 0, log_p + fw["entropy"].double()[:, None], 0.0) * (h.double()[:, None] if which != "log_probs" else 0.0)
    want = -p * (given + term)
    hot = torch.zeros_like(want).scatter(1, tokens.long().clamp(min=0)[:, None], 1.0)
    want = (want + hot * given) * scale
    size = scale * (p * (given.abs() + term.abs()) * (2 + log_p.abs().clamp(max=200)) + hot * given.abs())
    bound = 2 * HALF_ULP[dtype] * want.abs() + 2.0 ** -21 * size + FLOOR[dtype]
    grad = logits if in_place else make(grad_stride)
    gpu_backend.token_log_probs_backward(logits, tokens, fw["lse"], grad, grad_log_probs=g if which != "entropy" else None, entropy=fw["entropy"],
                                         grad_entropy=h if which != "log_probs" else None, scale=scale, stream=_stream())
    _within(grad, want, bound, "grad")
    if not in_place and grad_stride > vocab:
        gap = grad.as_strided((rows - 1, grad_stride - vocab), (grad_stride, 1), storage_offset=3 + vocab)
        assert (gap == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("large", [1e9, -1e20, 1e34])
def test_gradient_of_ruled_out_logits_under_large_gradients(gpu_backend, dtype, large):
    """What is ruled out, by -inf or by the type's lowest value, has gradient 0 whatever the entropy's gradient is."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(8)
    logits = (torch.randn((6, 1000), generator=gen, device="cuda") * 3).to(_torch_type(dtype))
    out_of = torch.rand(logits.shape, generator=gen, device="cuda") < 0.5
    logits[:3] = torch.where(out_of[:3], -math.inf, logits[:3])
    logits[3:] = torch.where(out_of[3:], torch.finfo(logits.dtype).min, logits[3:])
    tokens = torch.where(out_of, -1.0, 1.0).argmax(1).int()
    fw = _score(gpu_backend, logits, tokens, 0)
    g, h = torch.randn(6, generator=gen, device="cuda"), torch.full((6,), large, device="cuda")
    grad = torch.empty_like(logits)
    gpu_backend.token_log_probs_backward(logits, tokens, fw["lse"], grad, grad_log_probs=g, entropy=fw["entropy"], grad_entropy=h, stream=_stream())
    log_p = logits.double() - fw["lse"].double()[:, None]
    p = torch.exp(log_p)
    term = torch.where(p > 0, (log_p + fw["entropy"].double()[:, None]) * h.double()[:, None], 0.0)
    hot = torch.zeros_like(p).scatter(1, tokens.long()[:, None], g.double()[:, None])
    size = p * (g.double().abs()[:, None] + term.abs()) * (2 + log_p.abs().clamp(max=200)) + hot.abs()
    # beside the bound of the test above: ln p + entropy, of numbers below 16, may cancel down to their rounding
    bound = 2 * HALF_ULP[dtype] * size + 2.0 ** -21 * size + p * abs(large) * 16 * 2.0 ** -23
    assert (grad[out_of] == 0).all()
    _within(grad, hot - p * (g.double()[:, None] + term), bound, "grad")


@pytest.mark.gpu
def test_gradient_of_a_row_without_possible_tokens_is_finite(gpu_backend):
    import torch

    x = torch.full((2, 300), -math.inf, device="cuda", dtype=torch.bfloat16)
    x[1] = 1.0
    tokens = torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    fw = _score(gpu_backend, x, tokens, 0)
    grad, one = torch.empty_like(x), torch.ones(2, device="cuda")
    gpu_backend.token_log_probs_backward(x, tokens, fw["lse"], grad, grad_log_probs=one, entropy=fw["entropy"], grad_entropy=one, stream=_stream())
    assert grad[0, 4] == 1 and grad[0].count_nonzero() == 1 and grad.isfinite().all()


# ---- how they are called -------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_operators_on_the_backends_own_buffers_and_stream(gpu_backend):
    """Buffers and executables of the backend and the operators work on one stream: no waits between them."""
    be = gpu_backend
    rng = np.random.default_rng(0)
    logits = (rng.standard_normal((6, 3001)) * 3).astype(np.float32)
    b = be_mod.plan_mod.PlanBuilder()
    p = b.parameter(P.F32, [6, 3001])
    b.set_outputs([p + p])
    doubled = be.execute_executable(be.compile_executable(b), [be.buffer_from_host(logits / 2)])[0]
    tokens = be.buffer_from_host(np.arange(6, dtype=np.int32) * 100)
    out = {n: be.allocate_buffer(P.F32, [6]) for n in ("log_probs", "entropy", "lse")}
    ids, best = be.allocate_buffer(P.S32, [6, 4]), be.allocate_buffer(P.F32, [6, 4])
    be.token_log_probs(doubled, tokens, **out, top_ids=ids, top_log_probs=best)
    x = (logits / 2).astype(np.float64) * 2
    lse = np.log(np.exp(x).sum(1))
    assert np.abs(out["lse"].to_numpy() - lse).max() < 1e-5
    assert np.abs(out["log_probs"].to_numpy() - (x[np.arange(6), np.arange(6) * 100] - lse)).max() < 2e-5
    assert np.array_equal(ids.to_numpy(), np.argsort(-x, 1, kind="stable")[:, :4])
    destroyed = be.allocate_buffer(P.F32, [6])
    destroyed.destroy()
    with pytest.raises(be_mod.BackendError):
        be.token_log_probs(doubled, tokens, destroyed)


@pytest.mark.gpu
def test_operators_on_other_streams_and_in_graphs(gpu_backend):
    import torch

    c = _Case("bf16", 8, 2, 64, 16, [300, 41], seed=5)
    cache, q = c.handle(gpu_backend, track=True), c.randn(2, 8, 64)
    tracked = c.tracking()
    zero, order = c.weights.clone(), c.positions.clone()
    out = torch.zeros_like(q)
    want, _, p, bound, _, p_bound = c.attention(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)  # the inputs are written well after the call is made
        late.copy_(q)
        cache.attend(late, c.k, c.v, c.table, c.lengths, out, stream=side.cuda_stream)
    side.synchronize()
    _within(out, want, bound, "on a side stream")
    logits = torch.randn((4, 9000), generator=c.gen, device="cuda").bfloat16()
    tokens = torch.tensor([1, 2, 3, -1], dtype=torch.int32, device="cuda")
    scored = _score(gpu_backend, logits, tokens, 6, stream=_stream())
    graph = torch.cuda.CUDAGraph()
    again = {n: torch.zeros_like(v) for n, v in scored.items()}
    with torch.cuda.graph(graph):
        now = torch.cuda.current_stream().cuda_stream
        cache.attend(q, c.k, c.v, c.table, c.lengths, out, stream=now, **tracked)
        cache.evict(c.k, c.v, c.table, c.lengths, c.tokens, c.weights, c.positions, 200, recent=10, stream=now)
        gpu_backend.token_log_probs(logits, tokens, **again, stream=now)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    _within(out, want, bound, "in a graph")
    assert c.lengths.tolist() == [200, 41]
    assert all(torch.equal(again[n], scored[n]) for n in scored)
    c.lengths.copy_(torch.tensor([300, 41]))
    # the second replay sees the rows that the first one left in front
    graph.replay()
    torch.cuda.synchronize()
    assert c.lengths.tolist() == [200, 41] and all(torch.equal(again[n], scored[n]) for n in scored)


@pytest.mark.gpu
def test_a_cache_dropped_during_a_capture_does_not_end_it(gpu_backend):
    import torch

    in_use = lambda: gpu_backend.memory_stats()["bytes_in_use"]
    gc.collect()  # buffers that other tests have left
    gpu_backend.synchronize()
    before = in_use()
    cache = gpu_backend.paged_cache(P.BF16_CODE, 4, 8, 2, 64, 16, 100, track=True)
    held = in_use() - before
    assert held > 0
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        del cache
        x += 1
    graph.replay()
    assert x.tolist() == [2.0] * 8
    assert in_use() == before + held
    gpu_backend.synchronize()
    assert in_use() == before


@pytest.mark.gpu
def test_two_caches_on_two_streams(gpu_backend):
    import torch

    cases = [_Case("bf16", 32, 8, 128, 16, [3000 - 100 * i, 500], seed=i) for i in range(2)]
    handles, streams = [c.handle(gpu_backend) for c in cases], [torch.cuda.Stream() for _ in cases]
    qs = [c.randn(2, 32, 128) for c in cases]
    outs = [[torch.empty_like(q) for _ in range(8)] for q in qs]
    torch.cuda.synchronize()
    for i in range(8):
        for c, h, s, q, o in zip(cases, handles, streams, qs, outs):
            h.attend(q, c.k, c.v, c.table, c.lengths, o[i], stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c, q, o in zip(cases, qs, outs):
        want, _, _, bound, _, _ = c.attention(q)
        _within(o[0], want, bound, "out")
        assert all(torch.equal(o[0], x) for x in o[1:])
