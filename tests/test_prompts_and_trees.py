"""Packed prompts, trees of drafted tokens, page tables and slots against plain 64-bit forms and lists.

Tolerances follow from the arithmetic. A score is a sum of head_dim products in f32, off by at most
(head_dim + 16) * 2^-24 * sum |q k| * |scale| =: e. A probability is off by the factor e twice (its own score's and those of the sum) and
by 2^-17 for the exponential; in 16 bits it is rounded to the type (h = half a step) before it meets the values, but not in the sum, so a
weight is off by h more (2h are allowed), and the log-sum-exp by none of it. f16 holds probabilities below 2^-25 of the largest to multiples of 2^-35 only, half of which a key may lose. A
result is rounded once. What a row does not see must not enter at all, whatever it holds.
"""
import math

import numpy as np
import pytest

from pjrtx_b200 import backend as be_mod
from pjrtx_b200 import operators as ops
from pjrtx_b200 import plan as P
from tests.test_operators import CODE, GEOMETRY, _Array, _Case, _host_cache, _Placed, _stream, _torch_type, _within

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PROBABILITY = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of what a probability is held in
LEAST = {"f32": 0.0, "f16": 2.0 ** -36, "bf16": 0.0}              # what a key's probability may lose besides
SUBNORMAL = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _expected(dtype, q, k, v, scale):
    """One query row [d] over the keys it sees: result, log-sum-exp and their bounds."""
    import torch

    q, k, v = q.double(), k.double(), v.double()
    s = (k @ q) * scale
    e = float((k.abs() @ q.abs()).max()) * abs(scale) * (q.numel() + 16) * 2.0 ** -24
    p, lse = torch.softmax(s, 0), torch.logsumexp(s, 0)
    out = p @ v
    bound = (2 * e + 2.0 ** -17 + 2 * PROBABILITY[dtype]) * (p @ v.abs()) + LEAST[dtype] * v.abs().sum(0)
    bound = bound + HALF_STEP[dtype] * (out.abs() + bound) + SUBNORMAL[dtype]
    return out, lse, bound, e + 2.0 ** -17 + 2.0 ** -20 * (1 + abs(float(lse)))


class _Compared:
    """Collects rows and compares them at once."""

    def __init__(self):
        self.got, self.want, self.bound, self.lse, self.want_lse, self.lse_bound = ([] for _ in range(6))

    def add(self, dtype, out, lse, q, k, v, scale):
        w, l, b, lb = _expected(dtype, q, k, v, scale)
        for to, x in zip((self.got, self.want, self.bound, self.lse, self.want_lse, self.lse_bound), (out, w, b, lse, l, lb)):
            to.append(x)

    def check(self, what):
        import torch

        _within(torch.stack(self.got), torch.stack(self.want), torch.stack(self.bound), what)
        _within(torch.stack(self.lse), torch.stack(self.want_lse), torch.tensor(self.lse_bound, dtype=torch.float64), what + " lse")


# ---- packed prompts ------------------------------------------------------------------------------------------------


class _Prompts:
    def __init__(self, dtype, heads, kv_heads, head_dim, lengths, seed=0, front=0, behind=3):
        import torch

        self.torch, self.dtype, self.heads, self.kv_heads, self.head_dim, self.lengths = torch, dtype, heads, kv_heads, head_dim, list(lengths)
        gen = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.ends = np.cumsum([front] + self.lengths).tolist()
        self.tokens = self.ends[-1] + behind
        packed = torch.randn((self.tokens, heads + 2 * kv_heads, head_dim), generator=gen, device="cuda").to(_torch_type(dtype))
        packed[:, :heads] *= 2
        packed[:front], packed[self.ends[-1]:] = math.nan, math.nan  # rows of no sequence
        self.q, self.k, self.v = packed[:, :heads], packed[:, heads:heads + kv_heads], packed[:, heads + kv_heads:]
        self.starts = torch.tensor(self.ends, dtype=torch.int32, device="cuda")
        self.out = torch.full((self.tokens, heads, head_dim), 7.0, dtype=packed.dtype, device="cuda")
        self.lse = torch.full((self.tokens, heads), 7.0, device="cuda")

    def run(self, be, **more):
        be.prompt_attention(self.q, self.k, self.v, self.starts, self.out, **{"lse": self.lse, "stream": _stream(), **more})

    def check(self, scale=None, some=None, what="prompt", skip=()):
        """All rows of all heads, or `some` of them."""
        torch, rep = self.torch, self.heads // self.kv_heads
        scale = self.head_dim ** -0.5 if scale is None else scale
        c = _Compared()
        rows = [(b, i, h) for b, n in enumerate(self.lengths) if b not in skip for i in range(n) for h in range(self.heads)]
        if some and len(rows) > some:
            rng = np.random.default_rng(1)
            rows = [rows[j] for j in sorted(set(rng.integers(0, len(rows), some).tolist()) | {0, len(rows) - 1})]
        for b, i, h in rows:
            a = self.ends[b]
            c.add(self.dtype, self.out[a + i, h], self.lse[a + i, h], self.q[a + i, h], self.k[a:a + i + 1, h // rep], self.v[a:a + i + 1, h // rep], scale)
        if rows:
            c.check(what)
        assert (self.out[:self.ends[0]] == 7).all() and (self.out[self.ends[-1]:] == 7).all()
        assert (self.lse[:self.ends[0]] == 7).all() and (self.lse[self.ends[-1]:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", GEOMETRY + [(1, 1, 8), (3, 1, 24), (130, 1, 64), (7, 7, 72), (70, 1, 200)])
def test_prompts_over_lengths_and_heads(gpu_backend, dtype, heads, kv_heads, head_dim):
    p = _Prompts(dtype, heads, kv_heads, head_dim, [1, 0, 2, 33, 64, 65, 0, 129, 300], seed=heads + head_dim, front=2)
    p.run(gpu_backend)
    p.check(some=1500)
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths", [[1], [127], [128], [2500], [700, 1, 1025, 0], [3] * 300, [0, 0, 5], [40] * 33, [255, 256, 257, 511, 513]])
def test_prompts_of_many_lengths(gpu_backend, dtype, lengths):
    p = _Prompts(dtype, 8, 2, 128, lengths, seed=len(lengths))
    p.run(gpu_backend, scale=0.11)
    p.check(0.11, some=1200)
    first = p.out.clone()
    p.run(gpu_backend, scale=0.11, lse=None)
    assert p.torch.equal(first, p.out)  # the same bits again, and lse is not needed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_prompts_of_any_layout_and_scale(gpu_backend, dtype, scale):
    p = _Prompts(dtype, 6, 2, 64, [70, 5, 200], seed=3, behind=0)
    torch = p.torch
    p.q, p.k = p.q.permute(1, 0, 2).contiguous().permute(1, 0, 2), p.k.contiguous()
    wide = torch.zeros((p.tokens, 2, 80), dtype=p.v.dtype, device="cuda")
    wide[:, :, 8:72] = p.v
    p.v = wide[:, :, 8:72]
    p.out = torch.full((9, p.tokens, 64), 7.0, dtype=p.v.dtype, device="cuda")[1:7].permute(1, 0, 2)
    p.run(gpu_backend, scale=scale)
    p.check(scale, some=800)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_prompts_take_nothing_of_what_they_do_not_see(gpu_backend, dtype, heads, kv_heads, head_dim, value):
    """Infinities and NaN at a position enter the rows from there on, as the formula has it, and nothing before or in other sequences."""
    lengths, bad = [90, 300, 140], 130
    p = _Prompts(dtype, heads, kv_heads, head_dim, lengths, seed=9)
    a = p.ends[1]
    p.v[a + bad, :, 3] = value
    p.k[p.ends[2] + 100, 0] = math.nan
    p.run(gpu_backend)
    rep, c = heads // kv_heads, _Compared()
    for b, i in [(0, 89), (0, 5), (1, 0), (1, 64), (1, 127), (1, 128), (1, 129), (2, 0), (2, 63), (2, 99)]:
        for h in range(heads):
            r = p.ends[b]
            c.add(dtype, p.out[r + i, h], p.lse[r + i, h], p.q[r + i, h], p.k[r:r + i + 1, h // rep], p.v[r:r + i + 1, h // rep], head_dim ** -0.5)
    c.check("rows that do not see it")
    from_there = p.out[a + bad:p.ends[2]].float()
    assert (from_there[:, :, 3].isnan().all() if math.isnan(value) else (from_there[:, :, 3] == value).all())
    finite = [d for d in range(head_dim) if d != 3]
    assert from_there[:, :, finite].isfinite().all()
    c = _Compared()
    p.v[a + bad, :, 3] = 0  # the other dimensions do not depend on it
    for i in (bad, bad + 1, 299):
        for h in range(heads):
            w, l, bound, _ = _expected(dtype, p.q[a + i, h], p.k[a:a + i + 1, h // rep], p.v[a:a + i + 1, h // rep], head_dim ** -0.5)
            _within(p.out[a + i, h][finite], w[finite], bound[finite], "beside it")
    blind = p.out[p.ends[2] + 100:p.ends[3], :rep]
    assert blind.isnan().all() and p.lse[p.ends[2] + 100:p.ends[3], :rep].isnan().all()
    if kv_heads > 1:
        assert p.out[p.ends[2]:p.ends[3], rep:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_prompts_with_scores_far_apart(gpu_backend, dtype):
    p = _Prompts(dtype, 4, 2, 64, [400, 257], seed=5)
    p.q *= 12
    p.k[p.ends[0]:p.ends[0] + 200, :, 0] *= 20
    p.k[p.ends[1]:p.ends[2]] = p.k[p.ends[1]:p.ends[1] + 1]  # equal scores
    p.run(gpu_backend)
    p.check(some=900)


@pytest.mark.gpu
def test_prompts_that_see_only_scores_of_minus_infinity(gpu_backend):
    p = _Prompts("bf16", 2, 1, 64, [150], seed=6)
    p.q[:, :, 0] = 1
    p.k[:100, :, 0] = -math.inf  # the first hundred rows see nothing else
    p.run(gpu_backend)
    assert (p.out[:100] == 0).all() and (p.lse[:100] == -math.inf).all()
    c = _Compared()
    for i in (100, 149):
        c.add("bf16", p.out[i, 1], p.lse[i, 1], p.q[i, 1], p.k[100:i + 1, 0], p.v[100:i + 1, 0], 0.125)
    c.check("rows behind them")


@pytest.mark.gpu
@pytest.mark.parametrize("starts,held", [([0, 50, 40, 100], ()), ([-3, 50, 100, 120], (1, 2)), ([0, 50, 100, 10 ** 6], (0, 1))])
def test_starts_out_of_range_are_reported_and_not_followed(gpu_backend, starts, held):
    """Sequences that lie where they may are computed; where starts descend, rows belong to two sequences and their results are open."""
    p = _Prompts("bf16", 4, 2, 64, [120], seed=8)
    p.starts = p.torch.tensor(starts, dtype=p.torch.int32, device="cuda")
    p.run(gpu_backend)
    with pytest.raises(be_mod.BackendError, match="code 41"):
        gpu_backend.operators_status(stream=_stream())
    c = _Compared()
    for b in held:
        for i in range(starts[b], starts[b + 1], 7):
            c.add("bf16", p.out[i, 3], p.lse[i, 3], p.q[i, 3], p.k[starts[b]:i + 1, 1], p.v[starts[b]:i + 1, 1], 0.125)
    if held:
        c.check("the other sequences")
    assert held or (p.out[100:] == 7).all()  # rows of no sequence stay


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_offsets_beyond_32_bits(gpu_backend, dtype):
    import torch

    p = _Prompts(dtype, 2, 1, 64, [2, 3], seed=4, behind=0)
    stride = (1 << 29) + 64
    flat = torch.empty(4 * stride + 128, dtype=p.q.dtype, device="cuda")
    dense = p.q
    p.q = flat.as_strided(tuple(dense.shape), (stride, 64, 1))
    p.q.copy_(dense)
    p.run(gpu_backend)
    p.check()
    p.q, p.out = dense, flat.as_strided(tuple(p.out.shape), (stride, 64, 1))
    p.run(gpu_backend)
    p.check()
    for name in ("k", "v"):
        dense, spread = getattr(p, name), flat.as_strided(tuple(p.k.shape), (stride, 64, 1))
        spread.copy_(dense)
        setattr(p, name, spread)
        p.out = torch.empty(tuple(p.out.shape), dtype=p.out.dtype, device="cuda")
        p.run(gpu_backend)
        p.check()
        setattr(p, name, dense)


@pytest.mark.gpu
def test_prompts_of_no_tokens_and_no_sequences(gpu_backend):
    p = _Prompts("bf16", 4, 2, 64, [20], seed=8)
    p.starts = p.torch.zeros(1, dtype=p.torch.int32, device="cuda")
    p.run(gpu_backend)
    assert (p.out == 7).all()
    q = p.torch.empty((0, 4, 64), dtype=p.torch.bfloat16, device="cuda")
    gpu_backend.prompt_attention(q, q[:, :2], q[:, :2], p.starts, q, stream=_stream())
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
def test_prompts_and_trees_on_other_streams_and_in_graphs(gpu_backend):
    import torch

    p = _Prompts("bf16", 8, 2, 128, [300, 5, 77], seed=2)
    t = _Trees("bf16", 8, 2, 128, 16, [300, 0, 5], 12, seed=2)
    t.cache = t.case.handle_of_tree(gpu_backend)
    p.run(gpu_backend)
    t.run(gpu_backend)
    torch.cuda.synchronize()
    first = p.out.clone(), t.out.clone()
    p.out.fill_(7), t.out.fill_(7)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        p.run(gpu_backend)
        t.run(gpu_backend)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first[0], p.out) and torch.equal(first[1], t.out)
    # other lengths in the same graph
    p.starts.copy_(torch.tensor([0, 200, 200, 382], dtype=torch.int32))
    p.ends, p.lengths = [0, 200, 200, 382], [200, 0, 182]
    t.counts.copy_(torch.tensor([3, 12, 1], dtype=torch.int32))
    t.out.fill_(7), t.lse.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    p.check(some=300)
    t.counts_list = [3, 12, 1]
    t.check(some=300)


def _prompt_args(**change):
    a = dict(q=_Array("bfloat16", 9, 8, 64), k=_Array("bfloat16", 9, 2, 64), v=_Array("bfloat16", 9, 2, 64), starts=_Array("int32", 3),
             out=_Array("bfloat16", 9, 8, 64), lse=_Array("float32", 9, 8))
    a.update(change)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(q=_Array("int32", 9, 8, 64)), "element type s32"), (dict(q=_Array("bfloat16", 9, 8)), "q has shape"),
    (dict(k=_Array("bfloat16", 8, 2, 64)), "k has shape"), (dict(k=_Array("bfloat16", 9, 2, 32)), "k has shape"),
    (dict(v=_Array("bfloat16", 9, 4, 64)), "v has shape"), (dict(v=_Array("float16", 9, 2, 64)), "v has element type"),
    (dict(out=_Array("float32", 9, 8, 64)), "out has element type"), (dict(lse=_Array("float32", 9, 2)), "lse has shape"),
    (dict(starts=_Array("int64", 3)), "starts has element type"), (dict(starts=_Array("int32", 0)), "starts has shape"),
    (dict(starts=_Array("int32", 3, 1)), "starts has shape"), (dict(k=_Array("bfloat16", 9, 3, 64), v=_Array("bfloat16", 9, 3, 64)), "3 KV heads"),
    (dict(q=_Array("bfloat16", 9, 8, 64, strides=(512, 1, 8))), "dense"), (dict(q=_Array("bfloat16", 9, 8, 64, strides=(516, 64, 1))), "aligned"),
    (dict(out=_Array("bfloat16", 9, 8, 64, pointer=(1 << 20) + 8)), "aligned"), (dict(starts=_Array("int32", 3, pointer=0)), "null starts"),
    (dict(scale=math.nan), "not finite"), (dict(scale=math.inf), "not finite"),
    (dict(q=_Array("bfloat16", 9, 8, 60), k=_Array("bfloat16", 9, 2, 60), v=_Array("bfloat16", 9, 2, 60), out=_Array("bfloat16", 9, 8, 60)), "head dimension 60"),
    (dict(q=_Array("bfloat16", 9, 8, 264), k=_Array("bfloat16", 9, 2, 264), v=_Array("bfloat16", 9, 2, 264), out=_Array("bfloat16", 9, 8, 264)),
     "head dimension 264"), (dict(starts=_Array("int32", (1 << 20) + 2)), "sequences")])
def test_prompt_attention_refuses(backend, change, message):
    with pytest.raises(be_mod.BackendError, match=message):
        backend.prompt_attention(**_prompt_args(**change), stream=0)


@pytest.mark.parametrize("taken", ["q", "k", "v"])
def test_prompt_results_do_not_take_the_place_of_an_input(backend, taken):
    place = dict(q=2 << 20, k=3 << 20, v=4 << 20, out=5 << 20)
    place["out"] = place[taken]
    change = {n: _Array("bfloat16", 9, 2 if n in "kv" else 8, 64, pointer=at) for n, at in place.items()}
    with pytest.raises(be_mod.BackendError, match="can not take the place of an input"):
        backend.prompt_attention(**_prompt_args(**change), stream=0)


def test_prompt_structs_without_size_are_refused(backend):
    import ctypes

    lib = backend.lib
    assert not lib.pjrtx_b200_prompt_attention(0, None, None) and b"null argument" in lib.pjrtx_b200_last_error()
    assert not lib.pjrtx_b200_prompt_attention(0, ctypes.byref(ops.PromptAttentionArgs(8)), None) and b"struct_size" in lib.pjrtx_b200_last_error()
    for call in (lib.pjrtx_b200_paged_cache_attend_tree, lib.pjrtx_b200_paged_cache_store):
        assert not call(None, None, None, None) and b"null paged cache" in lib.pjrtx_b200_last_error()
    for call in (lib.pjrtx_b200_paged_cache_assign, lib.pjrtx_b200_paged_cache_path_slots):
        assert not call(None, None, None) and b"null paged cache" in lib.pjrtx_b200_last_error()


@pytest.mark.parametrize("says", ["get_device", "device"])
@pytest.mark.parametrize("where,message", [(-1, "on the host, device 1"), (0, "on device 0, device 1")])
def test_arrays_of_the_host_and_of_other_devices_are_refused(backend, where, message, says):
    def check(call, good):
        place = lambda at, a: _Placed(at, a, says)
        for name in good:
            if isinstance(good[name], _Array):
                with pytest.raises(be_mod.BackendError, match=f"{name} is {message}"):
                    call(**{n: place(where if n == name else 1, a) if isinstance(a, _Array) else a for n, a in good.items()}, stream=0)

    check(backend.prompt_attention, dict(_prompt_args(), device=1))
    cache = _host_cache()
    pools = dict(k_pages=_Array("bfloat16", 9, 16, 4, 64), v_pages=_Array("bfloat16", 9, 16, 4, 64))
    table = dict(page_table=_Array("int32", 2, 4), lengths=_Array("int32", 2))
    tree = dict(q=_Array("bfloat16", 2, 5, 8, 64), out=_Array("bfloat16", 2, 5, 8, 64), lse=_Array("float32", 2, 5, 8),
                k_new=_Array("bfloat16", 2, 5, 4, 64), v_new=_Array("bfloat16", 2, 5, 4, 64), parents=_Array("int32", 2, 5), counts=_Array("int32", 2))
    check(cache.attend_tree, dict(pools, **table, **tree))
    check(cache.store, dict(pools, k_new=_Array("bfloat16", 7, 4, 64), v_new=_Array("bfloat16", 7, 4, 64), slots=_Array("int32", 7)))
    assign = dict(table, held=_Array("int32", 2), free_pages=_Array("int32", 9), free_count=_Array("int32", 1), starts=_Array("int32", 3),
                  slots=_Array("int32", 7))
    check(cache.assign_pages, dict(assign, held_out=_Array("int32", 2), page_table_out=_Array("int32", 2, 4), free_pages_out=_Array("int32", 9),
                                   free_count_out=_Array("int32", 1)))
    check(cache.path_slots, dict(table, parents=_Array("int32", 2, 5), leaves=_Array("int32", 2), slots=_Array("int32", 2, 5),
                                 lengths_out=_Array("int32", 2)))


# ---- trees ---------------------------------------------------------------------------------------------------------


def _random_parents(rng, batch, nodes, chain=False):
    if chain:
        return np.tile(np.arange(nodes) - 1, (batch, 1))
    return np.array([[int(rng.integers(-1, i)) if i and rng.random() < 0.9 else -1 for i in range(nodes)] for _ in range(batch)])


def _way(parents, node):
    """Ancestors of a node and itself, root first."""
    way = []
    while node >= 0:
        way.insert(0, node)
        node = parents[node]
    return way


class _Trees:
    def __init__(self, dtype, heads, kv_heads, head_dim, page, lengths, nodes, seed=0, chain=False, layout="nhd", counts=None):
        self.case = case = _Case(dtype, heads, kv_heads, head_dim, page, lengths, seed=seed, layout=layout)
        case.handle_of_tree = lambda be: be.paged_cache(CODE[dtype], len(lengths) + 1, heads, kv_heads, head_dim, page, case.max_pages, tree=nodes)
        self.torch, self.dtype, self.nodes, rng = case.torch, dtype, nodes, np.random.default_rng(seed)
        batch = len(lengths)
        packed = case.randn(batch, nodes, heads + 2 * kv_heads, head_dim)
        packed[:, :, :heads] *= 2
        self.q, self.k, self.v = packed[:, :, :heads], packed[:, :, heads:heads + kv_heads], packed[:, :, heads + kv_heads:]
        self.parents_list = _random_parents(rng, batch, nodes, chain).tolist()
        self.counts_list = counts if counts is not None else [int(rng.integers(0, nodes + 1)) if i % 3 == 1 else nodes for i in range(batch)]
        for b, n in enumerate(self.counts_list):
            packed[b, n:] = math.nan
        as_ints = lambda x: self.torch.tensor(x, dtype=self.torch.int32, device="cuda")
        self.parents, self.counts = as_ints(self.parents_list), as_ints(self.counts_list)
        self.out = self.torch.full((batch, nodes, heads, head_dim), 7.0, dtype=packed.dtype, device="cuda")
        self.lse = self.torch.full((batch, nodes, heads), 7.0, device="cuda")
        self.cache = None

    def run(self, be, **more):
        c = self.case
        self.cache = self.cache or c.handle_of_tree(be)
        self.cache.attend_tree(self.q, c.k, c.v, c.table, c.lengths, self.out, self.k, self.v, self.parents,
                               **{"counts": self.counts, "lse": self.lse, "stream": _stream(), **more})

    def seen(self, b, i, g):
        """Keys and values that node i sees."""
        c, way = self.case, _way(self.parents_list[b], i)
        pg, row = c.places(b, c.lengths_list[b])
        return tuple(self.torch.cat([pool[pg, row, g], new[b, way, g]]) for pool, new in ((c.k, self.k), (c.v, self.v)))

    def check(self, scale=None, some=None, what="tree", skip=()):
        c = self.case
        rep, scale = c.heads // c.kv_heads, c.head_dim ** -0.5 if scale is None else scale
        rows = [(b, i, h) for b, n in enumerate(self.counts_list) if b not in skip for i in range(n) for h in range(c.heads)]
        if some and len(rows) > some:
            rng = np.random.default_rng(1)
            rows = [rows[j] for j in sorted(set(rng.integers(0, len(rows), some).tolist()) | {0, len(rows) - 1})]
        compared = _Compared()
        for b, i, h in rows:
            k, v = self.seen(b, i, h // rep)
            compared.add(self.dtype, self.out[b, i, h], self.lse[b, i, h], self.q[b, i, h], k, v, scale)
        if rows:
            compared.check(what)
        for b, n in enumerate(self.counts_list):
            assert (self.out[b, n:] == 7).all() and (self.lse[b, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", GEOMETRY + [(1, 1, 8), (130, 1, 64), (7, 7, 72), (70, 1, 200)])
@pytest.mark.parametrize("nodes", [1, 7, 64])
def test_trees_over_lengths_and_heads(gpu_backend, dtype, heads, kv_heads, head_dim, nodes):
    t = _Trees(dtype, heads, kv_heads, head_dim, 16, [1, 0, 63, 64, 65, 128, 300, 2], nodes, seed=heads + head_dim + nodes)
    t.run(gpu_backend)
    t.check(some=700)
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,nodes,chain", [([5000], 64, True), ([9000], 5, False), ([5000, 0, 1, 777], 33, False), ([64] * 40, 3, False),
                                                 ([0], 64, False), ([130, 20000], 17, True)])
def test_trees_of_many_lengths(gpu_backend, dtype, lengths, nodes, chain):
    t = _Trees(dtype, 16, 4, 128, 16, lengths, nodes, seed=len(lengths), chain=chain)
    t.run(gpu_backend, scale=0.09)
    t.check(0.09, some=500)
    first = t.out.clone()
    t.run(gpu_backend, scale=0.09, lse=None)
    assert t.torch.equal(first, t.out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,layout", [(1, "nhd"), (5, "hnd"), (7, "nhd"), (48, "nhd"), (128, "hnd"), (1000, "nhd")])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_trees_on_pages_of_any_size_and_layout(gpu_backend, dtype, page, layout, scale):
    t = _Trees(dtype, 8, 2, 64, page, [257, 3, 1000, 999], 9, seed=page, layout=layout)
    t.q = t.q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    t.out = t.torch.full((9, 4, 8, 64), 7.0, dtype=t.q.dtype, device="cuda").permute(1, 0, 2, 3)
    t.run(gpu_backend, scale=scale)
    t.check(scale, some=500)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_trees_take_nothing_of_what_they_do_not_see(gpu_backend, dtype, heads, kv_heads, head_dim, value):
    t = _Trees(dtype, heads, kv_heads, head_dim, 16, [100, 400], 20, seed=9, counts=[20, 20])
    t.v[:, 6, :, 3] = value
    t.k[:, 9, 0] = math.nan
    t.run(gpu_backend)
    rep, c = heads // kv_heads, _Compared()
    sees = {n: [n in _way(t.parents_list[b], i) for b in range(2) for i in range(20)] for n in (6, 9)}
    for b in range(2):
        for i in range(20):
            for h in range(heads):
                if not sees[6][b * 20 + i] and not (sees[9][b * 20 + i] and h < rep):
                    k, v = t.seen(b, i, h // rep)
                    c.add(dtype, t.out[b, i, h], t.lse[b, i, h], t.q[b, i, h], k, v, head_dim ** -0.5)
    c.check("nodes that do not see it")
    for j, (out, lse) in enumerate(zip(t.out.flatten(0, 1).float(), t.lse.flatten(0, 1))):
        if sees[9][j]:
            assert out[:rep].isnan().all() and lse[:rep].isnan().all()
        elif sees[6][j]:
            assert out[:, 3].isnan().all() if math.isnan(value) else (out[:, 3] == value).all()
            assert out[:, :3].isfinite().all() and out[:, 4:].isfinite().all()


@pytest.mark.gpu
def test_tree_pages_lengths_counts_and_parents_out_of_range_are_reported(gpu_backend):
    t = _Trees("bf16", 4, 2, 64, 16, [40, 40, 40], 6, seed=9, counts=[6, 6, 6])
    c, torch = t.case, t.torch
    good = c.table, c.lengths, t.parents
    def reported(message):
        t.out.fill_(7), t.lse.fill_(7)
        t.run(gpu_backend)
        with pytest.raises(be_mod.BackendError, match=message):
            gpu_backend.operators_status(stream=_stream())
        t.check(some=200, skip=(1,), what="the other sequences")
        c.table, c.lengths, t.parents = good
    for entry in (-1, 10 ** 6):
        c.table = c.table.clone()
        c.table[1, 1] = entry
        reported("code 40")
    for n in (-5, 49):
        c.lengths, c.table = c.lengths.clone(), c.table.clone()
        c.lengths[1], c.table[1, 2] = n, 0
        reported("code 41")
    for n in (-1, 7):
        t.counts[1] = n
        reported("code 41")
    t.counts[1] = 6
    for node, parent in ((2, 2), (3, 5), (0, 0), (4, -2), (5, 1 << 30)):
        t.parents = t.parents.clone()
        t.parents[1, node] = parent
        was = t.parents_list[1][node]
        t.parents_list[1][node] = -1  # what it counts as
        t.out.fill_(7), t.lse.fill_(7)
        t.run(gpu_backend)
        with pytest.raises(be_mod.BackendError, match="code 43"):
            gpu_backend.operators_status(stream=_stream())
        t.check(some=300)
        t.parents, t.parents_list[1][node] = good[2], was
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tree_offsets_beyond_32_bits(gpu_backend, dtype):
    import torch

    t = _Trees(dtype, 4, 1, 64, 16, [45], 5, seed=3, counts=[5])
    c, stride = t.case, (1 << 30) + 64
    for name in ("k", "v"):
        flat = torch.empty((c.k.shape[0] - 1) * stride + 16 * 64, dtype=t.q.dtype, device="cuda")
        pool = flat.as_strided(tuple(c.k.shape), (stride, 64, 64, 1))
        pool.copy_(getattr(c, name))
        setattr(c, name, pool)
    t.run(gpu_backend)
    t.check()
    # the same rows by their slots
    new = torch.randn((3, 1, 64), device="cuda").to(t.q.dtype)
    last = c.k.shape[0] - 1
    t.cache.store(c.k, c.v, new, new * 2, torch.tensor([last * 16 + 15, -1, 16], dtype=torch.int32, device="cuda"), stream=_stream())
    assert torch.equal(c.k[last, 15], new[0]) and torch.equal(c.v[1, 0], new[2] * 2)


@pytest.mark.gpu
def test_one_tree_handle_serves_batches_and_trees_of_different_sizes(gpu_backend):
    big = _Trees("bf16", 8, 2, 128, 16, [700, 1500, 3, 90], 40, seed=1)
    cache = gpu_backend.paged_cache(CODE["bf16"], 9, 8, 2, 128, 16, big.case.max_pages, tree=64)
    for lengths, nodes in (([700, 1500, 3, 90], 40), ([1400], 1), ([5], 64), ([0] * 9, 2), ([1500] * 3, 9)):
        t = _Trees("bf16", 8, 2, 128, 16, lengths, nodes, seed=nodes)
        t.case.table = t.torch.nn.functional.pad(t.case.table, (0, big.case.max_pages - t.case.table.shape[1]), value=-1).contiguous()
        t.cache = cache
        t.run(gpu_backend)
        t.check(some=150)


@pytest.mark.gpu
def test_tree_calls_refuse_bad_arguments(gpu_backend):
    cache = gpu_backend.paged_cache(P.BF16_CODE, 2, 8, 4, 64, 16, 4, tree=8)
    plain = gpu_backend.paged_cache(P.BF16_CODE, 2, 8, 4, 64, 16, 4)

    def base(batch=2, nodes=5):
        return dict(k_pages=_Array("bfloat16", 9, 16, 4, 64), v_pages=_Array("bfloat16", 9, 16, 4, 64), page_table=_Array("int32", batch, 4),
                    lengths=_Array("int32", batch), q=_Array("bfloat16", batch, nodes, 8, 64), out=_Array("bfloat16", batch, nodes, 8, 64),
                    k_new=_Array("bfloat16", batch, nodes, 4, 64), v_new=_Array("bfloat16", batch, nodes, 4, 64), parents=_Array("int32", batch, nodes))

    def refused(call, message, good, **change):
        with pytest.raises(be_mod.BackendError, match=message):
            call(**{**good, **change}, stream=0)

    tree = cache.attend_tree
    refused(tree, "9 nodes, the cache was made for up to 8", base(nodes=9))
    refused(plain.attend_tree, "5 nodes, the cache was made for up to 0", base())
    refused(tree, "a batch of 3", base(batch=3))
    refused(tree, "parents has shape", base(), parents=_Array("int32", 3, 5))
    refused(tree, "parents has element type", base(), parents=_Array("int64", 2, 5))
    refused(tree, "q has shape", base(), q=_Array("bfloat16", 2, 4, 8, 64))
    refused(tree, "out has element type", base(), out=_Array("float16", 2, 5, 8, 64))
    refused(tree, "lse has shape", base(), lse=_Array("float32", 2, 5, 4))
    refused(tree, "counts has shape", base(), counts=_Array("int32", 5))
    refused(tree, "differ", base(), v_new=_Array("bfloat16", 2, 5, 2, 64))
    refused(tree, "16-byte aligned", base(), q=_Array("bfloat16", 2, 5, 8, 64, strides=(2560, 515, 64, 1)))
    refused(tree, "16-byte aligned", base(), k_new=_Array("bfloat16", 2, 5, 4, 64, pointer=(1 << 20) + 2))
    refused(tree, "null parents", base(), parents=_Array("int32", 2, 5, pointer=0))
    refused(tree, "not finite", base(), scale=math.nan)
    for taken, shape in (("q", (2, 5, 8, 64)), ("k_new", (2, 5, 4, 64)), ("v_new", (2, 5, 4, 64))):
        refused(tree, "can not take the place of an input", base(), **{taken: _Array("bfloat16", *shape, pointer=2 << 20)},
                out=_Array("bfloat16", 2, 5, 8, 64, pointer=2 << 20))
    store = dict(k_pages=_Array("bfloat16", 9, 16, 4, 64), v_pages=_Array("bfloat16", 9, 16, 4, 64), k_new=_Array("bfloat16", 7, 4, 64),
                 v_new=_Array("bfloat16", 7, 4, 64), slots=_Array("int32", 7))
    refused(cache.store, "slots has shape", store, slots=_Array("int32", 6))
    refused(cache.store, "k_new has shape", store, k_new=_Array("bfloat16", 7, 2, 64))
    refused(cache.store, "k_pages has shape", store, k_pages=_Array("bfloat16", 9, 8, 4, 64))
    refused(cache.store, "null slots", store, slots=_Array("int32", 7, pointer=0))
    refused(cache.store, "aligned", store, k_new=_Array("bfloat16", 7, 4, 64, strides=(300, 64, 1)), v_new=_Array("bfloat16", 7, 4, 64, strides=(300, 64, 1)))
    huge = (1 << 27) + 1
    refused(cache.store, "slots have 32 bits", store, k_pages=_Array("bfloat16", huge, 16, 4, 64), v_pages=_Array("bfloat16", huge, 16, 4, 64))
    assign = dict(lengths=_Array("int32", 2), held=_Array("int32", 2), page_table=_Array("int32", 2, 4), free_pages=_Array("int32", 9),
                  free_count=_Array("int32", 1))
    refused(cache.assign_pages, "slots need the starts", assign, slots=_Array("int32", 7))
    refused(cache.assign_pages, "held has shape", assign, held=_Array("int32", 3))
    refused(cache.assign_pages, "free_count has shape", assign, free_count=_Array("int32", 2))
    refused(cache.assign_pages, "free_pages has shape", assign, free_pages=_Array("int32", 9, 1))
    refused(cache.assign_pages, "page_table has shape", assign, page_table=_Array("int32", 2, 5))
    refused(cache.assign_pages, "starts has shape", assign, slots=_Array("int32", 7), starts=_Array("int32", 2))
    refused(cache.assign_pages, "up to 2.31 - 1 rows", assign, free_pages=_Array("int32", huge))
    refused(cache.assign_pages, "0 pages", assign, free_pages=_Array("int32", 0))
    refused(cache.assign_pages, "null stack", assign, free_count=_Array("int32", 1, pointer=0))
    refused(cache.assign_pages, "a batch of 3", dict(assign, lengths=_Array("int32", 3), held=_Array("int32", 3), page_table=_Array("int32", 3, 4)))
    path = dict(page_table=_Array("int32", 2, 4), lengths=_Array("int32", 2), parents=_Array("int32", 2, 5), leaves=_Array("int32", 2),
                slots=_Array("int32", 2, 5))
    refused(cache.path_slots, "slots has shape", path, slots=_Array("int32", 2, 4))
    refused(cache.path_slots, "65 nodes", path, parents=_Array("int32", 2, 65), slots=_Array("int32", 2, 65))
    refused(cache.path_slots, "leaves has shape", path, leaves=_Array("int32", 3))
    refused(cache.path_slots, "null page table", path, leaves=_Array("int32", 2, pointer=0))
    for bad in (-1, 65):
        with pytest.raises(be_mod.BackendError, match=f"trees of {bad} nodes"):
            gpu_backend.paged_cache(P.BF16_CODE, 2, 8, 4, 64, 16, 4, tree=bad)
    cache.destroy()
    refused(cache.path_slots, "destroyed", path)


def test_a_cache_config_that_ends_before_the_trees_is_taken(backend):
    """What a program of an earlier header passes: refused for its element type, not for its size."""
    import ctypes

    lib, whole = backend.lib, ctypes.sizeof(ops.PagedCacheConfig)
    for size, message in ((whole - 8, b"element type"), (whole, b"element type"), (whole - 16, b"struct_size")):
        config = ops.PagedCacheConfig(size, P.S32, 0, 1, 1, 1, 64, 16, 1)
        assert not lib.pjrtx_b200_paged_cache_create(0, ctypes.byref(config)) and message in lib.pjrtx_b200_last_error()


# ---- page tables, slots, stored rows -------------------------------------------------------------------------------


def _assigned(lengths, held, table, free, page, max_pages):
    """The same by lists; lengths beyond the table leave a sequence as it is."""
    table, free, held = [list(r) for r in table], list(free), list(held)
    need = [-(-n // page) if 0 <= n <= page * max_pages else h for n, h in zip(lengths, held)]
    for b, n in enumerate(need):
        for c in range(n, held[b]):
            free.append(table[b][c])
            table[b][c] = -1
        held[b] = min(held[b], n)
    for b, n in enumerate(need):
        if n - held[b] > len(free):
            break
        for c in range(held[b], n):
            table[b][c] = free.pop()
        held[b] = n
    return held, table, free


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,max_pages,spare", [(1, 16, 40, 3), (7, 1, 9, 0), (8, 5, 30, 4), (33, 16, 12, -30), (600, 8, 50, -1000), (1000, 3, 7, 9),
                                                        (5, 16, 3000, 0), (9000, 4, 2, 0)])
def test_assign_pages(gpu_backend, batch, page, max_pages, spare, in_place):
    import torch

    rng = np.random.default_rng(batch + page)
    capacity = page * max_pages
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    pool, held = batch * max_pages + 5, rng.integers(0, max_pages + 1, batch)
    held[rng.random(batch) < 0.3] = 0
    pages = rng.permutation(pool)
    table = np.full((batch, max_pages), -1)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = pages[at:at + n]
        at += n
    cache = gpu_backend.paged_cache(P.BF16_CODE, batch, 2, 1, 8, page, max_pages)
    held, free = held.tolist(), pages[at:].tolist()
    for turn in range(4):
        lengths = rng.integers(0, capacity + 1, batch)
        kind = rng.random(batch)
        lengths = np.where(kind < 0.3, 0, np.where(kind < 0.6, np.minimum(capacity, np.asarray(held) * page + 1), lengths))
        if spare < 0 and turn % 2:
            free = free[:max(0, len(free) // 4)]
        new = [int(rng.integers(0, n + 1)) if rng.random() < 0.5 else min(1, int(n)) for n in lengths]
        starts = np.cumsum([2] + new)
        tokens = int(starts[-1]) + 5
        want_held, want_table, want_free = _assigned(lengths.tolist(), held, table.tolist(), free, page, max_pages)
        stack = np.full(pool, -1)
        stack[:len(free)] = free
        args = [ints(lengths), ints(held), ints(table), ints(stack), ints([len(free)])]
        was = [a.clone() for a in args]
        outs = {} if in_place else {n: torch.full_like(a, 77) for n, a in zip(("held_out", "page_table_out", "free_pages_out", "free_count_out"), args[1:])}
        slots = torch.full((tokens,), 77, dtype=torch.int32, device="cuda")
        cache.assign_pages(*args, starts=ints(starts), slots=slots, stream=_stream(), **outs)
        got = [x.cpu().numpy() for x in (args[1:] if in_place else outs.values())]
        assert got[0].tolist() == want_held and int(got[3][0]) == len(want_free)
        assert np.array_equal(got[1], np.asarray(want_table))
        assert got[2][:len(want_free)].tolist() == want_free and (got[2][len(want_free):] == -1).all()
        if not in_place:
            assert all(torch.equal(a, w) for a, w in zip(args, was))
        want_slots = np.full(tokens, -1)
        for b, m in enumerate(new):
            if want_held[b] * page >= lengths[b]:
                row = np.arange(lengths[b] - m, lengths[b])
                want_slots[starts[b]:starts[b] + m] = got[1][b, row // page] * page + row % page
        assert np.array_equal(slots.cpu().numpy(), want_slots)
        gpu_backend.operators_status(stream=_stream())
        held, table, free = got[0].tolist(), got[1], want_free
        if spare < 0:
            free = free + sorted(set(range(pool)) - set(free) - set(table[table >= 0].tolist()))[:100]
        have = set(table[table >= 0].tolist())
        assert len(have) == sum(held) and not have & set(free)  # no page in two places


@pytest.mark.gpu
def test_assign_pages_leaves_what_it_cannot_hold(gpu_backend):
    import torch

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.BF16_CODE, 4, 2, 1, 8, 4, 3)
    for lengths, held, want_held in (([4, 13, 5, 1], [0, 1, 0, 0], [1, 1, 2, 1]), ([4, -1, 5, 1], [0, 1, 0, 0], [1, 1, 2, 1]),
                                     ([4, 2, 5, 1], [0, 4, 0, 0], [1, 4, 2, 1]), ([4, 1 << 30, 5, 1], [0, 1, 0, 0], [1, 1, 2, 1])):
        table, h = ints([[-1, -1, -1], [9, -1, -1], [-1, -1, -1], [-1, -1, -1]]), ints(held)
        free, count, slots = ints([1, 2, 3, 4, 5, 6, 7, 8, 0, -1]), ints([8]), torch.full((4,), 77, dtype=torch.int32, device="cuda")
        cache.assign_pages(ints(lengths), h, table, free, count, starts=ints([0, 1, 2, 3, 4]), slots=slots, stream=_stream())
        with pytest.raises(be_mod.BackendError, match="code 41"):
            gpu_backend.operators_status(stream=_stream())
        assert h.tolist() == want_held and table.tolist() == [[8, -1, -1], [9, -1, -1], [7, 6, -1], [5, -1, -1]]
        assert int(count) == 4 and free.tolist()[:4] == [1, 2, 3, 4]
        # a token that its sequence has no row for, too
        assert slots.tolist()[0] == 35 and slots.tolist()[2:] == [24, 20] and (slots[1] == -1 or lengths[1] == 2)
    # a count of free pages that the stack cannot have: nothing is given or taken
    table, h, free, count = ints([[-1] * 3] * 4), ints([0] * 4), ints(list(range(10))), ints([11])
    cache.assign_pages(ints([1] * 4), h, table, free, count, stream=_stream())
    with pytest.raises(be_mod.BackendError, match="code 41"):
        gpu_backend.operators_status(stream=_stream())
    assert h.tolist() == [0] * 4 and (table == -1).all() and int(count) == 11 and free.tolist() == list(range(10))
    # a page of the stack that the pool does not have
    count, free = ints([2]), ints([3, 10] + [-1] * 8)
    cache.assign_pages(ints([1, 0, 0, 0]), h, table, free, count, starts=ints([0, 1, 1, 1, 1]), slots=slots, stream=_stream())
    with pytest.raises(be_mod.BackendError, match="code 40"):
        gpu_backend.operators_status(stream=_stream())
    assert slots.tolist() == [-1] * 4


@pytest.mark.gpu
def test_assign_pages_of_no_sequences(gpu_backend):
    import torch

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.BF16_CODE, 4, 2, 1, 8, 4, 3)
    empty, free, count = ints([]), ints([1, 2, -1]), ints([2])
    slots, out, count_out = ints([7, 7]), ints([0, 0, 0]), ints([0])
    cache.assign_pages(empty, empty, empty.reshape(0, 3), free, count, starts=ints([0]), slots=slots, free_pages_out=out, free_count_out=count_out,
                       stream=_stream())
    assert slots.tolist() == [-1, -1] and out.tolist() == [1, 2, -1] and int(count_out) == 2
    cache.path_slots(empty.reshape(0, 3), empty, empty.reshape(0, 5), empty, empty.reshape(0, 5), stream=_stream())
    pools = torch.zeros((2, 3, 4, 1, 8), device="cuda", dtype=torch.bfloat16)
    cache.store(pools[0], pools[1], pools[0, 0, :0], pools[1, 0, :0], empty, stream=_stream())
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,nodes,page", [(1, 1, 16), (5, 7, 3), (300, 64, 16), (33, 33, 1), (9, 32, 128)])
def test_path_slots(gpu_backend, batch, nodes, page, in_place):
    import torch

    rng = np.random.default_rng(batch)
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    lengths = rng.integers(0, 90, batch)
    max_pages = -(-(90 + nodes) // page)
    table = rng.permutation(batch * max_pages).reshape(batch, max_pages)
    parents, leaves = _random_parents(rng, batch, nodes, chain=batch == 33), rng.integers(-2, nodes, batch)
    leaves[0] = nodes - 1
    want, want_lengths = np.full((batch, nodes), -1), lengths.copy()
    for b in range(batch):
        for i, node in enumerate(_way(parents[b], leaves[b])):
            row = lengths[b] + i
            want[b, node] = table[b, row // page] * page + row % page
            want_lengths[b] = row + 1
    cache = gpu_backend.paged_cache(P.BF16_CODE, batch, 2, 1, 8, page, max_pages)
    n, out, slots = ints(lengths), torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros((batch, nodes), dtype=torch.int32, device="cuda")
    cache.path_slots(ints(table), n, ints(parents), ints(leaves), slots, lengths_out=None if in_place else out, stream=_stream())
    assert np.array_equal(slots.cpu().numpy(), want)
    assert np.array_equal((n if in_place else out).cpu().numpy(), want_lengths) and (in_place or n.tolist() == lengths.tolist())
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
def test_path_slots_out_of_range_are_reported(gpu_backend):
    import torch

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.BF16_CODE, 3, 2, 1, 8, 4, 2)
    good = dict(table=[[0, 1], [2, 3], [4, 5]], lengths=[3, 2, 4], parents=[[-1, 0, 1]] * 3, leaves=[1, 2, 0])
    want, want_lengths = [[3, 4, -1], [10, 11, 12], [20, -1, -1]], [5, 5, 5]
    for change, code, row, length in ((dict(table=[[0, 1], [2, -1], [4, 5]]), 40, [10, 11, -1], 5), (dict(lengths=[3, 6, 4]), 41, [-1] * 3, 6),
                                      (dict(lengths=[3, -2, 4]), 41, [-1] * 3, -2), (dict(leaves=[1, 3, 0]), 41, [-1] * 3, 2),
                                      (dict(leaves=[1, 1 << 30, 0]), 41, [-1] * 3, 2),
                                      (dict(parents=[[-1, 0, 1], [-1, 1, 1], [-1, 0, 1]]), 43, [-1, 10, 11], 4)):
        a = {n: ints(x) for n, x in {**good, **change}.items()}
        slots, out = torch.zeros((3, 3), dtype=torch.int32, device="cuda"), ints([0, 0, 0])
        cache.path_slots(a["table"], a["lengths"], a["parents"], a["leaves"], slots, lengths_out=out, stream=_stream())
        with pytest.raises(be_mod.BackendError, match=f"code {code}"):
            gpu_backend.operators_status(stream=_stream())
        assert slots.tolist() == [want[0], row, want[2]] and out.tolist() == [want_lengths[0], length, want_lengths[2]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv_heads,head_dim,page,layout", [("bf16", 8, 128, 16, "nhd"), ("f32", 2, 64, 5, "hnd"), ("f16", 1, 8, 3, "nhd"),
                                                                 ("f32", 3, 4, 64, "nhd"), ("bf16", 4, 256, 1, "hnd")])
@pytest.mark.parametrize("rows", [1, 37, 3000])
def test_store(gpu_backend, dtype, kv_heads, head_dim, page, layout, rows):
    import torch

    c = _Case(dtype, kv_heads, kv_heads, head_dim, page, [rows + 100], seed=rows, layout=layout)
    rng = np.random.default_rng(rows)
    slots = torch.tensor(rng.permutation(c.k.shape[0] * page)[:rows], dtype=torch.int32, device="cuda")
    slots[rows // 3::4] = -1 - (rows % 7)
    packed = c.randn(rows, 2 * kv_heads + 1, head_dim)
    k_new, v_new = packed[:, :kv_heads], packed[:, kv_heads + 1:]
    k, v = c.k.clone(), c.v.clone()
    there = (slots >= 0).nonzero()[:, 0]
    at = slots[there].long()
    k[at // page, at % page], v[at // page, at % page] = k_new[there], v_new[there]
    cache = c.handle(gpu_backend)
    cache.store(c.k, c.v, k_new, v_new, slots, stream=_stream())
    same = lambda x, y: bool(((x == y) | (x.isnan() & y.isnan())).all())
    assert same(c.k, k) and same(c.v, v)
    gpu_backend.operators_status(stream=_stream())
    slots[0] = c.k.shape[0] * page  # behind the pool
    k_new[0] = 5
    if rows > 1 and int(slots[1]) >= 0:
        k[int(slots[1]) // page, int(slots[1]) % page] = k_new[1]
    cache.store(c.k, c.v, k_new, v_new, slots, stream=_stream())
    with pytest.raises(be_mod.BackendError, match="code 40"):
        gpu_backend.operators_status(stream=_stream())
    assert same(c.k, k) and same(c.v, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompts_drafts_and_steps_on_one_cache(gpu_backend, dtype):
    """Pages for prompts, their attention and rows, a verified tree, its accepted tokens, and a decode step behind them: every result is
    that of plain attention over the tokens that a sequence has by then."""
    import torch

    batch, heads, kv_heads, dim, page, max_pages, nodes, pool = 3, 8, 2, 64, 8, 20, 6, 40
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda").to(_torch_type(dtype))
    stream = torch.cuda.Stream()
    cache = gpu_backend.paged_cache(CODE[dtype], batch, heads, kv_heads, dim, page, max_pages, tree=nodes)
    k_pages, v_pages = (torch.full((pool, page, kv_heads, dim), math.nan, dtype=_torch_type(dtype), device="cuda") for _ in "kv")
    table, held = ints([[-1] * max_pages] * batch), ints([0] * batch)
    free, count = ints(list(range(pool))), ints([pool])
    prompts = [37, 0, 64]
    starts = ints(np.cumsum([0] + prompts).tolist())
    q, k, v = randn(110, heads, dim), randn(110, kv_heads, dim), randn(110, kv_heads, dim)
    slots, out = torch.zeros(110, dtype=torch.int32, device="cuda"), torch.zeros_like(q)
    tree_q, tree_k, tree_v = randn(batch, nodes, heads, dim), randn(batch, nodes, kv_heads, dim), randn(batch, nodes, kv_heads, dim)
    parents, leaves = [[-1, 0, 0, 1, 3, 2]] * batch, [4, -1, 2]
    step_q, step_k, step_v = randn(batch, heads, dim), randn(batch, kv_heads, dim), randn(batch, kv_heads, dim)
    lengths, more = ints(prompts), ints([prompts[0] + nodes, 0, prompts[2] + nodes])
    tree_out, step_out = torch.zeros_like(tree_q), torch.zeros_like(step_q)
    tree_slots, parents_t, leaves_t, one = torch.zeros((batch, nodes), dtype=torch.int32, device="cuda"), ints(parents), ints(leaves), ints([1, 0, 1])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        on = dict(stream=stream.cuda_stream)
        cache.assign_pages(lengths, held, table, free, count, starts=starts, slots=slots, **on)
        gpu_backend.prompt_attention(q, k, v, starts, out, **on)
        cache.store(k_pages, v_pages, k, v, slots, **on)
        cache.assign_pages(more, held, table, free, count, **on)
        cache.attend_tree(tree_q, k_pages, v_pages, table, lengths, tree_out, tree_k, tree_v, parents_t, **on)
        cache.path_slots(table, lengths, parents_t, leaves_t, tree_slots, **on)
        cache.store(k_pages, v_pages, tree_k.flatten(0, 1), tree_v.flatten(0, 1), tree_slots.flatten(), **on)
        lengths += one
        cache.assign_pages(lengths, held, table, free, count, **on)
        cache.attend(step_q, k_pages, v_pages, table, lengths, step_out, k_new=step_k, v_new=step_v, **on)
    gpu_backend.operators_status(stream=stream.cuda_stream)
    ways = [_way(parents[b], leaves[b]) for b in range(batch)]
    total = [n + len(w) + (b != 1) for b, (n, w) in enumerate(zip(prompts, ways))]
    assert lengths.tolist() == total and held.tolist() == [-(-n // page) for n in total] and int(count) == pool - sum(held.tolist())
    rep = heads // kv_heads

    def add(got, q, b, h, tree, more=()):
        a, n, g = int(starts[b]), prompts[b], h // rep
        keys, values = (torch.cat([x[a:a + n, g], y[b, tree, g]] + [m[b:b + 1, g] for m in z]) for x, y, z in
                        ((k, tree_k, more[:1]), (v, tree_v, more[1:])))
        w, _, bound, _ = _expected(dtype, q, keys, values, dim ** -0.5)
        _within(got, w, bound, (b, h, tree))
    for h in range(heads):
        for b in (0, 2):
            a = int(starts[b])
            for i in (0, 20, prompts[b] - 1):
                w, _, bound, _ = _expected(dtype, q[a + i, h], k[a:a + i + 1, h // rep], v[a:a + i + 1, h // rep], dim ** -0.5)
                _within(out[a + i, h], w, bound, "prompt")
            add(step_out[b, h], step_q[b, h], b, h, ways[b], (step_k, step_v))
        for b in range(batch):
            for i in range(nodes):
                add(tree_out[b, i, h], tree_q[b, i, h], b, h, _way(parents[b], i))


@pytest.mark.gpu
def test_two_trees_on_two_streams(gpu_backend):
    """Handles of their own: calls of both under way at once."""
    import torch

    pairs = [(_Trees("bf16", 16, 4, 128, 16, [4000, 100], 24, seed=i), torch.cuda.Stream()) for i in range(2)]
    for t, _ in pairs:
        t.cache = t.case.handle_of_tree(gpu_backend)
    torch.cuda.synchronize()
    for _ in range(20):
        for t, side in pairs:
            t.run(gpu_backend, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for t, _ in pairs:
        t.check(some=150)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_more_prompts_than_an_axis_of_the_grid_has_blocks(gpu_backend, dtype):
    """A sequence of one token has its own value as the result, whose weight is one."""
    import torch

    sequences = 140000
    lengths = np.ones(sequences, np.int64)
    lengths[::7] = 0
    gen = torch.Generator(device="cuda").manual_seed(5)
    tokens = int(lengths.sum())
    x = torch.randn((tokens + 4, 4, 8), generator=gen, device="cuda").to(_torch_type(dtype))
    q, k, v = x[:, :2], x[:, 2:3], x[:, 3:]
    starts = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
    out, lse = torch.full((tokens + 4, 2, 8), 7.0, dtype=x.dtype, device="cuda"), torch.full((tokens + 4, 2), 7.0, device="cuda")
    gpu_backend.prompt_attention(q, k, v, starts, out, lse=lse, scale=0.3, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    want = v[:tokens].double().expand(tokens, 2, 8)
    bound = (2.0 ** -17 + 2 * PROBABILITY[dtype]) * want.abs() + LEAST[dtype] * want.abs()
    _within(out[:tokens], want, bound + HALF_STEP[dtype] * (want.abs() + bound) + SUBNORMAL[dtype], "values")
    products = q[:tokens].double() * k[:tokens].double() * 0.3
    score = products.sum(-1)
    _within(lse[:tokens], score, products.abs().sum(-1) * 24 * 2.0 ** -24 + 2.0 ** -17 + 2.0 ** -20 * (1 + score.abs()), "lse")
    assert (out[tokens:] == 7).all() and (lse[tokens:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_trees_of_a_large_batch(gpu_backend, dtype):
    lengths = np.random.default_rng(2).integers(0, 40, 3000).tolist()
    t = _Trees(dtype, 4, 2, 64, 8, lengths, 2, seed=2)
    t.run(gpu_backend)
    t.check(some=2500)
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 6])
def test_trees_on_shared_pages(gpu_backend, dtype, page):
    """Sequences may have pages in common: a prompt's, say."""
    t = _Trees(dtype, 8, 2, 128, page, [400, 400, 333], 5, seed=6)
    c = t.case
    shared = 300 // page
    c.table[1, :shared], c.table[2, :shared] = c.table[0, :shared].clone(), c.table[0, :shared].clone()
    t.run(gpu_backend)
    t.check(some=400)


@pytest.mark.gpu
def test_two_graphs_of_trees_on_one_handle(gpu_backend):
    """Their calls share the handle's workspace and follow each other on a stream."""
    import torch

    t = _Trees("bf16", 16, 4, 128, 16, [3000, 17], 9, seed=3, counts=[9, 9])
    t.run(gpu_backend)
    torch.cuda.synchronize()
    want = t.out.clone()
    others, side = torch.empty_like(t.out), torch.cuda.Stream()
    q = t.q * 0.5
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, change in zip(graphs, ({}, {"q": q, "out": others})):
        with torch.cuda.graph(graph, stream=side):
            c = t.case
            args = {"q": t.q, "out": t.out, **change}
            t.cache.attend_tree(args["q"], c.k, c.v, c.table, c.lengths, args["out"], t.k, t.v, t.parents, counts=t.counts, stream=_stream())
    t.out.fill_(7), others.fill_(7)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            for graph in graphs:
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(t.out, want)
    eager, c = torch.empty_like(want), t.case
    t.cache.attend_tree(q, c.k, c.v, c.table, c.lengths, eager, t.k, t.v, t.parents, counts=t.counts, stream=_stream())
    assert torch.equal(eager, others)


@pytest.mark.gpu
def test_pages_slots_and_rows_in_a_graph(gpu_backend):
    """One captured step that is replayed: the lengths grow, pages come as they are needed, and rows go where the slots say. The table is
    changed in place, the stack is not: its copy is what the next step reads."""
    import torch

    batch, page, max_pages, pool, kv_heads, dim = 5, 4, 6, 40, 2, 16
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.F32, batch, 2, kv_heads, dim, page, max_pages)
    k_pages, v_pages = (torch.zeros((pool, page, kv_heads, dim), device="cuda") for _ in "kv")
    lengths, held, table = ints([0] * batch), ints([0] * batch), ints([[-1] * max_pages] * batch)
    free, count, free_out, count_out = ints(list(range(pool))), ints([pool]), ints([7] * pool), ints([7])
    parents, leaves, path, after = ints([[-1, 0, 1]] * batch), ints([2, 0, 1, -1, 2]), torch.zeros((batch, 3), dtype=torch.int32, device="cuda"), ints([0] * batch)
    room = ints([0] * batch)
    k_new, v_new = torch.zeros((batch, 3, kv_heads, dim), device="cuda"), torch.zeros((batch, 3, kv_heads, dim), device="cuda")

    def step():
        torch.add(lengths, 3, out=room)
        cache.assign_pages(room, held, table, free, count, free_pages_out=free_out, free_count_out=count_out, stream=_stream())
        free.copy_(free_out), count.copy_(count_out)
        cache.path_slots(table, lengths, parents, leaves, path, lengths_out=after, stream=_stream())
        cache.store(k_pages, v_pages, k_new.flatten(0, 1), v_new.flatten(0, 1), path.flatten(), stream=_stream())
        lengths.copy_(after)

    step()  # before the capture
    for x, to in ((lengths, 0), (held, 0), (table, -1), (count, pool)):
        x.fill_(to)
    free.copy_(ints(list(range(pool))))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    steps, rows = 5, [[] for _ in range(batch)]
    for i in range(steps):
        k_new.copy_(torch.randn(k_new.shape, device="cuda")), v_new.copy_(k_new + 1)
        graph.replay()
        for b, n in enumerate([3, 1, 2, 0, 3]):
            rows[b] += list(k_new[b, :n].clone())
    gpu_backend.operators_status(stream=_stream())
    assert lengths.tolist() == [15, 5, 10, 0, 15]
    assert held.tolist() == [-(-(n * (steps - 1) + 3) // page) for n in [3, 1, 2, 0, 3]]
    used = table[table >= 0].tolist()
    assert len(set(used)) == len(used) == sum(held.tolist()) and int(count) == pool - len(used)
    assert sorted(used + free[:int(count)].tolist()) == list(range(pool))
    for b in range(batch):
        for t, row in enumerate(rows[b]):
            at = int(table[b, t // page]), t % page
            assert torch.equal(k_pages[at], row) and torch.equal(v_pages[at], row + 1)


@pytest.mark.gpu
def test_prompts_trees_and_rows_of_the_backends_own_buffers(gpu_backend):
    """DeviceBuffers on the backend's stream, with no waits between the calls."""
    be, rng = gpu_backend, np.random.default_rng(4)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    put = lambda x: be.buffer_from_host(np.ascontiguousarray(x))
    cache = be.paged_cache(P.F32, 1, 2, 1, 16, 4, 3, tree=3)
    q, k, v = f32(6, 2, 16), f32(6, 1, 16), f32(6, 1, 16)
    table, held, lengths = put(np.full((1, 3), -1, np.int32)), put(np.zeros(1, np.int32)), put(np.array([6], np.int32))
    starts, slots = put(np.array([0, 6], np.int32)), be.allocate_buffer(P.S32, [6])
    free, count = put(np.arange(4, dtype=np.int32)), put(np.array([4], np.int32))
    k_pages, v_pages = put(np.zeros((4, 4, 1, 16), np.float32)), put(np.zeros((4, 4, 1, 16), np.float32))
    out, tree_out = be.allocate_buffer(P.F32, [6, 2, 16]), be.allocate_buffer(P.F32, [1, 3, 2, 16])
    buffers = [put(x) for x in (q, k, v)]
    cache.assign_pages(lengths, held, table, free, count, starts=starts, slots=slots)
    be.prompt_attention(*buffers, starts, out)
    cache.store(k_pages, v_pages, buffers[1], buffers[2], slots)
    tree = [f32(1, 3, 2, 16), f32(1, 3, 1, 16), f32(1, 3, 1, 16)]
    parents, leaves, path = put(np.array([[-1, 0, 0]], np.int32)), put(np.array([2], np.int32)), be.allocate_buffer(P.S32, [1, 3])
    tree_buffers = [put(x) for x in tree]
    cache.attend_tree(tree_buffers[0], k_pages, v_pages, table, lengths, tree_out, tree_buffers[1], tree_buffers[2], parents)
    cache.path_slots(table, lengths, parents, leaves, path)
    be.operators_status()

    def expected(q, k, v):
        s = k.astype(np.float64) @ q.astype(np.float64) / 4
        p = np.exp(s - s.max())
        return p @ v.astype(np.float64) / p.sum()

    # scores off by 32 * 2^-24 * sum |q k| / 4 < 4e-5 twice, 2^-17 for the exponentials, values below 5
    for i in range(6):
        for h in range(2):
            assert np.abs(out.to_numpy()[i, h] - expected(q[i, h], k[:i + 1, 0], v[:i + 1, 0])).max() < 5e-4
    for i, way in enumerate(([0], [0, 1], [0, 2])):
        for h in range(2):
            want = expected(tree[0][0, i, h], np.concatenate([k[:, 0], tree[1][0, way, 0]]), np.concatenate([v[:, 0], tree[2][0, way, 0]]))
            assert np.abs(tree_out.to_numpy()[0, i, h] - want).max() < 5e-4
    assert table.to_numpy().tolist() == [[3, 2, -1]] and slots.to_numpy().tolist() == [12, 13, 14, 15, 8, 9]
    assert path.to_numpy().tolist() == [[10, -1, 11]] and lengths.to_numpy().tolist() == [8]
