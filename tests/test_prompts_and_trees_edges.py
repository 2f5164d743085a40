"""Packed prompts, trees of drafted tokens and page tables where they are easily a little off. Tolerances as in test_prompts_and_trees.py."""
import math
import os
import re
import subprocess
import sys

import numpy as np
import pytest

from pjrtx_b200 import backend as be_mod
from pjrtx_b200 import plan as P
from tests import test_prompts_and_trees as base
from tests.test_operators import _stream, _torch_type, _within

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40), (2, 2, 200)])
def test_every_row_of_a_warp_is_computed_once_more(gpu_backend, dtype, heads, kv_heads, head_dim):
    """Values of all dimensions at the ends of blocks spoil all rows before them: each is stored by its thread and again by its warp."""
    lengths = [64, 129, 300]
    p = base._Prompts(dtype, heads, kv_heads, head_dim, lengths, seed=head_dim)
    for b, n in enumerate(lengths):
        p.v[p.ends[b] + n - 1] = math.inf
    for _ in range(20):
        p.out.fill_(7)
        p.run(gpu_backend)
    rep, c = heads // kv_heads, base._Compared()
    for b, n in enumerate(lengths):
        a = p.ends[b]
        for i in range(0, n - 1, 3):
            for h in range(heads):
                c.add(dtype, p.out[a + i, h], p.lse[a + i, h], p.q[a + i, h], p.k[a:a + i + 1, h // rep], p.v[a:a + i + 1, h // rep], head_dim ** -0.5)
        assert (p.out[a + n - 1] == math.inf).all()
    c.check("rows before the last")


# A probability meets the values in 16 bits as two numbers, itself cut off and the rest rounded. The rest is below the last place that is kept, so that
# half of its own last place is 2^-16 of a bf16 or 2^-22 of an f16; an f16 that is subnormal, in 2^11 times the largest, may lose 2^-25.
TWO_NUMBERS = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}


@pytest.fixture
def finer(monkeypatch):
    """The module's bounds with what two numbers lose of a probability, once: the sum has it in f32."""
    monkeypatch.setattr(base, "PROBABILITY", {t: x / 2 for t, x in TWO_NUMBERS.items()})  # the bounds take it twice


def _level(q, v, axis):
    """Scores close to each other, whose own errors are small then, over values that nearly cancel."""
    q *= 0.05
    v.abs_()
    for i in range(1, v.shape[axis], 2):
        v.select(axis, i).neg_()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
@pytest.mark.parametrize("level", [False, True])
def test_prompts_are_as_exact_as_their_rounding(gpu_backend, finer, dtype, heads, kv_heads, head_dim, level):
    p = base._Prompts(dtype, heads, kv_heads, head_dim, [300, 1, 70, 0, 129], seed=heads)
    if level:
        _level(p.q, p.v, 0)
    p.run(gpu_backend)
    p.check(some=1500)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
@pytest.mark.parametrize("lengths,nodes,level", [([900, 0, 33], 1, False), ([900, 0, 33], 9, False), ([900, 0, 33], 64, False), ([0, 0, 0], 64, True)])
def test_trees_are_as_exact_as_their_rounding(gpu_backend, finer, dtype, heads, kv_heads, head_dim, lengths, nodes, level):
    t = base._Trees(dtype, heads, kv_heads, head_dim, 16, lengths, nodes, seed=nodes, counts=[nodes] * 3)
    if level:
        _level(t.q, t.v, 1)
    t.run(gpu_backend)
    t.check(some=900)


ODD = [(17, 0.5), (3, -5.0), (100, -17.0), (200, -30.0), (299, -60.0), (150, -80.0)]  # key and score; values of dimensions 2 j and 2 j + 1 are infinite


def _place_odd_values(k, v, gen):
    """Keys [300, heads, d] whose first elements are the scores, and their values."""
    k[:, :, 1:] = 0
    k[:, :, 0] = -(gen.initial_seed() % 7 + 53) * (0.1 + 0.9 * k[:, :, 0].float().abs().clamp(max=1)).to(k.dtype)
    k[40:42, :, 0] = -math.inf  # probability 0 with finite values: nothing, with infinite ones: NaN
    v[41, :, 24], v[41, :, 25] = math.inf, -math.inf
    for j, (t, score) in enumerate(ODD):
        k[t, :, 0] = score
        v[t, :, 2 * j] = math.inf
        v[t, :, 2 * j + 1] = -math.inf
    v[20, :, 0] = -math.inf  # both: NaN
    v[8, :, 1] = math.nan


def _check_odd(dtype, out, k, v, seen):
    """Rows of one head: out [rows, d] over scores k [keys] and values v [keys, d], row i over the keys of seen [rows, keys]; q is 1 and 0 elsewhere."""
    import torch

    k, v = k.double(), v.double()
    s = torch.where(seen, k, -math.inf)
    p = torch.softmax(s, 1)
    e = float(k[k.isfinite()].abs().max()) * (v.shape[1] + 16) * 2.0 ** -24
    plain = torch.where(v.isfinite(), v, 0)
    sees = lambda what: (p > 0).double() @ what.double() > 0
    plus, minus, nan = sees(v == math.inf), sees(v == -math.inf), (seen & v.isnan().any(1)).double() @ v.isnan().double() > 0
    nan |= (seen & (p == 0)).double() @ v.isinf().double() > 0
    odd, got = plus | minus | nan, out.double()
    want = torch.where(nan | plus & minus, math.nan, torch.where(plus, math.inf, -math.inf))[odd]
    assert ((got[odd] == want) | (got[odd].isnan() & want.isnan())).all(), (int((got[odd] != want).sum()), got[odd][:8], want[:8])
    want = p @ plain
    bound = (2 * e + 2.0 ** -17 + 2 * base.PROBABILITY[dtype]) * (p @ plain.abs()) + base.LEAST[dtype] * plain.abs().sum(0)
    bound = bound + base.HALF_STEP[dtype] * (want.abs() + bound) + base.SUBNORMAL[dtype]
    _within(got[~odd], want[~odd], bound[~odd], "beside the infinities")
    return int(odd.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
def test_prompts_keep_infinite_values_at_any_probability(gpu_backend, dtype, heads, kv_heads, head_dim):
    """A value that a row sees makes its dimension infinite however small its (f32) probability is, and nothing else."""
    import torch

    p = base._Prompts(dtype, heads, kv_heads, head_dim, [65, 300, 9], seed=head_dim)
    p.q[:, :, 0], p.q[:, :, 1:] = 1, 0
    a = p.ends[1]
    _place_odd_values(p.k[a:a + 300], p.v[a:a + 300], p.gen)
    p.run(gpu_backend, scale=1.0)
    seen = torch.ones((300, 300), dtype=torch.bool, device="cuda").tril()
    for h in range(heads):
        g = h // (heads // kv_heads)
        assert _check_odd(dtype, p.out[a:a + 300, h], p.k[a:a + 300, g, 0], p.v[a:a + 300, g], seen) > 1000
    p.check(1.0, some=300, skip=(1,))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (4, 2, 64), (2, 1, 256), (9, 3, 40)])
@pytest.mark.parametrize("nodes", [9, 64])
@pytest.mark.parametrize("page", [16, 6])
def test_trees_keep_infinite_values_at_any_probability(gpu_backend, dtype, heads, kv_heads, head_dim, nodes, page):
    """The same for cached rows, in parts and whole, and for nodes."""
    import torch

    t = base._Trees(dtype, heads, kv_heads, head_dim, page, [300, 4000, 0, 70], nodes, seed=head_dim, counts=[nodes, nodes - 1, nodes, nodes])
    c = t.case
    t.q[:, :, :, 0], t.q[:, :, :, 1:] = 1, 0
    for b in (0, 1):
        pg, row = c.places(b, c.lengths_list[b])
        c.k[pg, row, :, 1:] = 0
        c.k[pg, row, :, 0] = -40
        k, v = c.k[pg[-300:], row[-300:]], c.v[pg[-300:], row[-300:]]
        _place_odd_values(k, v, c.gen)
        c.k[pg[-300:], row[-300:]], c.v[pg[-300:], row[-300:]] = k, v
    t.k[:, :, :, 1:] = 0
    t.k[:, 5, :, 0] = -70
    t.v[:, 5, :, 20], t.v[:, 5, :, 21], t.v[:, 6, :, 22] = math.inf, -math.inf, math.nan
    t.run(gpu_backend, scale=1.0)
    gpu_backend.operators_status(stream=_stream())
    for b, n in enumerate(t.counts_list):
        length = c.lengths_list[b]
        seen = torch.zeros((n, length + nodes), dtype=torch.bool, device="cuda")
        seen[:, :length] = True
        for i in range(n):
            seen[i, [length + j for j in base._way(t.parents_list[b], i)]] = True
        pg, row = c.places(b, length)
        for h in range(heads):
            g = h // (heads // kv_heads)
            k, v = (torch.cat([pool[pg, row, g], new[b, :, g]]) for pool, new in ((c.k, t.k), (c.v, t.v)))
            assert _check_odd(dtype, t.out[b, :n, h], k[:, 0], v, seen) >= (14 * n if b < 2 else 1)
        assert (t.out[b, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rubbish", [0, -7, 63, 1 << 30])
def test_parents_behind_a_sequences_nodes_may_be_anything(gpu_backend, dtype, rubbish):
    t = base._Trees(dtype, 8, 2, 64, 16, [40, 100, 0, 33], 40, seed=12, counts=[7, 0, 39, 40])
    for b, n in enumerate(t.counts_list):
        t.parents[b, n:] = rubbish
    t.run(gpu_backend)
    t.check(some=300)
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("rubbish", [0, -7, 63, 1 << 30])
def test_parents_that_no_path_takes_may_be_anything(gpu_backend, rubbish):
    """Of idle sequences and behind a path's leaf; those up to the leaf are still looked at."""
    import torch

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.BF16_CODE, 4, 2, 1, 8, 4, 20)
    parents = torch.full((4, 64), rubbish, dtype=torch.int32, device="cuda")
    parents[1, :3], parents[3, :40] = ints([-1, 0, 0]), torch.arange(40, device="cuda").int() - 1
    table, lengths = torch.arange(80, device="cuda").int().reshape(4, 20), ints([3, 5, 9, 0])
    slots, out = torch.zeros((4, 64), dtype=torch.int32, device="cuda"), ints([0] * 4)
    cache.path_slots(table, lengths, parents, ints([-1, 2, -5, 39]), slots, lengths_out=out, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    want = [[-1] * 64 for _ in range(4)]
    want[1][0], want[1][2] = 85, 86
    want[3][:40] = range(240, 280)
    assert slots.tolist() == want and out.tolist() == [3, 7, 9, 40]
    cache.path_slots(table, lengths, parents, ints([-1, 3, -5, 39]), slots, lengths_out=out, stream=_stream())
    if rubbish:  # node 3 may have node 0 for its parent
        with pytest.raises(be_mod.BackendError, match="code 43"):
            gpu_backend.operators_status(stream=_stream())
    gpu_backend.operators_status(stream=_stream())


# Of head_dim 64 and 128 a loader has 32 rows of a block, of 256 16: pages of 8, 16 and 32 rows are a box each, of 64 to 128 several, of 24 and 48 not whole ones.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("page,layout", [(8, "nhd"), (16, "hnd"), (24, "nhd"), (32, "nhd"), (32, "hnd"), (48, "hnd"), (64, "nhd"), (96, "hnd"), (128, "nhd")])
@pytest.mark.parametrize("nodes", [5, 50])
def test_trees_on_pages_of_boxes(gpu_backend, finer, dtype, heads, kv_heads, head_dim, page, layout, nodes):
    """Blocks of whole boxes, and what is left of the last one; a table entry that names no page, in a box of its own or in one of several."""
    t = base._Trees(dtype, heads, kv_heads, head_dim, page, [1200, 128, 515, 127], nodes, seed=page + nodes, layout=layout, counts=[nodes, 1, nodes - 2, nodes])
    t.run(gpu_backend)
    t.check(some=250)
    gpu_backend.operators_status(stream=_stream())
    for entry in (-1, t.case.k.shape[0], 1 << 30):
        table = t.case.table.clone()
        t.case.table[0, 1200 // page // 2] = entry
        t.out.fill_(7), t.lse.fill_(7)
        t.run(gpu_backend)
        with pytest.raises(be_mod.BackendError, match="code 40"):
            gpu_backend.operators_status(stream=_stream())
        t.case.table = table
        t.check(some=120, skip=(0,), what="the other sequences")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("order", [(0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
@pytest.mark.parametrize("page", [16, 6])
def test_trees_on_pages_whose_axes_lie_in_any_order(gpu_backend, dtype, order, page):
    t = base._Trees(dtype, 6, 3, 64, page, [300, 0, 77], 9, seed=5)
    c, back = t.case, [order.index(i) for i in range(3)]
    c.k, c.v = (x.permute(*order, 3).contiguous().permute(*back, 3) for x in (c.k, c.v))
    t.run(gpu_backend)
    t.check(some=200)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_the_most_tokens_and_sequences(gpu_backend, dtype):
    """2^24 tokens of 2^20 sequences, one of which has most of them."""
    import torch

    tokens, count, long = 1 << 24, 1 << 20, 3000
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (torch.randn((tokens, 1, 8), generator=gen, device="cuda").to(_torch_type(dtype)) for _ in "qkv")
    lengths = torch.full((count,), 15, dtype=torch.int64)
    lengths[count // 3] = long
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    out, lse = torch.full_like(q, 7), torch.full((tokens, 1), 7.0, device="cuda")
    gpu_backend.prompt_attention(q, k, v, starts.int().cuda(), out, lse=lse, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    c, ends = base._Compared(), starts.tolist()
    for b in [0, 1, 77, count // 3 - 1, count // 3, count // 3 + 1, count - 2, count - 1] + np.random.default_rng(1).integers(0, count, 60).tolist():
        for i in (0, 7, int(lengths[b]) - 1):
            r, a = ends[b] + i, ends[b]
            c.add(dtype, out[r, 0], lse[r, 0], q[r, 0], k[a:r + 1, 0], v[a:r + 1, 0], 8 ** -0.5)
    c.check("most tokens")
    assert (out[ends[-1]:] == 7).all() and not (out[:ends[-1]] == 7).all(2).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads", [(65535, 65535), (65535, 1), (32768, 16384)])
def test_the_most_heads(gpu_backend, dtype, heads, kv_heads):
    p = base._Prompts(dtype, heads, kv_heads, 8, [2, 0, 3], seed=8)
    p.run(gpu_backend)
    p.check(some=400)
    t = base._Trees(dtype, heads, kv_heads, 8, 4, [5, 0], 3, seed=8, counts=[3, 2])
    t.run(gpu_backend)
    t.check(some=400)
    gpu_backend.operators_status(stream=_stream())


_GIVE_UP = """
import torch
from pjrtx_b200 import backend as be_mod
from pjrtx_b200 import plan as P
be = be_mod.Backend()
stream = torch.cuda.current_stream().cuda_stream
gen = torch.Generator(device="cuda").manual_seed(1)
rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()
batch, page, pages = 300, 1024, 400
cache = be.paged_cache(P.BF16_CODE, batch, 1, 1, 64, page, pages, tree=1)
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
k_pages, v_pages, table = rand(2, page, 1, 64), rand(2, page, 1, 64), (torch.arange(pages, device="cuda") % 2).int().repeat(batch, 1)
q, k, v = rand(batch, 1, 1, 64), rand(batch, 1, 1, 64), rand(batch, 1, 1, 64)
def run(rows):
    out = torch.zeros_like(q)
    cache.attend_tree(q, k_pages, v_pages, table, ints([rows] * batch), out, k, v, ints([[-1]] * batch), stream=stream)
    try:
        be.operators_status(stream=stream)
        status = "fine"
    except be_mod.BackendError as e:
        status = str(e)
    off = 0.0
    for b in range(0, batch, 50):
        keys, values = (torch.cat([x.reshape(-1, 64).repeat(pages // 2, 1)[:rows], y[b].reshape(1, 64)]).double() for x, y in ((k_pages, k), (v_pages, v)))
        off = max(off, float((torch.softmax(q[b, 0].double() @ keys.T / 8, 1) @ values - out[b, 0].double())[:, 1:].abs().max()))
    print(off < 0.01, status)
run(1500)
v_pages[1, 3, 0, 0] = float("inf")
run(page * pages)
v_pages[1, 3, 0, 0] = 0
run(1500)
"""


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_waits_that_run_out_end_the_call_and_are_reported(gpu_backend):
    """With a budget of a millisecond, and values that are looked through for an infinity for some milliseconds while the other warps wait for theirs: the
    kernel gives up, says so (44), and the next call is right."""
    done = subprocess.run([sys.executable, "-c", _GIVE_UP], capture_output=True, text=True, timeout=250, cwd=ROOT,
                          env={**os.environ, "PJRTX_B200_WAIT_TIMEOUT_MS": "1"})
    assert done.returncode == 0, done.stderr[-2000:]
    lines = done.stdout.splitlines()
    assert lines[0] == lines[2] == "True fine" and "code 44" in lines[1], lines
    done = subprocess.run([sys.executable, "-c", _GIVE_UP], capture_output=True, text=True, timeout=250, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.splitlines() == ["True fine"] * 3, (done.stdout, done.stderr[-2000:])


# ---- page tables ---------------------------------------------------------------------------------------------------


def test_blocks_of_a_cluster_are_known_to_run_before_one_writes_another(backend):
    """Shared memory of another block may be written once it has started, which the cluster's barrier tells."""
    kernels = os.path.join(ROOT, "pjrtx_b200", "csrc", "kernels")
    seen = 0
    for name in sorted(os.listdir(kernels)):
        with open(os.path.join(kernels, name)) as f:
            bodies = re.split(r"^__global__ ", f.read(), flags=re.M)[1:]
        for body in bodies:
            if "map_shared_rank" in body:
                seen += 1
                before = body[:body.index("map_shared_rank")]
                assert "barrier_wait" in before or "cluster.sync()" in before, (name, body[:120])
    assert seen >= 2


@pytest.mark.gpu
def test_assign_pages_while_other_kernels_hold_the_device(gpu_backend):
    """Blocks of the cluster start when there is room for them, and the tables are the same."""
    import torch

    rng = np.random.default_rng(3)
    batch, page, max_pages = 100, 16, 20
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    pool = batch * max_pages
    held = rng.integers(0, max_pages + 1, batch)
    pages, at = rng.permutation(pool), 0
    table = np.full((batch, max_pages), -1)
    for b, n in enumerate(held):
        table[b, :n] = pages[at:at + n]
        at += n
    free, lengths = pages[at:].tolist(), rng.integers(0, page * max_pages + 1, batch)
    want_held, want_table, want_free = base._assigned(lengths.tolist(), held.tolist(), table.tolist(), free, page, max_pages)
    stack = np.full(pool, -1)
    stack[:len(free)] = free
    args = [ints(lengths), ints(held), ints(table), ints(stack), ints([len(free)])]
    cache = gpu_backend.paged_cache(P.BF16_CODE, batch, 2, 1, 8, page, max_pages)
    p = base._Prompts("bf16", 32, 8, 128, [700] * 4, seed=4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(30):
        outs = [torch.full_like(a, 77) for a in args[1:]]
        side.wait_stream(torch.cuda.current_stream())
        p.run(gpu_backend)
        cache.assign_pages(*args, held_out=outs[0], page_table_out=outs[1], free_pages_out=outs[2], free_count_out=outs[3], stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        assert outs[0].tolist() == want_held and np.array_equal(outs[1].cpu().numpy(), want_table)
        assert outs[2][:len(want_free)].tolist() == want_free and int(outs[3]) == len(want_free)
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bad", [-1, -5, 400, 1 << 30])
def test_surplus_entries_that_name_no_page_go_nowhere(gpu_backend, in_place, bad):
    """What a sequence gives back counts as far as it is pages of the pool, and the others get nothing else."""
    import torch

    rng = np.random.default_rng(11)
    batch, page, max_pages, pool = 40, 4, 300, 400
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    held, need = np.zeros(batch, int), np.zeros(batch, int)
    held[[1, 5, 20, 39]], need[[1, 5, 20, 39]] = [200, 3, 40, 20], [10, 0, 39, 20]
    need[[0, 2, 6, 30]] = [3, 150, 9, 40]  # 202 in all, of 10 free ones and those that come back
    pages, at = rng.permutation(pool), 0
    table = np.full((batch, max_pages), -1)
    for b, n in enumerate(held):
        table[b, :n] = pages[at:at + n]
        at += n
    for b, columns in ((1, [10, 17, 42, 137, 138, 199]), (5, [0, 1, 2]), (20, [39])):
        table[b, columns] = bad
    free = pages[at:at + 10].tolist()
    good = lambda x: 0 <= x < pool
    want_free = free + [x for b in range(batch) for x in table[b, need[b]:held[b]].tolist() if good(x)]
    want_table, want_held = table.copy(), held.copy()
    for b in range(batch):
        want_table[b, need[b]:held[b]] = -1
        want_held[b] = min(held[b], need[b])
    assert len(want_free) == 10 + 190 - 6 and need[[0, 2, 6]].sum() <= len(want_free) < need[[0, 2, 6, 30]].sum()
    for b in (0, 2, 6):  # the last one's 40 are not there
        want_table[b, :need[b]] = [want_free.pop() for _ in range(need[b])]
        want_held[b] = need[b]
    stack = np.full(pool, -1)
    stack[:10] = free
    args = [ints(need * page), ints(held), ints(table), ints(stack), ints([10])]
    outs = {} if in_place else {n: torch.full_like(a, 77) for n, a in zip(("held_out", "page_table_out", "free_pages_out", "free_count_out"), args[1:])}
    cache = gpu_backend.paged_cache(P.BF16_CODE, batch, 2, 1, 8, page, max_pages)
    starts, slots = ints(range(batch + 1)), torch.zeros(batch, dtype=torch.int32, device="cuda")
    cache.assign_pages(*args, starts=starts, slots=slots, stream=_stream(), **outs)
    with pytest.raises(be_mod.BackendError, match="code 40"):
        gpu_backend.operators_status(stream=_stream())
    got = [x.cpu().numpy() for x in (args[1:] if in_place else outs.values())]
    assert got[0].tolist() == want_held.tolist() and np.array_equal(got[1], want_table)
    assert int(got[3][0]) == len(want_free) and got[2][:len(want_free)].tolist() == want_free
    assert slots[2] == want_table[2, 149] * page + 3 and slots[30] == -1
    # and the call after it, with what is left
    cache.assign_pages(ints([page] * batch), *[ints(x) for x in got], stream=_stream())
    gpu_backend.operators_status(stream=_stream())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 4095, 4096, 4097, 9000])
def test_slots_by_the_cluster_and_by_a_kernel_of_their_own(gpu_backend, tokens):
    import torch

    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    page, max_pages, lengths = 16, 400, [0, tokens // 2, 300, tokens - tokens // 2]
    new, rng = [0, tokens // 2, 0, tokens - tokens // 2], np.random.default_rng(tokens)
    table, starts = rng.permutation(4 * max_pages).reshape(4, max_pages), np.cumsum([0] + new)
    held = [-(-n // page) for n in lengths]
    cache = gpu_backend.paged_cache(P.BF16_CODE, 4, 2, 1, 8, page, max_pages)
    slots, free = torch.full((tokens,), 77, dtype=torch.int32, device="cuda"), ints([-1] * 4 * max_pages)
    cache.assign_pages(ints(lengths), ints(held), ints(table), free, ints([0]), starts=ints(starts), slots=slots, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    want = np.concatenate([table[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(lengths) if new[b]])
    assert np.array_equal(slots.cpu().numpy(), want)


@pytest.mark.gpu
def test_the_largest_batch_of_page_tables_and_paths(gpu_backend):
    """65535 sequences that grow by a page or give theirs back, and the slots of their paths."""
    import torch

    batch, page, max_pages = 65535, 2, 3
    b = torch.arange(batch, device="cuda").int()
    held, lengths = b % 4, (b * 7) % 7
    table = torch.full((batch, max_pages), -1, dtype=torch.int32, device="cuda")
    has = torch.arange(max_pages, device="cuda")[None] < held[:, None]
    table[has] = torch.arange(int(has.sum()), device="cuda").int()
    need = (lengths + page - 1) // page
    used, wanted = int(has.sum()), int((need - held).clamp(min=0).sum())
    pool = used + wanted
    stack = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    stack[:wanted] = torch.arange(used, pool, device="cuda").int()
    count = torch.tensor([wanted], dtype=torch.int32, device="cuda")
    cache = gpu_backend.paged_cache(P.BF16_CODE, batch, 2, 1, 8, page, max_pages)
    want = base._assigned(lengths.tolist(), held.tolist(), table.tolist(), stack[:wanted].tolist(), page, max_pages)
    cache.assign_pages(lengths, held, table, stack, count, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    assert held.tolist() == want[0] and table.tolist() == want[1] and stack[:int(count)].tolist() == want[2]
    n = (lengths - 1).clamp(min=0)
    parents, leaves, slots = torch.full((batch, 1), -1, dtype=torch.int32, device="cuda"), torch.where(lengths > 0, 0, -1).int(), torch.zeros((batch, 1), dtype=torch.int32, device="cuda")
    cache.path_slots(table, n, parents, leaves, slots, stream=_stream())
    gpu_backend.operators_status(stream=_stream())
    row = (lengths - 1).clamp(min=0).long()
    at = table.gather(1, (row // page)[:, None])[:, 0] * page + row % page
    assert torch.equal(slots[:, 0], torch.where(lengths > 0, at.int(), -1).int()) and torch.equal(n, lengths)
