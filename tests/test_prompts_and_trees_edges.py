"""Packed prompts, trees of drafted tokens and page tables where they are easily a little off. Tolerances as in test_prompts_and_trees.py."""
import math
import os
import re

import numpy as np
import pytest

from pjrtx_b200 import plan as P
from tests import test_prompts_and_trees as base
from tests.test_operators import _stream


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


# ---- page tables ---------------------------------------------------------------------------------------------------


def test_blocks_of_a_cluster_are_known_to_run_before_one_writes_another(backend):
    """Shared memory of another block may be written once it has started, which the cluster's barrier tells."""
    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pjrtx_b200", "csrc", "kernels")
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
