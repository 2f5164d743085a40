"""Packed prompts, trees of drafted tokens and page tables where they are easily a little off. Tolerances as in test_prompts_and_trees.py."""
import math

import pytest

from tests import test_prompts_and_trees as base
from tests.test_operators import _within


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
