"""Compactions whose rows cannot move batch by batch: long paths in any order,
which the header allows (jl_kv_compact)."""
import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from test_gpu_tree_rows import Moves

pytestmark = pytest.mark.gpu


def order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("pool", [J.KV_BF16, J.KV_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("ctx,paths", [
    ([30], [list(range(39, -1, -1))]),
    ([100], [list(range(199, -1, -1))]),
    ([70], [order(256, 1)]),
    ([10], [[5] * 30]),
    ([3, 90, 64], [order(40, 2), list(range(1, 18)), [20 - i for i in range(17)]]),
    ([128], [[16] * 16 + [0]]),        # the first entry that reads what an earlier batch wrote
    ([0], [list(range(16)) + [15]])], ids=["reversed40", "reversed200", "random256", "repeated", "three", "one-back", "last-of-first"])
@pytest.mark.parametrize("layers,kv_heads", [(1, 1), (5, 3), (9, 8)])
def test_long_paths_in_any_order(pool, ctx, paths, layers, kv_heads):
    m = Moves(len(ctx), ctx, paths, layers=layers, kv_heads=kv_heads, pool=pool, seed=len(paths[0]))
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want)
    assert m.status.item() == 0


def test_many_slabs_a_block():
    """More slabs than resident warps, so that a block walks several."""
    m = Moves(40, [37 * i % 90 for i in range(40)], [order(33, i) for i in range(40)], layers=36, kv_heads=8, seed=3, max_pages=2)
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want)


def test_bad_entries_in_a_long_path():
    """Negative entries and positions past the table are left out, the others move."""
    path = order(40, 5)
    m = Moves(1, [340], [path], seed=6)  # six pages: positions up to 383
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want) and m.status.item() == 0
    m = Moves(1, [360], [path], seed=6)
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want) and m.status.item() == 2
