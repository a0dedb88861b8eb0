"""The same call of tree attention gives the same bits, however its copies are
timed: items of many pages whose last page holds tree nodes and, behind them,
rows that were never written."""
import math

import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from tree_util import Call, PAGE, make_trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,pool", [(J.KV_F32, J.KV_BF16), (J.KV_BF16, J.KV_BF16), (J.KV_F32, J.KV_F32), (J.KV_BF16, J.KV_F32)],
                         ids=["f32-bf16pool", "bf16-bf16pool", "f32-f32pool", "bf16-f32pool"])
@pytest.mark.parametrize("ctx,nodes,table_pad", [([40000], [16], 0), ([4091], [5], 0), ([1500 - 37 * i for i in range(24)], [12] * 24, 0),
                                                 ([700 + 131 * i for i in range(8)], [32] * 8, 1000)],
                         ids=["long", "clusters", "whole", "ranges"])
def test_the_same_bits_every_time(dtype, pool, ctx, nodes, table_pad):
    """A page's V is cleared of the rows past the sequence while other pages are
    on their way; clearing the wrong one, or too early, changes bits now and then."""
    t = make_trees(ctx, nodes, 32, 8, dtype, pool, seed=len(ctx), table_pad=table_pad)
    for s, (c, n) in enumerate(zip(ctx, nodes)):
        if (c + n) % PAGE:
            t.v[t.table[s, (c + n) // PAGE].long(), :, (c + n) % PAGE:] = math.nan
    call = Call(t)
    call.run()
    want, lse = call.out.clone(), call.lse.clone()
    assert torch.isfinite(want[:t.rows]).all()
    for _ in range(60):
        call.out.fill_(7.5)
        call.run()
        assert torch.equal(call.out, want) and torch.equal(call.lse, lse)
    assert call.status.item() == 0
