"""Tree attention over the paged cache (jl_tree_attention) against its
definition in 64 bits: lengths from nothing to long contexts, ragged batches,
trees that end inside a page, across pages and past 64 nodes, rows that see
nothing, both row and pool types, shared heads, strides, bad pages, graphs,
streams and the refusals' neighbours that are allowed."""
import math

import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from tree_util import Call, HEAD, PAGE, ancestors, check_tree, make_trees

pytestmark = pytest.mark.gpu

TYPES = [(J.KV_F32, J.KV_BF16), (J.KV_BF16, J.KV_BF16), (J.KV_F32, J.KV_F32), (J.KV_BF16, J.KV_F32)]
IDS = ["f32-bf16pool", "bf16-bf16pool", "f32-f32pool", "bf16-f32pool"]
types = pytest.mark.parametrize("dtype,pool", TYPES, ids=IDS)


@types
@pytest.mark.parametrize("ctx,nodes", [
    (0, 1), (1, 1), (0, 5), (62, 1), (63, 1), (64, 1), (63, 2), (50, 14), (50, 15), (60, 64), (127, 65), (64, 64),
    (1000, 33), (5, 256), (130, 200)])
def test_one_sequence(dtype, pool, ctx, nodes):
    Call(make_trees([ctx], [nodes], 4, 2, dtype, pool, seed=ctx + nodes)).checked()


@types
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (2, 2), (4, 1), (6, 2), (10, 2), (16, 8), (32, 8), (16, 1), (128, 1)])
def test_shared_heads(dtype, pool, q_heads, kv_heads):
    Call(make_trees([70, 300], [9, 3], q_heads, kv_heads, dtype, pool, seed=q_heads)).checked()


@types
def test_ragged_batch(dtype, pool):
    """Sequences of very different lengths, some without nodes or committed
    positions, so that workers start and end inside items and skip sequences."""
    ctx = [0, 2000, 1, 64, 640, 63, 3, 0, 129, 1500]
    nodes = [3, 17, 1, 0, 64, 1, 0, 1, 40, 2]
    Call(make_trees(ctx, nodes, 8, 4, dtype, pool, seed=5, pad=6, extra_ld=24, table_pad=3)).checked()


@types
def test_chains_without_a_mask(dtype, pool):
    """NULL mask: a prompt's causal rows, a decode step, a linear verify pass."""
    Call(make_trees([0, 900, 77], [100, 1, 5], 8, 2, dtype, pool, bits=None, seed=8)).checked()


@types
def test_many_short_sequences(dtype, pool):
    """More items than workers: a worker walks several whole items."""
    n = 700
    Call(make_trees([i % 7 for i in range(n)], [1 + i % 3 for i in range(n)], 2, 2, dtype, pool, seed=9)).checked()


@types
def test_a_row_that_sees_nothing(dtype, pool):
    bits = [0] + ancestors([-1, 0, 0]) + [0b110]
    t = make_trees([0, 0, 100], [1, 3, 1], 4, 2, dtype, pool, bits=bits, seed=2)
    t.bits[-1] = 0  # the last row still has its committed positions
    c = Call(t)
    c.checked()
    assert (c.out[0] == 0).all() and (c.lse[0] == -math.inf).all()


@types
def test_a_node_need_not_see_itself(dtype, pool):
    bits = [0b1000, 0b1, 0b0101, 0b1111]
    Call(make_trees([66], [4], 4, 2, dtype, pool, bits=bits, seed=3)).checked()


@types
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, pool, bad):
    """Positions past the sequence, spare pages and nodes outside a row's mask
    may hold infinities and NaN; only rows that see them may show them."""
    t = make_trees([70, 64], [6, 5], 4, 2, dtype, pool, seed=4)
    t.bits[:] = ancestors([-1, 0, 0, 1, 1, 2]) + ancestors([-1, 0, 1, 0, 3])
    clean = Call(t)
    clean.run()
    want = clean.out.clone()
    used = {}
    for s, (c, n) in enumerate(zip(t.ctx, t.nodes)):
        for p in range(c + n):
            used.setdefault(int(t.table[s, p // PAGE]), set()).add(p % PAGE)
    for page in range(t.k.shape[0]):
        for at in range(PAGE):
            if at not in used.get(page, ()):
                t.k[page, :, at] = bad
                t.v[page, :, at] = bad
    # node 5 of the first tree (seen by itself only), node 4 of the second
    hidden = [(0, 5), (1, 4)]
    for s, node in hidden:
        p = t.ctx[s] + node
        t.k[t.table[s, p // PAGE].long(), :, p % PAGE] = bad
        t.v[t.table[s, p // PAGE].long(), :, p % PAGE, 3:40] = bad
    c = Call(t)
    c.run()
    rows = [r for r in range(11) if r not in (5, 10)]
    assert torch.equal(c.out[rows], want[rows])


@types
def test_a_seen_infinity_shows(dtype, pool):
    """An infinite value in one dim of a node that a row sees."""
    t = make_trees([70], [3], 4, 2, dtype, pool, bits=[0b1, 0b11, 0b101], seed=6)
    p = 71
    t.v[t.table[0, 1].long(), 1, p % PAGE, 9] = math.inf
    c = Call(t)
    c.run()
    out = c.out[:3].view(3, 4, HEAD)
    assert (out[1, 2:, 9] == math.inf).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[1, 2:, 9] = False
    assert torch.isfinite(out[keep]).all()


@types
def test_pages_outside_the_pool_are_masked(dtype, pool):
    t = make_trees([300, 200], [4, 4], 4, 2, dtype, pool, seed=7)
    t.table[0, 1] = 10 ** 6
    t.table[1, 0] = -5
    c = Call(t)
    c.run()
    check_tree(t, c.out, c.lse)
    assert c.status.item() == 1


@types
def test_lengths_out_of_range_are_cut(dtype, pool):
    """A tree larger than max_nodes, rows past the row count and a negative
    length: what is in range is computed, and the status says so."""
    t = make_trees([80, 40, 10], [9, 2, 2], 4, 2, dtype, pool, bits=None, seed=11)
    c = Call(t, max_nodes=5)
    c.ctx[1] = -3
    c.run(rows=12)
    assert c.status.item() == 2
    assert (c.out[5:9] == 7.5).all() and (c.out[12:] == 7.5).all()
    t2 = make_trees([80], [9], 4, 2, dtype, pool, bits=None, seed=11)
    t2.q, t2.k, t2.v, t2.table, t2.nodes = t.q[:5].contiguous(), t.k, t.v, t.table[:1].contiguous(), [5]
    c2 = Call(t2)
    c2.run()
    ref = c2.out[:5]
    assert torch.allclose(c.out[:5].float(), ref.float(), rtol=2e-2, atol=1e-5)


@types
def test_output_over_the_queries(dtype, pool):
    t = make_trees([500, 30], [8, 8], 8, 4, dtype, pool, seed=12, extra_ld=64)
    c = Call(t)
    c.run()
    want = c.out.clone()
    keep = t.q[:, 8 * HEAD:].clone()
    c.run(out=t.q.data_ptr(), out_ld=t.q.shape[1])
    assert torch.equal(t.q[:, :8 * HEAD], want)
    assert torch.equal(t.q[:, 8 * HEAD:], keep)


@types
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scales(dtype, pool, scale):
    """A flat and a sharp softmax, with a context whose scores rise along it
    (the running maximum moves on every page)."""
    t = make_trees([700], [6], 4, 2, dtype, pool, seed=13, scale=scale)
    for p in range(11):
        t.k[t.table[0, p].long()] *= 0.3 + 0.15 * p
    Call(t).checked()


@types
def test_weights_far_apart(dtype, pool):
    """The largest scores in the first pages, and far below them later: the
    weights of later pages underflow."""
    t = make_trees([900], [3], 2, 1, dtype, pool, seed=14, scale=1.0)
    t.k[t.table[0, 0].long()] *= 4
    Call(t).checked()


@types
def test_long_context(dtype, pool):
    t = make_trees([20011], [7], 8, 2, dtype, pool, seed=15)
    Call(t).checked()


@types
@pytest.mark.parametrize("table_pad", [0, 20, 100, 5000])
@pytest.mark.parametrize("seqs", [1, 3, 24])
def test_widths_of_the_page_table(dtype, pool, seqs, table_pad):
    """The work is cut by the pages a sequence may have: whole items, items
    shared by clusters of CTAs, even ranges.  Sequences without nodes, shorter
    than a cluster has CTAs, and trees past a tile's rows, in each."""
    ctx = [(977 * i + 700) % 1500 if i % 5 != 3 else i % 2 for i in range(seqs)]
    nodes = [(7 * i + 40) % 61 if i % 7 else 33 for i in range(seqs)]
    Call(make_trees(ctx, nodes, 8, 2, dtype, pool, seed=seqs + table_pad, table_pad=table_pad)).checked()


@types
@pytest.mark.parametrize("table_pad", [8, 100, 5000])
def test_values_that_are_not_finite_in_shared_items(dtype, pool, table_pad):
    """Nodes of a tree that spans the parts of an item: a value that only its own
    row sees reaches no other row."""
    n = 90
    t = make_trees([600], [n], 4, 2, dtype, pool, bits=[1 << i for i in range(n)], seed=3, table_pad=table_pad)
    page, row = t.table[0, 620 // PAGE].item(), 620 % PAGE
    t.v[page, :, row, 77] = math.inf
    c = Call(t)
    c.run()
    out = c.out[:n, :4 * HEAD].view(n, 4, HEAD)
    others = torch.arange(n) != 20
    assert (out[20, :, 77] == math.inf).all()
    assert torch.isfinite(out[others]).all()
    t.v[page, :, row, 77] = 0
    check = Call(t)
    check.run()
    assert torch.equal(check.out[:n][others], c.out[:n][others])


@types
def test_captured_and_replayed(dtype, pool):
    """Two calls in one graph, with lengths changed between replays."""
    a = Call(make_trees([300, 20], [7, 30], 4, 2, dtype, pool, seed=16))
    b = Call(make_trees([64], [12], 8, 8, dtype, pool, seed=17))
    a.run()
    b.run()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            a.run()
            b.run()
        for ctx in ([300, 20], [100, 34], [0, 1]):
            a.ctx.copy_(torch.tensor(ctx))
            a.t.ctx = ctx
            a.out.fill_(7.5)
            b.out.fill_(7.5)
            g.replay()
            st.synchronize()
            check_tree(a.t, a.out)
            check_tree(b.t, b.out)


@types
def test_two_streams_at_once(dtype, pool):
    calls = [Call(make_trees([2000, 64 * i], [8, 20], 8, 2, dtype, pool, seed=20 + i)) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c, s in zip(calls, streams):
            c.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        check_tree(c.t, c.out, c.lse)


def test_a_row_does_not_depend_on_stale_workspace():
    c = Call(make_trees([3000], [16], 8, 2, J.KV_BF16, J.KV_BF16, seed=30))
    c.run()
    want = c.out.clone()
    c.work.fill_(0)
    c.run()
    assert torch.equal(c.out, want)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements: pages beyond 4 GB."""
    pages, kv_heads = 70000, 4
    k = torch.zeros((pages, kv_heads, PAGE, HEAD), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    t = make_trees([200], [5], 8, kv_heads, J.KV_BF16, J.KV_BF16, seed=31)
    ids = [69999, 35000, 66000, 1]
    for i, p in enumerate(ids[:t.table.shape[1]]):
        k[p], v[p] = t.k[t.table[0, i].long()], t.v[t.table[0, i].long()]
        t.table[0, i] = p
    t.k, t.v = k, v
    Call(t).checked()
