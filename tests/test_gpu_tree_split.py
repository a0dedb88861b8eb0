"""Tree attention where its work is cut into even ranges that a second kernel
joins (wide page tables, long contexts): replayed graphs whose lengths change
which workers share an item, calls on several streams at once, outputs over the
queries and workspaces that hold anything.  Each test first makes sure that the
workspace is used."""
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from tree_util import Call, HEAD, check_tree, make_trees

pytestmark = pytest.mark.gpu

TYPES = [(J.KV_F32, J.KV_BF16), (J.KV_BF16, J.KV_BF16), (J.KV_F32, J.KV_F32), (J.KV_BF16, J.KV_F32)]
IDS = ["f32-bf16pool", "bf16-bf16pool", "f32-f32pool", "bf16-f32pool"]
types = pytest.mark.parametrize("dtype,pool", TYPES, ids=IDS)
WIDE = 5000  # pages that no sequence has: the cut goes by the table's width


def split_call(t):
    """A call whose workspace shows that items were shared: its entries and
    partial results were written."""
    c = Call(t)
    c.work.fill_(255)
    c.run()
    torch.cuda.synchronize()
    used = c.work.view(torch.uint8) != 255
    assert used[:64].any() and used[4096:].any()
    c.out.fill_(7.5)
    return c


@types
def test_stale_workspace(dtype, pool):
    """Nothing of a workspace's old contents shows, another call's results and
    NaN patterns among them."""
    c = split_call(make_trees([3000, 100], [16, 3], 8, 2, dtype, pool, seed=30, table_pad=WIDE))
    c.run()
    want, lse = c.out.clone(), c.lse.clone()
    other = split_call(make_trees([500, 2500, 40], [30, 2, 9], 8, 2, dtype, pool, seed=31, table_pad=WIDE))
    n = min(other.work.numel(), c.work.numel())
    for fill in (lambda: c.work.fill_(0), lambda: c.work.fill_(0x7F), lambda: c.work[:n].copy_(other.work[:n])):
        other.run()
        fill()
        c.out.fill_(7.5)
        c.run()
        assert torch.equal(c.out, want) and torch.equal(c.lse, lse)
    check_tree(c.t, c.out, c.lse)


@types
def test_one_workspace_for_calls_in_turn(dtype, pool):
    """Calls on one stream may share a workspace."""
    a = split_call(make_trees([3000], [16], 8, 2, dtype, pool, seed=32, table_pad=WIDE))
    b = split_call(make_trees([100, 1900], [5, 20], 8, 2, dtype, pool, seed=33, table_pad=WIDE))
    work = a.work if a.work.numel() > b.work.numel() else b.work
    for _ in range(5):
        for c in (a, b):
            c.run(workspace=work.data_ptr(), workspace_bytes=work.numel())
    for c in (a, b):
        check_tree(c.t, c.out, c.lse)


@types
def test_replayed_with_other_lengths(dtype, pool):
    t = make_trees([1800, 700, 300], [7, 30, 12], 8, 2, dtype, pool, seed=34, table_pad=WIDE)
    c = split_call(t)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.run()
            c.run()
        for ctx in ([1800, 700, 300], [5, 700, 0], [1800, 0, 17], [63, 64, 65], [1000, 1, 299]):
            c.ctx.copy_(torch.tensor(ctx))
            t.ctx = ctx
            c.out.fill_(7.5)
            g.replay()
            st.synchronize()
            check_tree(t, c.out, c.lse)
    assert c.status.item() == 0


@types
def test_several_streams_at_once(dtype, pool):
    calls = [split_call(make_trees([2000, 64 * i], [8, 20], 8, 2, dtype, pool, seed=40 + i, table_pad=WIDE)) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c, s in zip(calls, streams):
            c.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        check_tree(c.t, c.out, c.lse)


@types
def test_output_over_the_queries(dtype, pool):
    t = make_trees([2500, 30], [8, 8], 8, 4, dtype, pool, seed=45, extra_ld=64, table_pad=WIDE)
    c = split_call(t)
    c.run()
    want = c.out.clone()
    keep = t.q[:, 8 * HEAD:].clone()
    c.run(out=t.q.data_ptr(), out_ld=t.q.shape[1])
    assert torch.equal(t.q[:, :8 * HEAD], want)
    assert torch.equal(t.q[:, 8 * HEAD:], keep)


@types
def test_runs_of_pages_in_every_cut(dtype, pool):
    """Segments of more pages than a run: whole items (more of them than workers),
    shared ones, even ranges; rows whose maximum moves between the runs."""
    for ctx, nodes, pad in (([2500] * 160, [1] * 160, 0), ([9000], [3], 0), ([9000], [200], 0), ([6000] * 4, [40] * 4, 400)):
        t = make_trees([ctx[0]], [nodes[0]], 4, 2, dtype, pool, seed=len(ctx) + nodes[0], table_pad=pad)
        t.k[t.table[0, 60 % t.table.shape[1]].clamp_min(0).long()] *= 2.5
        for i in range(1, len(ctx)):  # other sequences share its pages and have other queries
            t.q = torch.cat([t.q, t.q[:nodes[0]].flip(0) * (1 + 0.1 * (i % 5))])
        t.table = t.table.repeat(len(ctx), 1).contiguous()
        t.ctx, t.nodes, t.bits = ctx, nodes, t.bits * len(ctx)
        Call(t).checked()


@pytest.mark.parametrize("dtype,pool", TYPES, ids=IDS)
def test_workspaces_stay_below_the_stated_size(dtype, pool):
    k = torch.zeros((1, 1, 64, HEAD), dtype=torch.float32, device="cuda")
    for kv_heads in (1, 2, 8):
        view = J.kv_pages(k.data_ptr(), k.data_ptr(), 1, kv_heads, pool)
        for group in (1, 2, 3, 4, 8, 16, 64, 128):
            for nodes in list(range(1, 66)) + [96, 127, 128, 129, 200, 255, 256]:
                n = J.tree_attention_workspace(view, q_heads=kv_heads * group, max_nodes=nodes, dtype=dtype)
                assert 0 < n <= J.TREE_WORKSPACE_BYTES


FIRST = """
import sys
sys.path[:0] = {paths!r}
import torch
import jalapeno as J
from tree_util import Call, check_tree, make_trees
for dtype, pool in ({pairs!r})[{which}:] + ({pairs!r})[:{which}]:
    t = make_trees([900, 20], [7, 3], 8, 2, dtype, pool, seed=1, table_pad={pad})
    c = Call.__new__(Call)
    J_ws = J.tree_attention_workspace
    J.tree_attention_workspace = lambda *a, **k: J.TREE_WORKSPACE_BYTES
    c.__init__(t)
    J.tree_attention_workspace = J_ws
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.run()
        g.replay()
    torch.cuda.synchronize()
    check_tree(t, c.out, c.lse)
print("ok")
"""


@pytest.mark.parametrize("pad", [0, WIDE], ids=["clusters", "ranges"])
@pytest.mark.parametrize("which", range(4), ids=IDS)
def test_first_call_is_captured(which, pad):
    """The process's first call of the operator lies in a capture."""
    r = subprocess.run([sys.executable, "-c", FIRST.format(paths=[p for p in sys.path if p], pairs=TYPES, which=which, pad=pad)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
