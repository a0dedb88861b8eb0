"""Norm, rotation and append of q|k|v rows (jl_qk_norm_rope), compaction
(jl_kv_compact) and copies of cache pages (jl_kv_copy_pages) against their
definitions."""
import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from tree_util import HEAD, PAGE, TYPES, half_step

pytestmark = pytest.mark.gpu

HALF = HEAD // 2
both = pytest.mark.parametrize("dtype,pool", [(J.KV_F32, J.KV_BF16), (J.KV_BF16, J.KV_BF16), (J.KV_F32, J.KV_F32),
                                              (J.KV_BF16, J.KV_F32)], ids=["f32-bf16", "bf16-bf16", "f32-f32", "bf16-f32"])


def rope_table(n, base=1e6):
    f = base ** (-torch.arange(HALF, dtype=torch.float64) / HALF)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().cuda()


class Rows:
    def __init__(self, n, q_heads, kv_heads, dtype, pool, seqs=3, max_pages=4, extra=0, seed=0, positions=500):
        g = torch.Generator().manual_seed(seed)
        self.n, self.q_heads, self.kv_heads, self.dtype, self.pool_type = n, q_heads, kv_heads, dtype, pool
        self.ld = (q_heads + 2 * kv_heads) * HEAD + extra
        self.qkv = torch.randn((n, self.ld), generator=g).to(TYPES[dtype]).cuda()
        self.q = torch.full((n + 1, q_heads * HEAD + extra), 3.0, dtype=TYPES[dtype], device="cuda")
        self.qw = (1 + 0.3 * torch.randn(HEAD, generator=g)).bfloat16().cuda()
        self.kw = (1 + 0.3 * torch.randn(HEAD, generator=g)).bfloat16().cuda()
        self.rope = rope_table(positions)
        pages = seqs * max_pages + 2
        self.table = torch.randperm(pages, generator=g)[:seqs * max_pages].view(seqs, max_pages).int().cuda()
        self.k = torch.randn((pages, kv_heads, PAGE, HEAD), generator=g).to(TYPES[pool]).cuda()
        self.v = torch.randn((pages, kv_heads, PAGE, HEAD), generator=g).to(TYPES[pool]).cuda()
        places = torch.randperm(seqs * max_pages * PAGE, generator=g)[:n]  # distinct places
        self.seq = (places // (max_pages * PAGE)).int().cuda()
        self.slot = (places % (max_pages * PAGE)).int().cuda()
        self.pos = torch.randint(0, positions, (n,), generator=g).int().cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.eps = 1e-6

    def run(self, **kw):
        a = dict(qkv=self.qkv.data_ptr(), qkv_ld=self.ld, q=self.q.data_ptr(), q_ld=self.q.shape[1], rows=self.n,
                 q_heads=self.q_heads, rope=self.rope.data_ptr(), positions=self.rope.shape[0], pos=self.pos.data_ptr(),
                 page_table=self.table.data_ptr(), max_pages=self.table.shape[1], dtype=self.dtype,
                 q_norm=self.qw.data_ptr(), k_norm=self.kw.data_ptr(), eps=self.eps, slot=self.slot.data_ptr(),
                 seq=self.seq.data_ptr(), seqs=self.table.shape[0], status=self.status.data_ptr(),
                 stream=torch.cuda.current_stream().cuda_stream)
        a.update(kw)
        J.qk_norm_rope(J.kv_pages(self.k.data_ptr(), self.v.data_ptr(), self.k.shape[0], self.kv_heads, self.pool_type), **a)

    def want(self, qw=True, kw=True):
        """(q, k pool, v pool) in 64 bits from the current inputs."""
        f = torch.float64
        x = self.qkv[:, :(self.q_heads + 2 * self.kv_heads) * HEAD].to(f).view(self.n, -1, HEAD)
        ok = (self.pos >= 0) & (self.pos < self.rope.shape[0])
        cs = self.rope.to(f)[torch.where(ok, self.pos, 0).long()][:, None]

        def turn(y, w):
            if w is not None:
                y = y / (y.square().mean(-1, keepdim=True) + self.eps).sqrt() * w.to(f)
            a, b = y[..., :HALF], y[..., HALF:]
            return torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)

        q = self.q.to(f).clone()
        new = turn(x[:, :self.q_heads], self.qw if qw else None).reshape(self.n, -1)
        q[:self.n, :self.q_heads * HEAD][ok] = new[ok]
        kk = turn(x[:, self.q_heads:self.q_heads + self.kv_heads], self.kw if kw else None)
        k, v = self.k.to(f).clone(), self.v.to(f).clone()
        slot, seq, table = self.slot.tolist(), self.seq.tolist(), self.table.tolist()
        for r in range(self.n):
            if ok[r] and 0 <= slot[r] < len(table[0]) * PAGE and 0 <= seq[r] < len(table):
                page = table[seq[r]][slot[r] // PAGE]
                if 0 <= page < k.shape[0]:
                    k[page, :, slot[r] % PAGE] = kk[r]
                    v[page, :, slot[r] % PAGE] = x[r, self.q_heads + self.kv_heads:]
        return q, k, v

    def check(self, want):
        """One rounding into the output's type, and in f32: the sum of 128
        squares (64 half steps after the root), the root, the division, three
        products and a sum: 72 half steps of a magnitude of at most the two
        terms of the rotation."""
        for got, ref in zip((self.q, self.k, self.v), want):
            size = ref.abs()
            near = torch.cat([size[..., HALF:], size[..., :HALF]], -1) if got.dim() == 4 else None
            if near is None:
                w = self.q_heads * HEAD
                y = size[:, :w].reshape(size.shape[0], self.q_heads, 2, HALF)
                near = size.clone()
                near[:, :w] = y.flip(2).reshape(size.shape[0], w)
            slack = 72 * 2.0 ** -24 * 2 * (size + near)  # |a|, |b| <= |rotated pair| (both of its parts together)
            assert ((got.double() - ref).abs() <= half_step(got.dtype) * size * (1 + 1e-4) + slack + 1e-30).all()


@both
@pytest.mark.parametrize("n,q_heads,kv_heads", [(1, 1, 1), (5, 32, 8), (64, 16, 8), (300, 6, 2), (700, 5, 5)])
def test_norm_rope(dtype, pool, n, q_heads, kv_heads):
    r = Rows(n, q_heads, kv_heads, dtype, pool, extra=8, seed=n)
    want = r.want()
    r.run()
    r.check(want)
    assert r.status.item() == 0


@both
def test_in_place(dtype, pool):
    r = Rows(37, 8, 2, dtype, pool, seed=1)
    want, rest = r.want(), r.qkv[:, 8 * HEAD:].clone()
    r.run(q=r.qkv.data_ptr(), q_ld=r.ld)
    assert torch.equal(r.qkv[:, 8 * HEAD:], rest)
    r.q[:37] = r.qkv[:, :8 * HEAD]
    r.check(want)


@both
def test_defaults(dtype, pool):
    """No slots (slot is the position), no sequences (sequence 0), no norms."""
    r = Rows(50, 4, 2, dtype, pool, seqs=1, seed=2, positions=256)
    r.slot = torch.randperm(256)[:50].int().cuda()
    r.pos, r.seq = r.slot, torch.zeros_like(r.slot)
    want = r.want(qw=False, kw=False)
    r.run(slot=0, seq=0, q_norm=0, k_norm=0)
    r.check(want)


@both
def test_only_keys_are_normed(dtype, pool):
    r = Rows(9, 4, 2, dtype, pool, seed=3)
    want = r.want(qw=False)
    r.run(q_norm=0)
    r.check(want)


@both
def test_rows_that_are_not_appended(dtype, pool):
    r = Rows(60, 4, 2, dtype, pool, seed=4)
    r.slot[::3] = -1
    r.slot[1] = -2 ** 31
    want = r.want()
    r.run()
    r.check(want)
    assert r.status.item() == 0


@pytest.mark.parametrize("what,bits", [("pos", 2), ("pos_low", 2), ("slot", 2), ("seq", 2), ("page", 1)])
def test_indices_out_of_range_are_skipped(what, bits):
    r = Rows(20, 4, 2, J.KV_F32, J.KV_BF16, seed=5)
    if what == "pos":
        r.pos[3] = r.rope.shape[0]
    if what == "pos_low":
        r.pos[3] = -1
    if what == "slot":
        r.slot[3] = 4 * PAGE
    if what == "seq":
        r.seq[3] = 3
    if what == "page":
        r.table[r.seq[3].long(), (r.slot[3] // PAGE).long()] = r.k.shape[0]
    want = r.want()
    r.run()
    r.check(want)
    assert r.status.item() == bits
    r.run(status=0)  # the word may be left out


def test_zero_and_huge_rows():
    """A row of zeros stays zero (eps keeps the division finite); squares that
    are large but finite do not overflow."""
    r = Rows(3, 2, 1, J.KV_F32, J.KV_F32, seed=6)
    r.qkv[0] = 0
    r.qkv[1] *= 1e15
    want = r.want()
    r.run()
    assert (r.q[0, :2 * HEAD] == 0).all()
    r.check(want)


# ---- compaction ---------------------------------------------------------------------


class Moves:
    def __init__(self, seqs, ctx, paths, layers=3, kv_heads=2, pool=J.KV_BF16, seed=0, max_pages=6):
        g = torch.Generator().manual_seed(seed)
        self.pages, self.layers, self.kv_heads = seqs * max_pages + 1, layers, kv_heads
        self.pool = torch.randn((layers, 2, self.pages, kv_heads, PAGE, HEAD), generator=g).to(TYPES[pool]).cuda()
        self.table = torch.randperm(self.pages, generator=g)[:seqs * max_pages].view(seqs, max_pages).int().cuda()
        self.ctx, self.paths = ctx, paths
        self.ld = max(1, max(len(p) for p in paths))
        self.path = torch.tensor([p + [0] * (self.ld - len(p)) for p in paths], dtype=torch.int32, device="cuda")
        self.len = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
        self.dctx = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        half = self.pool[0, 0].numel() * self.pool.element_size()
        self.view = J.kv_pages(self.pool.data_ptr(), self.pool.data_ptr() + half, self.pages, kv_heads, pool, layers, 2 * half)

    def want(self):
        new, table = self.pool.clone(), self.table.tolist()
        for s, (c, path) in enumerate(zip(self.ctx, self.paths)):
            for i, node in enumerate(path):
                (a, t), (b, u) = divmod(c + node, PAGE), divmod(c + i, PAGE)
                if a < len(table[s]) and b < len(table[s]):
                    new[:, :, table[s][b], :, u] = self.pool[:, :, table[s][a], :, t]
        return new

    def run(self, **kw):
        a = dict(seqs=len(self.ctx), ctx=self.dctx.data_ptr(), path=self.path.data_ptr(), path_ld=self.ld,
                 path_len=self.len.data_ptr(), page_table=self.table.data_ptr(), max_pages=self.table.shape[1],
                 status=self.status.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        a.update(kw)
        J.kv_compact(self.view, **a)


@pytest.mark.parametrize("pool", [J.KV_BF16, J.KV_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("ctx,paths", [
    ([0], [[0]]), ([10], [[0, 2, 5]]), ([62], [[0, 1, 3, 9]]), ([63, 64, 0], [[1, 2], [], [0, 7, 8, 30]]),
    ([5], [[3, 2, 1, 0]]),                       # any order
    ([60], [[7, 7, 0, 7]]),                      # repeated entries
    ([100], [list(range(1, 200))]),              # a long path over four pages
    ([7, 9, 64, 128], [[0, 4, 6, 8, 11, 15, 16, 20, 31, 40, 41, 44, 50, 51, 60, 61, 63]] * 4)])
def test_compaction(pool, ctx, paths):
    m = Moves(len(ctx), ctx, paths, pool=pool, seed=len(paths[0]))
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want)
    assert m.status.item() == 0


def test_compaction_out_of_range_is_skipped():
    m = Moves(2, [300, 20], [[0, 200], [0, 3]], seed=1)
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want) and m.status.item() == 2
    m = Moves(1, [20], [[2, 5]], seed=2)
    m.table[0, 0] = m.pages
    want = m.pool.clone()
    m.run()
    assert torch.equal(m.pool, want) and m.status.item() == 1
    m = Moves(1, [20], [[2, -1, 5]], seed=2)
    m.paths = [[2, 1, 5]]  # the negative entry is left out, the others move
    want = m.want()
    m.run()
    assert torch.equal(m.pool, want) and m.status.item() == 2


# ---- copies of pages -----------------------------------------------------------------


@pytest.mark.parametrize("pool", [J.KV_BF16, J.KV_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layers,kv_heads,n", [(1, 1, 1), (3, 2, 5), (2, 3, 64), (1, 2, 65), (2, 1, 1500)])
def test_page_copies(pool, layers, kv_heads, n):
    g = torch.Generator().manual_seed(n)
    pages = 2 * n + 1
    p = torch.randn((layers, 2, pages, kv_heads, PAGE, HEAD), generator=g).to(TYPES[pool]).cuda()
    order = torch.randperm(pages, generator=g).tolist()
    dst, src = order[:n], order[n:2 * n]
    if n > 3:
        src[1] = src[2] = src[0]
    rows = torch.randint(1, PAGE + 1, (n,), generator=g).tolist()
    half = p[0, 0].numel() * p.element_size()
    view = J.kv_pages(p.data_ptr(), p.data_ptr() + half, pages, kv_heads, pool, layers, 2 * half)
    for r in (rows, None):
        want = p.clone()
        for a, b, m in zip(src, dst, r or [PAGE] * n):
            want[:, :, b, :, :m] = p[:, :, a, :, :m]
        J.kv_copy_pages(view, src, dst, r, stream=torch.cuda.current_stream().cuda_stream)
        assert torch.equal(p, want)


def test_captured_moves():
    """A captured copy carries its page list; a captured compaction reads its
    paths at each replay."""
    m = Moves(1, [10], [[0, 3, 4]], seed=9)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            m.run()
            src, dst = [0], [1]
            J.kv_copy_pages(m.view, src, dst, [17], stream=st.cuda_stream)
            del src, dst
        for path in ([0, 3, 4], [1, 2, 9]):
            m.paths = [path]
            m.path.copy_(torch.tensor([path]))
            want = m.want()
            want[:, :, 1, :, :17] = want[:, :, 0, :, :17].clone()
            g.replay()
            st.synchronize()
            assert torch.equal(m.pool, want)
