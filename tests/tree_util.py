"""Definitions, in 64 bits, of the operators of tree-shaped speculation, and
random inputs for them (torch tensors on any device)."""
from __future__ import annotations

import dataclasses
import math

import torch

import jalapeno as J

HEAD, PAGE = 128, 64
TYPES = {J.KV_F32: torch.float32, J.KV_BF16: torch.bfloat16}


def half_step(dtype) -> float:
    """Largest relative error of rounding to `dtype` once."""
    return torch.finfo(dtype).eps / 2


def ancestors(parents):
    """Rows of the tree's mask as Python integers: a node sees itself and the
    nodes it descends from."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return rows


def mask_words(rows, words, device):
    """[rows][words] int64 whose bits are those of the Python integers."""
    out = torch.zeros((len(rows), words), dtype=torch.int64)
    for i, r in enumerate(rows):
        for w in range(words):
            x = r >> (64 * w) & (1 << 64) - 1
            out[i, w] = x - (1 << 64) if x >> 63 else x
    return out.to(device)


@dataclasses.dataclass
class Trees:
    """Inputs of one tree_attention call."""
    q: torch.Tensor         # [rows + pad][q_ld]
    k: torch.Tensor         # [pages][kv_heads][64][128]
    v: torch.Tensor
    table: torch.Tensor     # [seqs][max_pages]
    ctx: list
    nodes: list
    bits: list              # a mask (Python integer) per row, or None: chains
    q_heads: int
    scale: float = 0.0

    @property
    def rows(self):
        return sum(self.nodes)

    def starts(self):
        s = [0]
        for n in self.nodes:
            s.append(s[-1] + n)
        return s


def make_trees(ctx, nodes, q_heads=4, kv_heads=2, dtype=J.KV_F32, pool=J.KV_BF16, bits="random", seed=0, pad=0,
               extra_ld=0, spare=3, table_pad=0, device="cuda", scale=0.0):
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-(c + n) // PAGE)) for c, n in zip(ctx, nodes)]
    most, total = max(need) + table_pad, sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (most - n))  # past the sequence: no page
        at += n
    shape = (total, kv_heads, PAGE, HEAD)
    k, v = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
    q = 1.5 * torch.randn((sum(nodes) + pad, q_heads * HEAD + extra_ld), generator=g)
    if bits == "random":
        bits = []
        for n in nodes:
            u = torch.rand(n, generator=g).tolist()
            bits += ancestors([-1] + [int(u[i] * i) for i in range(1, n)] if n else [])
    return Trees(q.to(TYPES[dtype]).to(device), k.to(TYPES[pool]).to(device), v.to(TYPES[pool]).to(device),
                 torch.tensor(rows, dtype=torch.int32, device=device), list(ctx), list(nodes), bits, q_heads, scale)


def tree_reference(t: Trees):
    """(out, lse, spread) of every row in 64 bits; spread bounds the weighted
    mean of |v| and the rounding of the scores, for the tolerances."""
    f, dev = torch.float64, t.q.device
    pages, kv_heads = t.k.shape[:2]
    group = t.q_heads // kv_heads
    out = torch.zeros((t.rows, t.q_heads, HEAD), dtype=f, device=dev)
    lse = torch.full((t.rows, t.q_heads), -math.inf, dtype=f, device=dev)
    amp = torch.zeros((t.rows, t.q_heads), dtype=f, device=dev)     # sum of w |v|, largest dim
    noise = torch.zeros((t.rows, t.q_heads), dtype=f, device=dev)   # largest sum |q_i k_i| * scale
    scale = t.scale or HEAD ** -0.5
    start, table = t.starts(), t.table.cpu().tolist()
    for s, (c, n) in enumerate(zip(t.ctx, t.nodes)):
        for j in range(n):
            r = start[s] + j
            seen = list(range(c)) + [c + i for i in range(n) if (t.bits[r] >> i & 1 if t.bits is not None else i <= j)]
            seen = [p for p in seen if p // PAGE < len(table[s]) and 0 <= table[s][p // PAGE] < pages]
            if not seen:
                continue
            pg = torch.tensor([table[s][p // PAGE] for p in seen], device=dev)
            at = torch.tensor([p % PAGE for p in seen], device=dev)
            k, v = t.k[pg, :, at].to(f), t.v[pg, :, at].to(f)       # [seen][kv_heads][128]
            q = t.q[r, :t.q_heads * HEAD].to(f).view(kv_heads, group, HEAD)
            x = torch.einsum("hgd,phd->hgp", q, k) * scale
            z = torch.logsumexp(x, -1)
            w = torch.exp(x - z[..., None])
            out[r] = torch.einsum("hgp,phd->hgd", w, v).reshape(t.q_heads, HEAD)
            lse[r] = z.reshape(-1)
            amp[r] = torch.einsum("hgp,phd->hgd", w, v.abs()).amax(-1).reshape(-1)
            noise[r] = (torch.einsum("hgd,phd->hgp", q.abs(), k.abs()).amax(-1) * scale).reshape(-1)
    return out, lse, amp, noise


def check_tree(t: Trees, out, lse=None):
    """Holds a call's outputs to the definition.  A score is a sum of 128
    products and carries at most 128 half steps of f32 of the sum of their
    magnitudes (`noise`); a weight then is off by twice that relatively
    (numerator and sum), plus eight f32 half steps for the exponential, the
    running sums and the joins; an output by that much of `amp`, and by the
    rounding into its type."""
    ref, z, amp, noise = tree_reference(t)
    e = 2.0 ** -24
    slack = 2 * 128 * e * noise + 8 * e + 2.0 ** -21  # and the exponential's own 2^-22 twice
    got = out[:t.rows, :t.q_heads * HEAD].double().view(t.rows, t.q_heads, HEAD)
    bound = half_step(out.dtype) * ref.abs() * (1 + 1e-6) + (slack * amp)[..., None] + 1e-30
    far = (got - ref).abs() - bound
    assert torch.isfinite(got).all()
    assert (far <= 0).all(), f"off by {far.max().item():.3g} past the bound (rel L2 {((got - ref).norm() / ref.norm()).item():.3g})"
    if lse is not None:
        got = lse[:t.rows].double()
        none = z == -math.inf
        assert torch.equal(got == -math.inf, none)
        assert ((got - z).abs()[~none] <= (slack + 4 * e * z.abs())[~none]).all()
    return ((out[:t.rows, :t.q_heads * HEAD].double().view_as(ref) - ref).norm() / ref.norm().clamp_min(1e-30)).item()


class Call:
    """A tree_attention call's device buffers."""

    def __init__(self, t: Trees, max_nodes=None, lse=True, status=True, device="cuda"):
        self.t = t
        dev = t.q.device
        self.pool_type = J.KV_F32 if t.k.dtype == torch.float32 else J.KV_BF16
        self.dtype = J.KV_F32 if t.q.dtype == torch.float32 else J.KV_BF16
        self.max_nodes = max_nodes or max(max(t.nodes), 1)
        self.words = -(-self.max_nodes // 64)
        self.mask = None if t.bits is None else mask_words(t.bits, self.words, dev)
        self.start = torch.tensor(t.starts(), dtype=torch.int32, device=dev)
        self.ctx = torch.tensor(t.ctx, dtype=torch.int32, device=dev)
        self.out = torch.full((t.q.shape[0], t.q_heads * HEAD), 7.5, dtype=t.q.dtype, device=dev)
        self.lse = torch.full((t.q.shape[0], t.q_heads), 7.5, device=dev) if lse else None
        self.status = torch.zeros(1, dtype=torch.int32, device=dev) if status else None
        self.pool = J.kv_pages(t.k.data_ptr(), t.v.data_ptr(), t.k.shape[0], t.k.shape[1], self.pool_type)
        self.work = torch.full((J.tree_attention_workspace(self.pool, q_heads=t.q_heads, max_nodes=self.max_nodes,
                                                           dtype=self.dtype) + 16,), 255, dtype=torch.uint8, device=dev)

    def args(self, **kw):
        t = self.t
        a = dict(q=t.q.data_ptr(), q_ld=t.q.shape[1], out=self.out.data_ptr(), out_ld=self.out.shape[1], rows=t.rows,
                 q_heads=t.q_heads, seqs=len(t.nodes), max_nodes=self.max_nodes, row_start=self.start.data_ptr(),
                 ctx=self.ctx.data_ptr(), page_table=t.table.data_ptr(), max_pages=t.table.shape[1],
                 workspace=self.work.data_ptr(), workspace_bytes=self.work.numel(),
                 mask=0 if self.mask is None else self.mask.data_ptr(), mask_words=self.words, dtype=self.dtype,
                 scale=t.scale, lse=0 if self.lse is None else self.lse.data_ptr(),
                 status=0 if self.status is None else self.status.data_ptr(),
                 stream=torch.cuda.current_stream(t.q.device).cuda_stream)
        a.update(kw)
        return a

    def run(self, **kw):
        J.tree_attention(self.pool, **self.args(**kw))
        return self.out

    def checked(self, **kw):
        """Runs and checks: outputs, untouched rows, no status, and the same
        bits from a second call."""
        self.run(**kw)
        first = self.out.clone()
        rel = check_tree(self.t, self.out, self.lse)
        assert (self.out[self.t.rows:] == 7.5).all()
        if self.lse is not None:
            assert (self.lse[self.t.rows:] == 7.5).all()
        if self.status is not None:
            assert self.status.item() == 0
        self.run(**kw)
        assert torch.equal(first, self.out)
        return rel
