"""How many bits tree attention keeps: inputs for which every lost bit of a
weight, a value or a sum adds up in one direction."""

import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from tree_util import Call, HEAD, PAGE, make_trees, tree_reference

pytestmark = pytest.mark.gpu

POOLS = pytest.mark.parametrize("pool", [J.KV_BF16, J.KV_F32], ids=["bf16pool", "f32pool"])


def pieces(x, n):
    """x as n bf16 pieces and their sum in 64 bits."""
    out, rest = [], x.double()
    for _ in range(n):
        out.append(rest.to(torch.bfloat16))
        rest = rest - out[-1].double()
    return out, sum(p.double() for p in out)


def one_page(pool, nodes, heads, seed):
    """A sequence of one full page, which all rows see, and nothing else: no row
    sees a node.  scale 1."""
    return make_trees([PAGE], [nodes], heads, 1, J.KV_BF16, pool, bits=[0] * nodes, seed=seed, scale=1.0, device="cpu")


def to_gpu(t):
    for f in ("q", "k", "v", "table"):
        setattr(t, f, getattr(t, f).cuda())
    return t


# What is left in f32, relative to the sum of weighted magnitudes: the
# exponential (2^-22) and its argument (|s| < 8 and c2 once each, 16 * 2^-24), the sum of
# 64 weights in 16 steps and their join (18 * 2^-24), at most 16 additions to the
# accumulator that cut (16 * 2^-23), and the division.
F32 = 2.0 ** -22 + (16 + 18 + 32 + 2) * 2.0 ** -24


def held(out, ref, amp, bits):
    """Rounded once from within `bits` + F32 of the weighted magnitudes."""
    half = 2.0 ** (torch.floor(torch.log2(ref.abs())) - 8)
    far = (out.double() - ref).abs() - half * (1 + 1e-9) - (bits + F32) * amp
    assert (far <= 0).all(), f"{(far > 0).sum().item()} of {far.numel()} outputs too far, by {far.max().item():.3g}"


@POOLS
def test_weights_are_rounded_to_nearest(pool):
    """63 keys with one and the same weight, so that what is lost of it is not
    averaged away, beside one of weight 1 whose value is zero.  Two rounded bf16
    pieces are 2^-17 of a weight off at most."""
    nodes, heads = 64, 8
    t = one_page(pool, nodes, heads, 1)
    g = torch.Generator().manual_seed(2)
    a, score = pieces(0.05 + 4 * torch.rand(nodes * heads, generator=g), 3)
    q = torch.zeros(nodes * heads, HEAD)
    for d, p in enumerate(a):
        q[:, d] = p.float()
    t.q = q.view(nodes, heads * HEAD).to(torch.bfloat16)
    page = t.table[0, 0].long()
    t.k[page] = 0
    t.k[page, :, 1:, :3] = -1
    v = (1 + torch.rand(HEAD, generator=g)).to(torch.bfloat16)
    t.v[page] = v.to(t.v.dtype)
    t.v[page, :, 0] = 0
    w = torch.exp(-score)
    ref = (63 * w / (1 + 63 * w))[:, None] * v.double()
    c = Call(to_gpu(t))
    c.run()
    held(c.out.cpu().view(nodes * heads, HEAD), ref, ref, 2.0 ** -17)


def test_values_of_an_f32_pool():
    """bf16 rows, weights of one: values whose low bits are all ones.  Two bf16
    pieces, the second rounded, are 2^-16 of a value off at most."""
    nodes, heads = 1, 64
    t = one_page(J.KV_F32, nodes, heads, 3)
    g = torch.Generator().manual_seed(4)
    t.q[:] = 0
    out = []
    for _ in range(40):
        bits = torch.randint(0, 2 ** 7, (HEAD,), generator=g) << 16 | 1 << 15 | torch.randint(0, 2 ** 7, (HEAD,), generator=g) << 8 | 255
        v = (bits + (127 << 23)).int().view(torch.float32)  # in [1, 2)
        page = t.table[0, 0].long()
        t.v[page] = v
        c = Call(to_gpu(t))
        c.run()
        out.append((c.out.cpu().view(nodes * heads, HEAD)[:1], v.double()))
        t.v = t.v.cpu()
    held(torch.cat([o for o, _ in out]), torch.stack([v for _, v in out]), torch.stack([v for _, v in out]), 2.0 ** -16)


def test_second_pieces_meet():
    """bf16 rows over an f32 pool: weights and values with second pieces as large
    as they get."""
    nodes, heads = 64, 8
    t = one_page(J.KV_F32, nodes, heads, 5)
    g = torch.Generator().manual_seed(6)
    # weights near 0.5 + 2^-9 - 2^-13 and the like: half a step of the first piece above it
    first = 0.5 + torch.randint(0, 120, (nodes * heads,), generator=g) * 2.0 ** -8
    a, score = pieces(-torch.log(first.double() + 2.0 ** -9 - 2.0 ** -13), 3)
    q = torch.zeros(nodes * heads, HEAD)
    for d, p in enumerate(a):
        q[:, d] = p.float()
    t.q = q.view(nodes, heads * HEAD).to(torch.bfloat16)
    page = t.table[0, 0].long()
    t.k[page] = 0
    t.k[page, :, 1:, :3] = -1
    v = 1 + torch.randint(0, 2 ** 7, (HEAD,), generator=g) * 2.0 ** -7 + 2.0 ** -7 - 2.0 ** -14  # two pieces hold it
    t.v[page] = v.float()
    t.v[page, :, 0] = 0
    w = torch.exp(-score)
    ref = (63 * w / (1 + 63 * w))[:, None] * v.double()
    c = Call(to_gpu(t))
    c.run()
    held(c.out.cpu().view(nodes * heads, HEAD), ref, ref, 2.0 ** -17)


def tails_of_24_bits(pool, rows, seed):
    """Queries, keys, values and weights whose third pieces matter: a row's q and
    the keys' k are one number each with 24 random bits, so that a score is one
    product, the weight of 63 keys its exponential, and the output that weight
    times a value, beside one key of weight 1 and value 0.  Returns (a, kappa, v):
    score -a * kappa; over a bf16 pool kappa is 1 and v is bf16."""
    g = torch.Generator().manual_seed(seed)
    a = (0.05 + 7 * torch.rand(rows, generator=g)).float()
    v = 1 + torch.rand(HEAD, generator=g)
    if pool == J.KV_BF16:
        return a, 1.0, v.to(torch.bfloat16).float()
    return a, float(torch.tensor(1 + 2.0 ** -7 - 2.0 ** -14 - 2.0 ** -16 + 2.0 ** -17, dtype=torch.float32)), v


# A score is below 8; its pieces' products are exact, and of the additions the
# cuts of the first part (two, 2^-23 each) and the two roundings of the parts' sum
# count, 6 half steps of 2^-24, of 8 taken; the weight is off by that relatively.
# The output's own rounding is f32's.
KEPT = F32 + 8 * 8 * 2.0 ** -24 + 2.0 ** -24


def far_of(out, a, kappa, v):
    w = torch.exp(-a.double() * kappa)
    ref = (63 * w / (1 + 63 * w))[:, None] * v.double()
    return ((out.double() - ref).abs() / ref).amax().item()


@POOLS
def test_f32_rows_keep_24_bits(pool):
    """Every third piece, of Q, of the weights and of an f32 pool's K and V: without
    one of them the largest error is several times the bound (next test)."""
    nodes, heads = 64, 8
    t = one_page(pool, nodes, heads, 9)
    a, kappa, v = tails_of_24_bits(pool, nodes * heads, 10)
    q = torch.zeros(nodes * heads, HEAD)
    q[:, 5] = a
    t.q = q.view(nodes, heads * HEAD)
    page = t.table[0, 0].long()
    t.k[page] = 0
    t.k[page, :, 1:, 5] = -kappa
    t.v[page] = v.to(t.v.dtype)
    t.v[page, :, 0] = 0
    c = Call(to_gpu(t))
    c.run()
    assert far_of(c.out.cpu().view(nodes * heads, HEAD), a, kappa, v) <= KEPT


@pytest.mark.parametrize("dtype", [J.KV_F32, J.KV_BF16], ids=["f32", "bf16"])
@POOLS
def test_long_sums(dtype, pool):
    """40 sequences of 12000 positions with values of one sign, so that what the
    additions lose does not cancel.  f32: a run has fewer than 96 additions that cut
    half of 2^-23 of the running sum on average, which is half of its last value
    on average, 96 * 2^-25; runs, weights and parts are added to nearest, 250
    roundings that average out, 16 * 2^-24; and a score's 24 cuts, 24 * 2^-24 of a
    sum whose largest part is below 8, in weights that sum to one.  bf16: the
    rounding, and 512 cuts and the pieces (2^-17 and 2^-16)."""
    seqs, pages, kv_heads = 40, 12, 8
    t = make_trees([700], [1], kv_heads, kv_heads, dtype, pool, seed=7, spare=0)
    assert t.k.shape[0] == pages - 1
    t.v.copy_(1 + t.v.float().abs())
    width = -(-12001 // PAGE)
    g = torch.Generator().manual_seed(8)
    t.table = torch.randint(0, t.k.shape[0], (seqs, width), generator=g).int().cuda()  # pages are shared
    t.ctx, t.nodes, t.bits = [12000 - 31 * s for s in range(seqs)], [1] * seqs, None
    t.q = (1.5 * torch.randn((seqs, kv_heads * HEAD), generator=g)).to(t.q.dtype).cuda()
    c = Call(t)
    c.run()
    ref = tree_reference(t)[0]
    got = c.out.double().view_as(ref)
    off = ((got - ref).norm(dim=(1, 2)) / ref.norm(dim=(1, 2))).max().item()
    if dtype == J.KV_F32:
        assert off < 96 * 2.0 ** -25 + (16 + 24) * 2.0 ** -24, off
    else:
        rounded = ((ref.to(c.out.dtype).double() - ref).norm(dim=(1, 2)) / ref.norm(dim=(1, 2))).max().item()
        bias = ((got - ref).sum() / ref.sum()).abs().item()  # the rounding itself has none
        assert off < 1.02 * rounded and bias < 512 * 2.0 ** -25 + 2.0 ** -17 + 2.0 ** -16, (off, rounded, bias)
    assert c.status.item() == 0
