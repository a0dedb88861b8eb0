"""Cases of the operators of tree-shaped speculation over the paged KV cache.

A speculative round that drafts a tree instead of a chain runs, for each
layer, the norms of queries and keys with the position rotation and the
append to the pages (a node's position is its depth, its slot is its index),
then the attention of the tree's nodes over the committed positions and over
the nodes that each one descends from.  After acceptance the accepted nodes'
rows are moved together in the cache; a sequence that forks shares its full
pages and copies the page it ends in.

``own`` False: the operators in elementary torch operations.  ``own`` True:
the engine's kernels (``jalapenos-at-home_b200/jalapeno.py``).
"""
import math

import torch

own = False

HEAD, HALF, PAGE = 128, 64, 64
ROPE_BASE = 1e6  # Qwen3
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # one sequence of the 0.6B's head layout early in its text, a tree of eight nodes: latency
        dict(name="attn_1seq_8nodes_97", op="attn", seqs=1, q_heads=16, kv_heads=8, nodes=8, ctx=97, rows="f32", pool="bf16",
             tree="random", ragged=False, blank=False, pad=0, lse=False),
        # the 8B verifying a chain of k = 4 drafts and its correction at a 4096-token context
        dict(name="attn_1seq_chain5_4096", op="attn", seqs=1, q_heads=32, kv_heads=8, nodes=5, ctx=4091, rows="f32", pool="bf16",
             tree="chain", ragged=False, blank=False, pad=0, lse=False),
        # a batch of eight with trees of 32 nodes, lengths of their own, and rows that another pass fills
        dict(name="attn_8seq_32nodes_ragged", op="attn", seqs=8, q_heads=32, kv_heads=8, nodes=32, ctx=4300, rows="bf16",
             pool="bf16", tree="random", ragged=True, blank=True, pad=7, lse=True),
        # the largest batch and tree: 32 sequences of 4096 tokens, 64 nodes each
        dict(name="attn_32seq_64nodes_4096", op="attn", seqs=32, q_heads=32, kv_heads=8, nodes=64, ctx=4096, rows="bf16",
             pool="bf16", tree="random", ragged=False, blank=False, pad=0, lse=False),
        # near the context limit, one sequence, a wide shallow tree
        dict(name="attn_1seq_16nodes_40000", op="attn", seqs=1, q_heads=32, kv_heads=8, nodes=16, ctx=40000, rows="bf16",
             pool="bf16", tree="wide", ragged=False, blank=False, pad=0, lse=False),
        # the reference precision: an f32 pool
        dict(name="attn_4seq_12nodes_f32pool", op="attn", seqs=4, q_heads=16, kv_heads=8, nodes=12, ctx=1500, rows="f32",
             pool="f32", tree="random", ragged=True, blank=False, pad=0, lse=False),
        # one verify pass's rows, the 8B's heads
        dict(name="norm_5rows_f32", op="norm", rows_n=5, q_heads=32, kv_heads=8, seqs=1, rows="f32", pool="bf16", skip=False),
        # 32 sequences of 64 nodes; some rows are not appended
        dict(name="norm_2048rows_bf16", op="norm", rows_n=2048, q_heads=32, kv_heads=8, seqs=32, rows="bf16", pool="bf16", skip=True),
        # a long prompt of the 1.7B's heads, odd length
        dict(name="norm_12001rows_f32", op="norm", rows_n=12001, q_heads=16, kv_heads=8, seqs=1, rows="f32", pool="bf16", skip=False),
        # one accepted path of four nodes, all layers of the 8B
        dict(name="compact_1seq_4of16", op="compact", layers=36, kv_heads=8, seqs=1, nodes=16, path=4, ctx=130, pool="bf16"),
        # 32 sequences, up to nine accepted nodes of 64 each
        dict(name="compact_32seq_9of64", op="compact", layers=36, kv_heads=8, seqs=32, nodes=64, path=9, ctx=150, pool="bf16"),
        # eight forks of one prefix: the page each one ends in, partly filled, and 56 whole pages moved together
        dict(name="copy_64pages", op="copy", layers=36, kv_heads=8, pages=64, partial=8, pool="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "norm", "compact", "copy"])
    pool = rng.choice(["bf16", "bf16", "bf16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8])
    if op == "attn":
        group = rng.choice([1, 2, 2, 4, 4, 5, 8])
        seqs, nodes = _log(rng, 1, 32), _log(rng, 1, 96)
        most = 32 * 4096 * 64 * 32 // (4 if pool == "f32" else 1)  # the largest listed case's products
        ctx = _log(rng, 1, max(64, min(40000, most // (seqs * nodes * kv_heads * group), 131072 // seqs)))
        return dict(op="attn", seqs=seqs, q_heads=kv_heads * group, kv_heads=kv_heads, nodes=nodes, ctx=ctx,
                    rows=rng.choice(["f32", "bf16"]), pool=pool, tree=rng.choice(["random", "random", "wide", "chain"]),
                    ragged=rng.random() < 0.6, blank=rng.random() < 0.3, pad=rng.choice([0, 0, 3]), lse=rng.random() < 0.5)
    if op == "norm":
        return dict(op="norm", rows_n=_log(rng, 1, 12000), q_heads=kv_heads * rng.choice([1, 2, 2, 4]), kv_heads=kv_heads,
                    seqs=_log(rng, 1, 32), rows=rng.choice(["f32", "bf16"]), pool=pool, skip=rng.random() < 0.5)
    layers = rng.choice([1, 28, 36, rng.randint(1, 40)])
    if op == "compact":
        nodes = _log(rng, 2, 128)
        return dict(op="compact", layers=layers, kv_heads=kv_heads, seqs=_log(rng, 1, 32), nodes=nodes,
                    path=rng.randint(1, min(nodes, 24)), ctx=rng.randint(0, 200), pool=pool)
    pages = _log(rng, 1, 64 if pool == "bf16" else 32)
    return dict(op="copy", layers=layers, kv_heads=kv_heads, pages=pages, partial=rng.randint(0, pages), pool=pool)


# ---------------------------------------------------------------------------
# inputs


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _host(seed, salt):
    g = torch.Generator()
    g.manual_seed(seed * 7919 + salt)
    return g


def _sizes(case):
    """Committed positions and nodes of each sequence (host lists), by the case alone."""
    n, g = case["seqs"], _host(1, 17)
    ctx, nodes = [case["ctx"]] * n, [case["nodes"]] * n
    if case.get("ragged"):
        u = torch.rand(2, n, generator=g).tolist()
        ctx = [int(round(case["ctx"] * (0.3 + 0.7 * a))) for a in u[0]]
        nodes = [1 + int((case["nodes"] - 1) * b) for b in u[1]]
        ctx[0], nodes[0] = case["ctx"], case["nodes"]
    if case.get("blank"):
        ctx[-1] = 0
    return ctx, nodes


def _tree(kind, n, g):
    """Parents of n nodes (node 0 is the pending token, -1 its parent)."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "wide":
        return [-1] + [0] * (n - 1)
    u = torch.rand(n, generator=g).tolist()
    return [-1] + [int(u[i] * i) for i in range(1, n)]


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def _masks(parents, words):
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return [[_signed(r >> (64 * w) & (1 << 64) - 1) for w in range(words)] for r in rows]


def _pool(layers, pages, kv_heads, dtype, seed, salt):
    """Keys and values of all layers as the engine lays them out."""
    shape = (layers, 2, pages, kv_heads, PAGE, HEAD)
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV, dtype=TYPES[dtype])


def _table(lengths, seed, spare=2):
    """A page table over shuffled pages of the pool: [seqs][most pages], and the pool's pages."""
    need = [max(1, -(-t // PAGE)) for t in lengths]
    most, total = max(need), sum(need) + spare
    order = torch.randperm(total, generator=_host(seed, 5)).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [order[at]] * (most - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), total


def _rope(positions):
    """Cosines and sines of every position's angles: [positions][64][2] f32."""
    f = ROPE_BASE ** (-torch.arange(HALF, device=DEV, dtype=torch.float64) / HALF)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    return {"attn": _prepare_attn, "norm": _prepare_norm, "compact": _prepare_compact, "copy": _prepare_copy}[case["op"]](case, seed)


def _prepare_attn(case, seed):
    (ctx, nodes), g = _sizes(case), _host(seed, 23)
    start = [0]
    for n in nodes:
        start.append(start[-1] + n)
    rows, words = start[-1], -(-case["nodes"] // 64)
    mask = [r for n in nodes for r in _masks(_tree(case["tree"], n, g), words)]
    if case["blank"]:  # a node that sees nothing: its sequence has no committed positions either
        mask[-1] = [0] * words
    table, pages = _table([c + n for c, n in zip(ctx, nodes)], seed)
    dt = TYPES[case["rows"]]
    width = case["q_heads"] * HEAD
    # the q rows lie in the q|k|v rows of a pass
    ld = width + 2 * case["kv_heads"] * HEAD
    qkv = 1.5 * torch.randn((rows + case["pad"], ld), generator=_gen(seed, 1), device=DEV)
    pool = _pool(1, pages, case["kv_heads"], case["pool"], seed, 2)[0]
    return dict(op="attn", rows=rows, seqs=case["seqs"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], most=case["nodes"],
                qkv=qkv.to(dt), pool=pool, table=table, words=words, type=case["rows"], pool_type=case["pool"],
                ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), start=torch.tensor(start, dtype=torch.int32, device=DEV),
                mask=torch.tensor(mask, dtype=torch.int64, device=DEV),
                out=torch.randn((rows + case["pad"], width), generator=_gen(seed, 3), device=DEV).to(dt),
                lse=torch.zeros((rows + case["pad"], case["q_heads"]), device=DEV) if case["lse"] else None,
                work=torch.empty(48 << 20, dtype=torch.uint8, device=DEV))


def _prepare_norm(case, seed):
    n, seqs = case["rows_n"], case["seqs"]
    g = _host(seed, 3)
    per = -(-n // seqs)
    ctx = torch.randint(0, 300, (seqs,), generator=_host(1, 3))
    seq = torch.arange(n) // per
    index = torch.arange(n) % per
    slot = ctx[seq] + index  # rows of one sequence are appended one behind the other
    depth = (torch.rand(n, generator=g) * torch.clamp(index + 1, max=1 << 20)).long() if seqs > 1 else index
    pos = ctx[seq] + depth   # a node's position is its depth
    if case["skip"]:
        slot[torch.rand(n, generator=g) < 0.1] = -1
    table, pages = _table([int(c) + per for c in ctx], seed)
    ld = (case["q_heads"] + 2 * case["kv_heads"]) * HEAD
    dt = TYPES[case["rows"]]
    i32 = lambda t: t.to(torch.int32).to(DEV)  # noqa: E731
    return dict(op="norm", rows=n, seqs=seqs, q_heads=case["q_heads"], kv_heads=case["kv_heads"], type=case["rows"],
                pool_type=case["pool"], qkv=torch.randn((n, ld), generator=_gen(seed, 1), device=DEV).to(dt),
                q=torch.zeros((n, case["q_heads"] * HEAD), dtype=dt, device=DEV),
                qw=(1 + 0.2 * torch.randn(HEAD, generator=_gen(seed, 4), device=DEV)).bfloat16(),
                kw=(1 + 0.2 * torch.randn(HEAD, generator=_gen(seed, 5), device=DEV)).bfloat16(),
                rope=_rope(300 + per), pos=i32(pos), slot=i32(slot), seq=i32(seq), table=table,
                pool=_pool(1, pages, case["kv_heads"], case["pool"], seed, 2)[0])


def _prepare_compact(case, seed):
    n = case["seqs"]
    g = _host(seed, 11)
    ctx = [int(case["ctx"] * (0.5 + 0.5 * u)) for u in torch.rand(n, generator=_host(1, 11)).tolist()]
    path, count = [], []
    for _ in range(n):  # ancestors in order: node 0 (the pending token) first
        k = case["path"] - int(torch.randint(0, max(1, case["path"] // 2), (1,), generator=g))
        path.append([0] + sorted((1 + torch.randperm(case["nodes"] - 1, generator=g)[:case["path"] - 1]).tolist()))
        count.append(k)
    table, pages = _table([c + case["nodes"] for c in ctx], seed)
    return dict(op="compact", layers=case["layers"], seqs=n, kv_heads=case["kv_heads"], pool_type=case["pool"], table=table,
                ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), path=torch.tensor(path, dtype=torch.int32, device=DEV),
                count=torch.tensor(count, dtype=torch.int32, device=DEV),
                pool=_pool(case["layers"], pages, case["kv_heads"], case["pool"], seed, 2))


def _prepare_copy(case, seed):
    n = case["pages"]
    g = _host(seed, 13)
    order = torch.randperm(2 * n, generator=g).tolist()
    dst = order[:n]
    src = order[n:]
    rows = [PAGE] * n
    for i in range(case["partial"]):  # forks of one prefix: the same source page, its filled rows
        src[i] = src[0]
        rows[i] = 1 + int(torch.randint(0, PAGE, (1,), generator=g))
    return dict(op="copy", layers=case["layers"], kv_heads=case["kv_heads"], pool_type=case["pool"], src=src, dst=dst, rows=rows,
                pool=_pool(case["layers"], 2 * n, case["kv_heads"], case["pool"], seed, 2))


# ---------------------------------------------------------------------------
# one pass


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "norm": _plain_norm, "compact": _plain_compact, "copy": _plain_copy}[state["op"]](state)


def _plain_attn(s):
    rows, B, most, Hq, Hk = s["rows"], s["seqs"], s["most"], s["q_heads"], s["kv_heads"]
    width = s["table"].shape[1] * PAGE
    ctx, start = s["ctx"].long(), s["start"].long()
    nodes = start[1:] - start[:-1]
    # rows of each sequence, padded to the largest tree
    j = torch.arange(most, device=DEV)
    live = j < nodes[:, None]
    at = torch.where(live, start[:-1, None] + j, 0)
    q = s["qkv"][:, :Hq * HEAD].float()[at].view(B, most, Hk, Hq // Hk, HEAD)
    keys, values = (s["pool"][i][s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(B, Hk, width, HEAD) for i in (0, 1))
    scores = q.permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, HEAD) @ keys.transpose(2, 3) / math.sqrt(HEAD)
    # visible: the committed positions, and the nodes that the mask has
    p = torch.arange(width, device=DEV)
    node = p - ctx[:, None]
    inside = (node >= 0) & (node < nodes[:, None])
    n = torch.where(inside, node, 0)
    words = s["mask"][at]  # [B][most][words]
    word = words.gather(2, (n >> 6)[:, None, :].expand(B, most, width))
    seen = (node < 0)[:, None, :] | inside[:, None, :] & (word >> (n & 63)[:, None, :] & 1 == 1)
    seen = seen[:, None, :, None, :].expand(B, Hk, most, Hq // Hk, width).reshape(B, Hk, -1, width)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    values = torch.where((p < (ctx + nodes)[:, None])[:, None, :, None], values, 0.0)
    o = weights @ values / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total))[..., 0]
    o = o.view(B, Hk, most, Hq // Hk, HEAD).permute(0, 2, 1, 3, 4).reshape(B, most, Hq * HEAD)
    lse = lse.view(B, Hk, most, Hq // Hk).permute(0, 2, 1, 3).reshape(B, most, Hq)
    # back to the rows; those behind the last sequence stay
    r = torch.arange(rows, device=DEV)
    of = torch.searchsorted(start[1:].contiguous(), r, right=True)
    flat = of * most + r - start[of]
    out = s["out"]
    out[:rows] = o.reshape(B * most, -1)[flat].to(out.dtype)
    if s["lse"] is None:
        return {"out": out}
    s["lse"][:rows] = lse.reshape(B * most, -1)[flat]
    return {"out": out, "lse": s["lse"]}


def _plain_norm(s):
    rows, Hq, Hk = s["rows"], s["q_heads"], s["kv_heads"]
    x = s["qkv"].float().view(rows, Hq + 2 * Hk, HEAD)
    h, v = x[:, :Hq + Hk], x[:, Hq + Hk:]
    w = torch.cat([s["qw"].float().expand(Hq, HEAD), s["kw"].float().expand(Hk, HEAD)])
    h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w
    c, sn = s["rope"][s["pos"].long()].unbind(-1)
    c, sn = c[:, None], sn[:, None]
    a, b = h[..., :HALF], h[..., HALF:]
    h = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    q = h[:, :Hq].reshape(rows, -1).to(s["qkv"].dtype)
    keep = s["slot"] >= 0
    slot = torch.where(keep, s["slot"], 0).long()
    page = s["table"][s["seq"].long(), slot // PAGE].long()
    pool = s["pool"]
    for i, new in ((0, h[:, Hq:]), (1, v)):
        pool[i][page[keep], :, (slot % PAGE)[keep]] = new[keep].to(pool.dtype)
    return {"q": q, "pool": pool}


def _plain_compact(s):
    k = torch.arange(s["path"].shape[1], device=DEV)
    to = s["ctx"].long()[:, None] + k
    of = torch.where(k < s["count"][:, None], s["ctx"].long()[:, None] + s["path"].long(), to)
    p, t = s["pool"], s["table"].long()
    seq = torch.arange(s["seqs"], device=DEV)[:, None]
    p[:, :, t[seq, to // PAGE], :, to % PAGE] = p[:, :, t[seq, of // PAGE], :, of % PAGE]
    return p


def _plain_copy(s):
    p = s["pool"]
    src, dst, rows = (torch.tensor(s[k], device=DEV) for k in ("src", "dst", "rows"))
    whole = (torch.arange(PAGE, device=DEV) < rows[:, None])[:, None, :, None]
    p[:, :, dst] = torch.where(whole, p[:, :, src], p[:, :, dst])
    return p


def _jalapeno():
    import sys
    at = "jalapenos-at-home_b200"
    if at not in sys.path:
        sys.path.insert(0, at)
    import jalapeno
    return jalapeno


def _own(s):
    J = _jalapeno()
    real = {"f32": J.KV_F32, "bf16": J.KV_BF16}
    stream = torch.cuda.current_stream().cuda_stream
    pool = s["pool"]
    half = pool[0].numel() * pool.element_size() // (1 if pool.dim() == 5 else 2)
    pages = J.kv_pages(pool.data_ptr(), pool.data_ptr() + half, pages=pool.shape[-4], kv_heads=s["kv_heads"],
                       dtype=real[s["pool_type"]], layers=1 if pool.dim() == 5 else s["layers"], layer_stride=2 * half)
    if s["op"] == "attn":
        J.tree_attention(pages, q=s["qkv"].data_ptr(), q_ld=s["qkv"].shape[1], out=s["out"].data_ptr(), out_ld=s["out"].shape[1],
                         rows=s["rows"], q_heads=s["q_heads"], dtype=real[s["type"]], seqs=s["seqs"], max_nodes=s["most"],
                         row_start=s["start"].data_ptr(), ctx=s["ctx"].data_ptr(), mask=s["mask"].data_ptr(), mask_words=s["words"],
                         page_table=s["table"].data_ptr(), max_pages=s["table"].shape[1],
                         lse=0 if s["lse"] is None else s["lse"].data_ptr(), workspace=s["work"].data_ptr(),
                         workspace_bytes=s["work"].numel(), stream=stream)
        return {"out": s["out"]} if s["lse"] is None else {"out": s["out"], "lse": s["lse"]}
    if s["op"] == "norm":
        J.qk_norm_rope(pages, qkv=s["qkv"].data_ptr(), qkv_ld=s["qkv"].shape[1], q=s["q"].data_ptr(), q_ld=s["q"].shape[1],
                       rows=s["rows"], q_heads=s["q_heads"], dtype=real[s["type"]], q_norm=s["qw"].data_ptr(), k_norm=s["kw"].data_ptr(),
                       eps=EPS, rope=s["rope"].data_ptr(), positions=s["rope"].shape[0], pos=s["pos"].data_ptr(),
                       slot=s["slot"].data_ptr(), seq=s["seq"].data_ptr(), page_table=s["table"].data_ptr(), seqs=s["seqs"],
                       max_pages=s["table"].shape[1], stream=stream)
        return {"q": s["q"], "pool": pool}
    if s["op"] == "compact":
        J.kv_compact(pages, seqs=s["seqs"], ctx=s["ctx"].data_ptr(), path=s["path"].data_ptr(), path_ld=s["path"].shape[1],
                     path_len=s["count"].data_ptr(), page_table=s["table"].data_ptr(), max_pages=s["table"].shape[1], stream=stream)
        return pool
    J.kv_copy_pages(pages, s["src"], s["dst"], s["rows"], stream=stream)
    return pool


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    el = {"f32": 4, "bf16": 2}
    if case["op"] == "attn":
        ctx, nodes = _sizes(case)
        keys = sum(c + n for c, n in zip(ctx, nodes))
        rows = sum(nodes)
        kv = 2 * keys * case["kv_heads"] * HEAD * el[case["pool"]]
        io = 2 * rows * case["q_heads"] * HEAD * el[case["rows"]] + rows * (8 * -(-case["nodes"] // 64) + 4 * case["q_heads"] * case["lse"])
        pairs = sum((c + (n + 1) / 2) * n for c, n in zip(ctx, nodes))
        return {"bytes": kv + io, "flops": 4 * pairs * case["q_heads"] * HEAD}
    if case["op"] == "norm":
        n, heads = case["rows_n"], case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": n * HEAD * (heads * el[case["rows"]] + case["q_heads"] * el[case["rows"]] + 2 * case["kv_heads"] * el[case["pool"]]
                                     + 4) + 12 * n, "flops": n * HEAD * (case["q_heads"] + case["kv_heads"]) * 8}
    row = 2 * case["layers"] * case["kv_heads"] * HEAD * el[case["pool"]]  # one position, all layers
    if case["op"] == "compact":
        mean = case["path"] - (max(1, case["path"] // 2) - 1) / 2
        return {"bytes": 2 * row * mean * case["seqs"], "flops": 0}
    return {"bytes": 2 * row * (PAGE * case["pages"] - case["partial"] * (PAGE - 1) / 2), "flops": 0}


# ---------------------------------------------------------------------------
# the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "attn":
        Hq, Hk = case["q_heads"], case["kv_heads"]
        out, lse = s["out"].to(f), None if s["lse"] is None else s["lse"].to(f)
        start, ctx, table, masks = s["start"].tolist(), s["ctx"].tolist(), s["table"].long(), s["mask"].tolist()
        for b in range(case["seqs"]):
            lo, hi, c = start[b], start[b + 1], ctx[b]
            n = hi - lo
            k, v = (s["pool"][i][table[b]].to(f).transpose(0, 1).flatten(1, 2)[:, :c + n] for i in (0, 1))
            bits = torch.tensor([[masks[r][t // 64] >> (t % 64) & 1 for t in range(n)] for r in range(lo, hi)], device=DEV).bool()
            seen = torch.cat([torch.ones((n, c), dtype=torch.bool, device=DEV), bits], 1)
            some = seen.any(1)
            q = s["qkv"][lo:hi, :Hq * HEAD].to(f).view(n, Hq, HEAD)
            for h in range(Hq):
                x = (q[:, h] @ k[h // (Hq // Hk)].T / HEAD ** 0.5).masked_fill(~seen, -math.inf)
                z = torch.logsumexp(x, 1)
                w = torch.exp(x - torch.where(some, z, 0.0)[:, None])
                out[lo:hi, h * HEAD:(h + 1) * HEAD] = w @ v[h // (Hq // Hk)]
                if lse is not None:
                    lse[lo:hi, h] = z
        return {"out": out} if lse is None else {"out": out, "lse": lse}
    if case["op"] == "norm":
        n, Hq, Hk = case["rows_n"], case["q_heads"], case["kv_heads"]
        x = s["qkv"].to(f).view(n, Hq + 2 * Hk, HEAD)
        z = torch.complex(s["rope"][..., 0].to(f), s["rope"][..., 1].to(f))[s["pos"].long()][:, None]

        def turn(part, w):
            y = part * torch.rsqrt(part.square().sum(-1, keepdim=True) / HEAD + EPS) * w.to(f)
            t = torch.complex(y[..., :HALF], y[..., HALF:]) * z
            return torch.cat([t.real, t.imag], -1)

        pool = s["pool"].to(f)
        k, v = turn(x[:, Hq:Hq + Hk], s["kw"]), x[:, Hq + Hk:]
        put = (s["slot"] >= 0).nonzero()[:, 0]
        at = s["slot"][put].long()
        page = s["table"][s["seq"][put].long(), at // PAGE].long()
        where = (page[:, None], torch.arange(Hk, device=DEV)[None], (at % PAGE)[:, None])
        pool[0].index_put_(where, k[put])
        pool[1].index_put_(where, v[put])
        return {"q": turn(x[:, :Hq], s["qw"]).reshape(n, -1), "pool": pool}
    if case["op"] == "compact":
        old, new, table = s["pool"], s["pool"].clone(), s["table"].tolist()
        for b, (c, k) in enumerate(zip(s["ctx"].tolist(), s["count"].tolist())):
            for i, node in enumerate(s["path"][b].tolist()[:k]):
                (a, t), (e, u) = divmod(c + node, PAGE), divmod(c + i, PAGE)
                new[:, :, table[b][e], :, u] = old[:, :, table[b][a], :, t]
        return new
    new = s["pool"].clone()
    for a, b, n in zip(s["src"], s["dst"], s["rows"]):
        new[:, :, b, :, :n] = s["pool"][:, :, a, :, :n]
    return new
