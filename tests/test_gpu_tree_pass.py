"""Trees of drafted tokens on a model's cache (jl_predict_tree,
jl_cache_compact) and forks of a cache (jl_cache_fork).

A node's prediction must be that of its path predicted as a chain: against the
engine's own passes on a fork of the cache and against the oracle.  Tolerances:
an f32 pool is held to the engine's own bound of 1e-5 relative L2 (the kernels
differ in summation order only); on a bf16 pool last-bit differences of f32 K/V
round to neighbouring bf16 values, which alone reaches 1e-4 (see
test_gpu_prefill_tc.py), so logits are held to 2e-4."""
import dataclasses
import gc

import numpy as np
import pytest

import jalapeno as J
import oracle as O
from gpu_util import compare_streams, rel_l2, top2_margin

pytestmark = pytest.mark.gpu

TINY = O.PRESETS["tiny"]
DRAFT = O.PRESETS["tiny-draft"]
TOL = {J.KV_F32: 1e-5, J.KV_BF16: 2e-4}


def config(q_heads=8, kv_heads=2, **kw):
    return dataclasses.replace(TINY, name=f"tiny-q{q_heads}-kv{kv_heads}", q_heads=q_heads, kv_heads=kv_heads,
                               max_positions=1024, **kw)


def tree(n, vocab, seed):
    rng = np.random.default_rng(seed)
    parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, n)]
    return O.prompt_ids(n, vocab, seed), parents


def path_of(node, parents):
    p = []
    while node >= 0:
        p.append(node)
        node = parents[node]
    return p[::-1]


def same_ids(ids, lg, want_ids, want_lg):
    for i, (a, b) in enumerate(zip(ids, want_ids)):
        assert a == b or top2_margin(want_lg[i]) < 1e-3, (i, a, b)


@pytest.mark.parametrize("kv", [J.KV_BF16, J.KV_F32], ids=["bf16pool", "f32pool"])
@pytest.mark.parametrize("mxfp4", [True, False], ids=["mxfp4", "bf16"])
@pytest.mark.parametrize("ctx,n", [(0, 1), (1, 5), (63, 16), (64, 17), (130, 40), (200, 100)])
def test_nodes_predict_as_their_paths(kv, mxfp4, ctx, n):
    cfg = config()
    m = J.Model.from_config(cfg, 3, mxfp4=mxfp4, kv_dtype=kv)
    c = m.cache()
    if ctx:
        m.predict(O.prompt_ids(ctx, cfg.vocab, 5), c)
    tokens, parents = tree(n, cfg.vocab, 7 + n)
    ids, lg = m.predict_tree(tokens, parents, c, logits=True)
    assert c.len == ctx
    for node in range(0, n, max(1, n // 12)):
        f = c.fork()
        want, wlg = m.predict([tokens[i] for i in path_of(node, parents)], f, logits=True)
        assert rel_l2(lg[node], wlg[0]) < TOL[kv], (node, rel_l2(lg[node], wlg[0]))
        same_ids([ids[node]], lg[node:node + 1], want, wlg)


@pytest.mark.parametrize("heads", [(2, 2), (4, 2), (16, 2), (6, 2)], ids=["group1", "group2", "group8", "group3"])
def test_against_the_oracle(heads):
    cfg = config(*heads, layers=2)
    ref = O.Model.synthetic(cfg, 3, mxfp4=True)
    m = J.Model.from_config(cfg, 3, mxfp4=True)
    prompt = O.prompt_ids(90, cfg.vocab, 5)
    tokens, parents = tree(21, cfg.vocab, 1)
    c = m.cache()
    m.predict(prompt, c)
    ids, lg = m.predict_tree(tokens, parents, c, logits=True)
    for node in (0, 3, 8, 20):
        rc = ref.cache(round_bf16=True)
        want, wlg = ref.predict(prompt + [tokens[i] for i in path_of(node, parents)], rc, logits=True)
        assert rel_l2(lg[node], wlg[0]) < 2e-4
        same_ids([ids[node]], lg[node:node + 1], want, wlg)


def test_a_chain_predicts_as_predict():
    cfg = config()
    m = J.Model.from_config(cfg, 4, mxfp4=True, kv_dtype=J.KV_F32)
    c = m.cache()
    m.predict(O.prompt_ids(70, cfg.vocab, 5), c)
    t = O.prompt_ids(9, cfg.vocab, 6)
    ids, lg = m.predict_tree(t, list(range(-1, 8)), c, logits=True)
    want, wlg = m.predict(t, c, all=True, logits=True)
    assert rel_l2(lg, wlg) < 1e-5
    same_ids(ids, lg, want, wlg)


@pytest.mark.parametrize("kv", [J.KV_BF16, J.KV_F32], ids=["bf16pool", "f32pool"])
@pytest.mark.parametrize("ctx", [10, 58, 64, 120])
def test_compaction_keeps_a_path(kv, ctx):
    """After a path is kept the cache predicts as one that was given the
    path's tokens, also when the tree lies across a page boundary."""
    cfg = config()
    m = J.Model.from_config(cfg, 5, mxfp4=True, kv_dtype=kv)
    prompt = O.prompt_ids(ctx, cfg.vocab, 5)
    tokens, parents = tree(30, cfg.vocab, 2)
    node = max(range(30), key=lambda i: len(path_of(i, parents)))
    path = path_of(node, parents)
    assert len(path) > 2 and path != list(range(len(path)))
    a, b = m.cache(), m.cache()
    m.predict(prompt, a)
    m.predict(prompt, b)
    m.predict_tree(tokens, parents, a)
    a.compact(path)
    m.predict([tokens[i] for i in path], b)
    assert a.len == b.len == ctx + len(path)
    more = O.prompt_ids(6, cfg.vocab, 9)
    ids, lg = m.predict(more, a, all=True, logits=True)
    want, wlg = m.predict(more, b, all=True, logits=True)
    assert rel_l2(lg, wlg) < TOL[kv]
    same_ids(ids, lg, want, wlg)


def test_compaction_of_nothing_and_of_a_prefix():
    cfg = config()
    m = J.Model.from_config(cfg, 5, mxfp4=True)
    c = m.cache()
    m.predict(O.prompt_ids(20, cfg.vocab, 5), c)
    m.predict_tree([1, 2, 3], [-1, 0, 1], c)
    c.compact([])
    assert c.len == 20
    with pytest.raises(J.JlError):  # the tree is gone
        c.compact([0])
    m.predict_tree([1, 2, 3], [-1, 0, 1], c)
    c.compact([0, 1])  # nothing to move
    assert c.len == 22


def test_tree_refusals():
    cfg = config()
    m = J.Model.from_config(cfg, 5, mxfp4=True, max_pass_rows=64, kv_pool_tokens=2048)
    c = m.cache()
    m.predict(O.prompt_ids(5, cfg.vocab, 5), c)
    bad = [([], []), ([1, 2], [-1, 1]), ([1, 2], [-1, 2]), ([1], [-2]), ([1], [0]), ([cfg.vocab], [-1]),
           ([1] * 65, [-1] * 65), ([1] * 257, [-1] * 257)]
    for t, p in bad:
        with pytest.raises(J.JlError) as e:
            m.predict_tree(t, p, c)
        assert e.value.status == J.JL_ERR_INVALID_ARG and e.value.message
        assert c.len == 5
    with pytest.raises(ValueError):
        m.predict_tree([1, 2], [-1], c)
    m.predict_tree([1, 2, 3, 4], [-1, 0, 0, 2], c)
    for path in ([1], [0, 3], [0, 1, 2], [2], [0, 0], [4], [0, 2, 3, 3, 3]):
        with pytest.raises(J.JlError) as e:
            c.compact(path)
        assert e.value.status == J.JL_ERR_INVALID_ARG
        assert c.len == 5
    c.compact([0, 2, 3])
    assert c.len == 8
    for drop in (lambda: m.predict([1], c), lambda: c.truncate(6)):
        m.predict_tree([1], [-1], c)
        drop()
        with pytest.raises(J.JlError):
            c.compact([0])
    other = J.Model.from_config(DRAFT, 1, mxfp4=True)
    with pytest.raises(J.JlError):
        other.predict_tree([1], [-1], c)


def test_a_tree_must_fit_the_context():
    cfg = dataclasses.replace(config(), max_positions=64)
    m = J.Model.from_config(cfg, 5, mxfp4=True)
    c = m.cache()
    m.predict(O.prompt_ids(60, cfg.vocab, 5), c)
    with pytest.raises(J.JlError):
        m.predict_tree([1] * 5, [-1] * 5, c)
    m.predict_tree([1] * 4, [-1] * 4, c)


# ---- forks ---------------------------------------------------------------------------


@pytest.mark.parametrize("kv", [J.KV_BF16, J.KV_F32], ids=["bf16pool", "f32pool"])
@pytest.mark.parametrize("at", [0, 1, 63, 64, 100, 128])
def test_forks_go_their_own_ways(kv, at):
    cfg = config()
    m = J.Model.from_config(cfg, 6, mxfp4=True, kv_dtype=kv)
    prompt = O.prompt_ids(128, cfg.vocab, 5)
    a = m.cache()
    m.predict(prompt, a)
    f = a.fork(at)
    assert f.len == at and a.len == 128
    ta, tf = O.prompt_ids(30, cfg.vocab, 11), O.prompt_ids(30, cfg.vocab, 12)
    ra, rf = [], []
    for x, y in zip(ta, tf):  # in turns
        ra.append(m.predict([x], a, logits=True)[1])
        rf.append(m.predict([y], f, logits=True)[1])
    for toks, got, n in ((ta, ra, 128), (tf, rf, at)):
        c = m.cache()
        if n:
            m.predict(prompt[:n], c)
        want = [m.predict([t], c, logits=True)[1] for t in toks]
        assert np.array_equal(np.concatenate(got), np.concatenate(want))


def test_a_write_into_a_shared_page_copies_it():
    """Truncated below a shared page's end, either cache may write there
    without the other seeing it."""
    cfg = config()
    m = J.Model.from_config(cfg, 6, mxfp4=True)
    prompt = O.prompt_ids(200, cfg.vocab, 5)
    a = m.cache()
    m.predict(prompt, a)
    f, g = a.fork(), a.fork(150)
    a.truncate(70)
    m.predict(O.prompt_ids(100, cfg.vocab, 13), a)     # rewrites pages 1 and 2
    g.truncate(0)
    m.predict(O.prompt_ids(64, cfg.vocab, 14), g)      # rewrites page 0
    c = m.cache()
    m.predict(prompt, c)
    for x in (1, 2, 3):
        assert np.array_equal(m.predict([x], f, logits=True)[1], m.predict([x], c, logits=True)[1])
    c = m.cache()
    m.predict(prompt[:70], c)
    m.predict(O.prompt_ids(100, cfg.vocab, 13), c)
    assert np.array_equal(m.predict([9], a, logits=True)[1], m.predict([9], c, logits=True)[1])


def test_a_tree_on_a_fork_leaves_the_original_alone():
    cfg = config()
    m = J.Model.from_config(cfg, 6, mxfp4=True)
    prompt = O.prompt_ids(100, cfg.vocab, 5)
    a, c = m.cache(), m.cache()
    m.predict(prompt, a)
    m.predict(prompt, c)
    f = a.fork()
    tokens, parents = tree(40, cfg.vocab, 3)
    m.predict_tree(tokens, parents, f)
    f.compact([0])
    assert np.array_equal(m.predict([5], a, logits=True)[1], m.predict([5], c, logits=True)[1])


def test_forks_share_pages():
    """640 tokens are ten pages; with a pool of sixteen, twenty forks fit only
    shared.  Pages return when their last holder goes, in any order."""
    cfg = config()
    m = J.Model.from_config(cfg, 6, mxfp4=True, kv_pool_tokens=1024)
    prompt = O.prompt_ids(640, cfg.vocab, 5)
    for _ in range(3):
        a = m.cache()
        m.predict(prompt, a)
        forks = [a.fork() for _ in range(20)]
        inner = [a.fork(600) for _ in range(6)]  # each copies the page it ends in
        for call in (lambda: a.fork(600), lambda: m.predict([1], forks[0])):
            with pytest.raises(J.JlError) as e:
                call()
            assert e.value.status == J.JL_ERR_OOM
        del inner, e, call
        gc.collect()  # the error's frames hold caches
        want = m.predict([1], forks[0], logits=True)[1]
        del a
        assert np.array_equal(m.predict([1], forks[1], logits=True)[1], want)
        del forks
        gc.collect()
    c = m.cache()
    m.predict(O.prompt_ids(1000, cfg.vocab, 5), c)  # the whole pool is free again


def test_fork_refusals():
    m = J.Model.from_config(config(), 6, mxfp4=True)
    c = m.cache()
    m.predict([1, 2, 3], c)
    with pytest.raises(J.JlError) as e:
        c.fork(4)
    assert e.value.status == J.JL_ERR_INVALID_ARG
    f = c.fork(0)
    assert f.len == 0
    m.free()
    with pytest.raises(J.JlError) as e:
        c.fork(1)
    assert "freed" in e.value.message


# ---- together ------------------------------------------------------------------------


def best(row, k):
    return [int(i) for i in np.argsort(-row, kind="stable")[:k]]


def tree_decode(target, draft, prompt, count, width=2, depth=3):
    """Greedy decode by trees: the draft's best `width` tokens of every node, to
    `depth`; the target verifies the tree, and the path that agrees with it is
    kept in the target's cache."""
    tc, dc = target.cache(), draft.cache()
    out, accepted = list(prompt), 0
    pending = target.predict(prompt, tc)[0]
    draft.predict(prompt, dc)
    while len(out) - len(prompt) < count:
        tokens, parents, level = [pending], [-1], [(0, dc.fork())]
        kept = None  # the draft's cache with the pending token
        for d in range(depth):
            grown = []
            for node, cache in level:
                row = draft.predict([tokens[node]], cache, logits=True)[1][0]
                kept = kept or cache
                if d + 1 == depth:
                    continue
                for t in best(row, width):
                    tokens.append(t)
                    parents.append(node)
                    grown.append((len(tokens) - 1, cache.fork()))
            level = grown
        ids = target.predict_tree(tokens, parents, tc)
        path, node = [0], 0
        while True:
            child = [i for i in range(len(tokens)) if parents[i] == node and tokens[i] == ids[node]]
            if not child:
                break
            node = child[0]
            path.append(node)
        tc.compact(path)
        accepted += len(path) - 1
        for i in path:
            out.append(tokens[i])
        if len(path) > 1:
            draft.predict([tokens[i] for i in path[1:]], kept)
        dc, pending = kept, ids[node]
    return out[:len(prompt) + count], accepted


@pytest.mark.parametrize("kv", [J.KV_BF16, J.KV_F32], ids=["bf16pool", "f32pool"])
@pytest.mark.parametrize("same", [True, False], ids=["draft-is-target", "other-draft"])
def test_tree_decode_follows_the_target(kv, same):
    """Decoding by trees gives the target's greedy stream: every token is
    compared with the oracle decoding the same tokens."""
    cfg = config(layers=2)
    ref = O.Model.synthetic(cfg, 3, mxfp4=True)
    m = J.Model.from_config(cfg, 3, mxfp4=True, kv_dtype=kv, kv_pool_tokens=8192)
    d = J.Model.from_config(cfg, 3 if same else 8, mxfp4=True, kv_dtype=kv, kv_pool_tokens=8192)
    prompt = O.prompt_ids(50, cfg.vocab, 5)
    got, accepted = tree_decode(m, d, prompt, 40)
    check = compare_streams(got, ref, prompt, 40, round_bf16=kv == J.KV_BF16)
    assert check.compared == 40 or got[-1] == ref.eos or ref.eos in got[len(prompt):]
    assert accepted > 20 if same else accepted >= 0
