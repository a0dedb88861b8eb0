"""Refusals of the operators of tree-shaped speculation: every bad argument is
an error with a message before anything reaches a device (no GPU needed)."""
import ctypes

import numpy as np
import pytest

import jalapeno as J

HOST = np.zeros(1 << 16, np.uint8)
P = (HOST.ctypes.data + 255) // 256 * 256  # an aligned address that is not device memory


def pool(**kw):
    a = dict(k=P, v=P, pages=8, kv_heads=2)
    a.update(kw)
    return J.kv_pages(**a)


def attn(pool_kw={}, **kw):
    a = dict(q=P, q_ld=512, out=P + 4096, out_ld=512, rows=4, q_heads=4, seqs=1, max_nodes=4, row_start=P, ctx=P,
             page_table=P, max_pages=4, workspace=P, workspace_bytes=J.TREE_WORKSPACE_BYTES)
    a.update(kw)
    J.tree_attention(pool(**pool_kw), **a)


def norm(pool_kw={}, **kw):
    a = dict(qkv=P, qkv_ld=1024, q=P + 4096, q_ld=512, rows=4, q_heads=4, rope=P, positions=10, pos=P, page_table=P,
             max_pages=4)
    a.update(kw)
    J.qk_norm_rope(pool(**pool_kw), **a)


def compact(pool_kw={}, **kw):
    a = dict(seqs=1, ctx=P, path=P, path_ld=4, path_len=P, page_table=P, max_pages=4)
    a.update(kw)
    J.kv_compact(pool(**pool_kw), **a)


def refused(call, *args, words=(), **kw):
    with pytest.raises(J.JlError) as e:
        call(*args, **kw)
    assert e.value.status == J.JL_ERR_INVALID_ARG
    assert e.value.message
    for w in words if isinstance(words, tuple) else (words,):
        assert w in e.value.message, e.value.message


@pytest.mark.parametrize("call", [attn, norm, compact])
@pytest.mark.parametrize("kw,words", [
    (dict(k=0), "k and v"), (dict(v=0), "k and v"), (dict(k=P + 8), "aligned"), (dict(dtype=7), "dtype"),
    (dict(pages=0), "page"), (dict(kv_heads=0), "kv heads"), (dict(kv_heads=-1), "kv heads"), (dict(layers=0), "layer"),
    (dict(pages=1 << 30), "2^31"), (dict(layers=2, layer_stride=16), "layer")])
def test_pools(call, kw, words):
    refused(call, kw, words=words)


@pytest.mark.parametrize("kw,words", [
    (dict(q=0), "non-null"), (dict(out=0), "non-null"), (dict(row_start=0), "non-null"), (dict(ctx=0), "non-null"),
    (dict(page_table=0), "non-null"), (dict(q=P + 4), "aligned"), (dict(out=P + 8), "aligned"), (dict(q_ld=511), "q_ld"),
    (dict(q_ld=504), "q_ld"), (dict(out_ld=256), "out_ld"), (dict(rows=-1), "negative"), (dict(seqs=-1), "negative"),
    (dict(q_heads=0), "query heads"), (dict(q_heads=5, q_ld=1024, out_ld=1024), "query heads"),
    (dict(q_heads=258, q_ld=1 << 16, out_ld=1 << 16), "query heads"), (dict(max_nodes=0), "max_nodes"),
    (dict(max_nodes=257), "max_nodes"), (dict(dtype=2), "dtype"), (dict(mask=P, mask_words=0), "mask"),
    (dict(mask=P, mask_words=1, max_nodes=65), "mask"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=(1 << 24) + 1), "max_pages"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(out=P, out_ld=520), "out over q"), (dict(mask=P + 4, mask_words=1), "8-byte"),
    (dict(ctx=P + 2), "4-byte"), (dict(row_start=P + 1), "4-byte"), (dict(page_table=P + 2), "4-byte"), (dict(lse=P + 2), "4-byte"),
    (dict(status=P + 2), "4-byte"), (dict(seqs=1 << 20, max_pages=1 << 20), "2^31")])
def test_tree_attention(kw, words):
    refused(attn, words=words, **kw)


@pytest.mark.parametrize("kw,words", [
    (dict(qkv=0), "non-null"), (dict(q=0), "non-null"), (dict(rope=0), "non-null"), (dict(pos=0), "non-null"),
    (dict(page_table=0), "non-null"), (dict(qkv=P + 2), "aligned"), (dict(rope=P + 8), "aligned"), (dict(q_norm=P + 2), "aligned"),
    (dict(qkv_ld=1023), "qkv_ld"), (dict(qkv_ld=1000), "qkv_ld"), (dict(q_ld=500), "q_ld"), (dict(rows=-1), "negative"),
    (dict(q_heads=0), "query head"), (dict(dtype=5), "dtype"), (dict(seqs=0), "sequence"), (dict(max_pages=0), "pages"),
    (dict(positions=0), "position"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(q=P, q_ld=512), "q over qkv"), (dict(pos=P + 2), "4-byte"), (dict(slot=P + 1), "4-byte"), (dict(seq=P + 2), "4-byte"),
    (dict(status=P + 3), "4-byte")])
def test_norm_rope(kw, words):
    refused(norm, words=words, **kw)


@pytest.mark.parametrize("kw,words", [
    (dict(ctx=0), "non-null"), (dict(path=0), "non-null"), (dict(path_len=0), "non-null"), (dict(page_table=0), "non-null"),
    (dict(seqs=-1), "sequences"), (dict(seqs=65536), "sequences"), (dict(path_ld=0), "path_ld"), (dict(path_ld=257), "path_ld"),
    (dict(max_pages=0), "max_pages"), (dict(path=P + 2), "4-byte"), (dict(ctx=P + 2), "4-byte")])
def test_compaction(kw, words):
    refused(compact, words=words, **kw)


@pytest.mark.parametrize("src,dst,rows,words", [
    ([8], [0], None, "outside"), ([0], [-1], None, "outside"), ([0], [0], None, "both source and destination"),
    ([0, 1], [2, 2], None, "two copies"), ([0, 1], [1, 2], None, "both"), ([0], [1], [0], "rows"), ([0], [1], [65], "rows"),
    ([0] * 9, list(range(9)), None, "copies")])
def test_page_copies(src, dst, rows, words):
    refused(J.kv_copy_pages, pool(), src, dst, rows, words=words)


def test_page_copies_of_different_lengths():
    with pytest.raises(ValueError):
        J.kv_copy_pages(pool(), [0, 1], [2])
    with pytest.raises(ValueError):
        J.kv_copy_pages(pool(), [0], [2], [1, 2])


def test_null_structures():
    n = ctypes.c_size_t()
    assert J.lib.jl_tree_attention(None, None) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_tree_attention_workspace(None, ctypes.byref(n)) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_qk_norm_rope(None, None) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_kv_compact(None, None) == J.JL_ERR_INVALID_ARG
    out = ctypes.c_void_p()
    assert J.lib.jl_predict_tree(None, None, None, None, 0, None, None) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_cache_fork(None, 0, ctypes.byref(out)) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_cache_compact(None, None, 0) == J.JL_ERR_INVALID_ARG
    assert J.lib.jl_kv_copy_pages(None, None, None, None, 0, None) == J.JL_ERR_INVALID_ARG


def test_nothing_to_do_is_not_an_error():
    attn(rows=0)
    attn(seqs=0)
    norm(rows=0)
    compact(seqs=0)
    # an empty tensor has no address
    attn(rows=0, q=0, out=0, row_start=0, ctx=0, page_table=0, workspace=0, workspace_bytes=0)
    norm(rows=0, qkv=0, q=0, pos=0, page_table=0)
    compact(seqs=0, ctx=0, path=0, path_len=0, page_table=0)
    J.kv_copy_pages(pool(), [], [])


def test_host_memory_is_refused():
    """With a device: not device memory.  Without one: no device."""
    for call in (attn, norm, compact):
        with pytest.raises(J.JlError) as e:
            call()
        assert e.value.status in (J.JL_ERR_INVALID_ARG, J.JL_ERR_NO_DEVICE)
        if J.device_count():
            assert "not device memory" in e.value.message
