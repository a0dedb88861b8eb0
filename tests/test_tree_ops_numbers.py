"""Page ids, rows, parents and paths that do not fit the C ABI's types are
refused by the Python calls instead of naming another page or node (no GPU
needed)."""
import types

import numpy as np
import pytest

import jalapeno as J

HOST = np.zeros(1 << 12, np.uint8)
P = (HOST.ctypes.data + 255) // 256 * 256

BIG = [[2 ** 32 + 1], [-2 ** 32], np.array([2 ** 32 + 1]), [1.5], np.array([0.0])]


@pytest.mark.parametrize("bad", BIG)
def test_page_copies(bad):
    pool = J.kv_pages(k=P, v=P, pages=8, kv_heads=2)
    for a in ((bad, [2]), ([2], bad), ([2], [3], bad)):
        with pytest.raises(ValueError):
            J.kv_copy_pages(pool, *a)


@pytest.mark.parametrize("bad", BIG)
def test_trees(bad):
    m = types.SimpleNamespace(_h=None, vocab=10)
    with pytest.raises(ValueError):
        J.Model.predict_tree(m, [1], bad, types.SimpleNamespace(_h=None))
    with pytest.raises(ValueError):
        J.Cache.compact(types.SimpleNamespace(_h=None), bad)


def test_what_fits_is_passed_on():
    """Tuples, arrays of any whole type and empty lists reach the library."""
    pool = J.kv_pages(k=P, v=P, pages=8, kv_heads=2)
    J.kv_copy_pages(pool, (), ())
    for src in ([9], (9,), np.array([9], np.uint8), np.array([9])):
        with pytest.raises(J.JlError) as e:
            J.kv_copy_pages(pool, src, [1])
        assert "outside" in e.value.message
