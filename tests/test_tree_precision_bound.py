"""The bound of test_gpu_tree_precision.py's 24-bit test on the CPU: the operator
in 64 bits is within it, and with one third piece of 8 bits left out, of Q, of the
weights or of K or V, it is not (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

import jalapeno as J
from test_gpu_tree_precision import KEPT, far_of, tails_of_24_bits


def two_pieces(x, rounded):
    """The first 16 bits of x, as two bf16 pieces hold them."""
    out, rest = torch.zeros_like(x), x
    for _ in range(2):
        p = rest.float().to(torch.bfloat16).double() if rounded else (rest.float().view(torch.int32) & -65536).view(torch.float32).double()
        out, rest = out + p, rest - p
    return out


@pytest.mark.parametrize("pool,lost", [(p, x) for p in (J.KV_BF16, J.KV_F32) for x in ("nothing", "q", "w") + ("k", "v") * (p == J.KV_F32)])
def test_a_lost_piece_is_seen(pool, lost):
    a, kappa, v = tails_of_24_bits(pool, 512, 10)
    q, k, val = a.double(), torch.tensor(kappa, dtype=torch.float64), v.double()
    if lost == "q":
        q = two_pieces(q, True)  # queries are rounded into pieces, the others cut
    if lost == "k":
        k = two_pieces(k, False)
    if lost == "v":
        val = two_pieces(val, False)
    w = torch.exp(-q * k)
    top = two_pieces(w.float().double(), False) if lost == "w" else w
    out = (63 * top / (1 + 63 * w))[:, None] * val
    far = far_of(out, a, kappa, v)
    if lost == "nothing":
        assert far < KEPT / 1e3
    else:
        assert far > 2 * KEPT, far / KEPT
