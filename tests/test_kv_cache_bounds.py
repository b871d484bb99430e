"""What the bounds of the paged attention's GPU tests can tell apart, on the
CPU: mistakes are planted in the 64-bit form and have to fall outside them."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_kv_cache import BF16, F16, F32, block_values, expected  # noqa: E402


def case(dtype, new, n, d, hq=4, hk=2):
    g = torch.Generator().manual_seed(n + new)
    q = torch.randn(new, hq, d, generator=g).to(dtype)
    k = torch.randn(hk, n, d, generator=g).to(dtype)
    return q, k, block_values(n, d, "cpu").to(dtype).expand(hk, n, d)


def attention(q, k, v, scale, seen):
    """[m, hq, d] in 64 bits, of the keys in `seen` alone."""
    m, hq, d = q.shape
    x = q.double().reshape(m, k.shape[0], -1, d)
    s = torch.einsum("mhgd,hnd->mhgn", x, k.double()) * scale
    w = torch.where(seen, s, -math.inf).softmax(-1)
    return torch.einsum("mhgn,hnd->mhgd", w, v.double()).reshape(m, hq, d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new, n, d", [(1, 40000, 128), (3, 40000, 128), (1, 12000, 64)])
@pytest.mark.parametrize("lost", [64, 128, 576])
def test_a_lost_piece_shows(dtype, new, n, d, lost):
    q, k, v = case(dtype, new, n, d)
    want, tol = expected(q, [k], [v], [0], [new], 1 / math.sqrt(d), False, 0)
    seen = torch.ones(n, dtype=torch.bool)
    assert ((attention(q, k, v, 1 / math.sqrt(d), seen) - want).abs() <= tol).all()
    for first in (0, n // 2, n - lost):
        some = seen.clone()
        some[first:first + lost] = False
        assert ((attention(q, k, v, 1 / math.sqrt(d), some) - want).abs() > tol).any(-1).all()  # in every row


@pytest.mark.parametrize("new, n, d, types", [(1, 40000, 128, [BF16]), (3, 7000, 64, [BF16, F16])])
@pytest.mark.parametrize("short", ["queries", "keys", "both"])
def test_f32_of_fewer_bits_shows(new, n, d, types, short):
    """Queries or keys rounded to bf16; to f16 where the keys are not so many
    that their sum's own bound (n 2^-24 of it) is as large."""
    q, k, v = case(F32, new, n, d)
    want, tol = expected(q, [k], [v], [0], [new], 1.0, False, 0)
    seen = torch.ones(n, dtype=torch.bool)
    for dtype in types:
        q1 = q.to(dtype) if short != "keys" else q
        k1 = k.to(dtype) if short != "queries" else k
        assert ((attention(q1, k1, v, 1.0, seen) - want).abs() > tol).any(-1).all()
