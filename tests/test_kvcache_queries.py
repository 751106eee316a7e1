"""Attention over the quantised cache with queries whose elements differ much
in size."""

import pytest
import torch

from cdq_lrr_b200 import _lib as L
from test_kvcache import BF, check, filled, int32, normal, roomy, rotate, tables, values

pytestmark = pytest.mark.gpu


def expected(c, q, pos, scale, rope=None):
    """One sequence and one kv head, q [n, G, hd], in 64 bits, and how far the kernel's result may be off: a query
    element enters the first product to 2^-11 of itself or 2^-20 of its row's largest, which moves scores and so
    numerator and denominator; weights to 2^-11 (2^-32 of the largest), sums and exponentials to 2^-13, the result
    to half a bf16 step."""
    K, V = (x[0, 0] for x in values(c))
    n, G, hd = q.shape
    out = torch.zeros(n, G, hd, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(n):
        m = pos + i + 1
        x = q[i].cpu().double()
        if rope is not None:
            x = rotate(x, rope[0][pos + i].cpu(), rope[1][pos + i].cpu())
        off = x.abs() * 2.0 ** -11 + x.abs().amax(-1, keepdim=True) * 2.0 ** -20
        p = torch.softmax(x @ K[:m].T * scale, -1)
        d = (off @ K[:m].abs().T).amax(-1, keepdim=True) * abs(scale)
        out[i] = p @ V[:m]
        bound[i] = (p @ V[:m].abs()) * (torch.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -13 + m * 2.0 ** -32) + out[i].abs() * 2.0 ** -8
    return out, bound


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [0, 6, 9, 12])
@pytest.mark.parametrize("turned", [False, True])
def test_one_large_query_element(hd, bits, turned):
    """One query element 2^bits of the others', over keys that have next to nothing there: the other elements decide.
    Both kernels (the second cache takes the tensor-memory one)."""
    n, G, Lm = 50, 2, 400
    g = torch.Generator().manual_seed(bits)
    k, v = torch.randn(1, Lm, 1, hd, generator=g), torch.randn(1, Lm, 1, hd, generator=g)
    k[..., (5, hd // 2 + 5)] = 0
    c = filled(3, 1, 1, Lm, hd, "e4m3")
    c.append(k.to(BF).cuda(), v.to(BF).cuda(), int32(0))
    q = normal(7, 1, n, G, hd, scale=2.0)
    q[..., 5] = 2.0 * 2.0 ** bits
    rope = tables(Lm, hd) if turned else None
    pos = Lm - n
    want, bound = expected(c, q[0], pos, hd ** -0.5, rope)
    for x in (c, roomy(c, n * G)):
        check(x.attend(q, int32(pos), rope=rope)[0], want, bound)
    assert L.kernel_error() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_of_any_magnitude(hd):
    """Query rows of all sizes: the bound is relative to each row's own largest element."""
    n, G, Lm = 64, 2, 300
    c = filled(5, 1, 1, Lm, hd, "e4m3")
    q = normal(9, 1, n, G, hd)
    e = torch.arange(n, device="cuda").float() - n / 2
    q = (q.float() * torch.exp2(e / 8)[None, :, None, None]).to(BF)
    want, bound = expected(c, q[0], Lm - n, 0.3)
    for x in (c, roomy(c, n * G)):
        check(x.attend(q, int32(Lm - n), scale=0.3)[0], want, bound)
    assert L.kernel_error() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [10, 12, 14])
def test_small_query_elements_that_err_alike(hd, bits):
    """The elements beside a large one are 2 (1 + 2^-5) in the first half and 2 in the second, with keys of ones in
    one half each and no weight on the large one: what is left of the difference decides between two groups of
    positions, and whatever an element loses is lost hd / 2 times."""
    n, G, Lm = 50, 2, 400
    k, v = torch.zeros(1, Lm, 1, hd), torch.ones(1, Lm, 1, hd)
    k[:, ::2, :, 1:hd // 2], k[:, 1::2, :, hd // 2 + 1:] = 1, 1
    v[:, 1::2] = -1
    c = filled(3, 1, 1, Lm, hd, "e4m3")
    c.append(k.to(BF).cuda(), v.to(BF).cuda(), int32(0))
    q = torch.full((1, n, G, hd), 2.0, dtype=BF, device="cuda")
    q[..., :hd // 2] = 2.0 + 2.0 ** -4
    q[..., 0] = 2.0 ** (bits + 1)
    scale = 8 / hd
    want, bound = expected(c, q[0], Lm - n, scale)
    for x in (c, roomy(c, n * G)):
        check(x.attend(q, int32(Lm - n), scale=scale)[0], want, bound)
    assert L.kernel_error() == 0
