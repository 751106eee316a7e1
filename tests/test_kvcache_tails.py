"""Attention over the quantised cache where one position has nearly all of the
weight and very many share the rest: the small weights' sum counts."""
import math

import pytest
import torch

from cdq_lrr_b200 import _lib as L
from test_kvcache import BF, QuantKVCache, check, int32, values

pytestmark = pytest.mark.gpu


def sunk(B, kv, Lm, hd, fmt, sink):
    """A cache whose heads all hold the same: the key of position `sink` is 4 in its first element, every other key
    zero; its value lies in the first half of the elements, those of the others in the second."""
    g = torch.Generator().manual_seed(Lm + sink)
    k, v = torch.zeros(1, Lm, 1, hd), torch.zeros(1, Lm, 1, hd)
    k[0, sink, 0, 0] = 4.0
    v[..., hd // 2:] = 1.0 + torch.rand(1, Lm, 1, hd // 2, generator=g)
    v[0, sink, 0, hd // 2:] = 0
    v[0, sink, 0, :hd // 2] = 1.0 + torch.rand(hd // 2, generator=g)
    c = QuantKVCache(B, kv, Lm, hd, fmt)
    shape = (B, Lm, kv, hd)
    c.append(k.to(BF).cuda().expand(shape), v.to(BF).cuda().expand(shape), int32(*[0] * B))
    return c


def expected(c, n, pos, q0, scale):
    """Rows 0 .. n - 1 of one head [n, hd] in 64 bits, and how far the kernel's may be off: a weight p s (s the value's
    scale) is rounded to half under a reference at least 2^7 below the largest of them, to 2^-11 of itself or, below
    2^-14, to half of 2^-24: 2^-32 of the largest. Queries are exact in half, scores off by 2^-20 of them at most,
    sums and exponentials by 2^-13 in all, the result by half a bf16 step."""
    one = QuantKVCache.from_buffers(*(t[:1, :1].clone() for t in (c.k, c.v, c.k_scale, c.v_scale)))
    K, V = (x[0, 0] for x in values(one))
    s_v = one.v_scale[0, 0].cpu().double().reshape(c.max_len, -1)
    codes = V.abs() / (s_v if c.fmt == "e4m3" else s_v.repeat_interleave(32, -1))
    out, bound = [], []
    for i in range(n):
        m = pos + i + 1
        s = K[:m, 0] * q0 * scale
        p = torch.softmax(s, 0)
        d = float(s.abs().max()) * 2.0 ** -20
        o = p @ V[:m]
        floor = 2.0 ** -32 * float((p[:, None] * s_v[:m]).max()) * codes[:m].sum(0)
        out.append(o)
        bound.append((p @ V[:m].abs()) * (math.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -13) + floor + o.abs() * 2.0 ** -8)
    return torch.stack(out), torch.stack(bound)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [23.2, 24.9, 25.1, 27.3])
@pytest.mark.parametrize("B,kv,Lm,n,G,sink", [
    (1, 1, 128, 1, 1, 0),        # one unit
    (2, 1, 700, 3, 2, 130),      # a cluster of CTAs
    (1, 2, 5000, 1, 7, 4000),    # segments cut over the device
    (40, 16, 6000, 1, 3, 5),     # whole segments of many units a CTA
    (37, 8, 4100, 9, 2, 40),     # the same, tiles of 16 and 24 rows
    (37, 4, 1024, 50, 2, 3),     # e4m3: the tensor-memory kernel, a segment a CTA
    (40, 8, 4100, 40, 2, 700),   # and several
])
def test_a_long_tail_under_one_position(fmt, hd, bits, B, kv, Lm, n, G, sink):
    """Each of the other positions has 2^-bits of the largest weight; their values' elements are zero in its own."""
    c = sunk(B, kv, Lm, hd, fmt, sink)
    q = torch.zeros(B, n, kv * G, hd, dtype=BF, device="cuda")
    q[..., 0] = 8.0
    scale = bits * math.log(2) / 32
    got = c.attend(q, int32(*[Lm - n] * B), scale=scale)
    want, bound = expected(c, n, Lm - n, 8.0, scale)
    want, bound = (x[None, :, None].expand(B, n, kv * G, hd) for x in (want, bound))
    check(got, want, bound)
    assert L.kernel_error() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_long_tail_behind_a_prefix(fmt, hd):
    """The position with the weight is in the prefix, the tail behind it there and in each sequence's own cache."""
    bits, P, B, n, Lm = 25.1, 9000, 30, 4, 300
    pre, c = sunk(1, 1, P, hd, fmt, 11), sunk(B, 1, Lm, hd, fmt, Lm - 1)
    q = torch.zeros(B, n, 2, hd, dtype=BF, device="cuda")
    q[..., 0] = 8.0
    scale = bits * math.log(2) / 32
    pos = Lm - 1 - n                    # (its own large key is not seen)
    got = c.attend(q, int32(*[pos] * B), scale=scale, prefix=pre, prefix_len=int32(P))
    both = QuantKVCache(1, 1, P + Lm, hd, fmt)
    for x, y, z in zip((both.k, both.v, both.k_scale, both.v_scale), (pre.k, pre.v, pre.k_scale, pre.v_scale),
                       (c.k, c.v, c.k_scale, c.v_scale)):
        x[:, :, :P].view(torch.uint8).copy_(y.view(torch.uint8))
        x[:, :, P:].view(torch.uint8).copy_(z[:1].view(torch.uint8))
    want, bound = expected(both, n, P + pos, 8.0, scale)
    check(got, *(x[None, :, None].expand(B, n, 2, hd) for x in (want, bound)))
    assert L.kernel_error() == 0


@pytest.mark.parametrize("fmt,B,kv,n,G", [
    ("e2m1", 74, 8, 1, 2),       # a segment a CTA, 32,768 positions a warp
    ("e4m3", 74, 8, 1, 2),
    ("e4m3", 37, 4, 37, 2),      # the tensor-memory kernel, 65,536 positions a stream
])
@pytest.mark.parametrize("bits", [25.1, 27.3])
def test_tails_of_131072_positions(fmt, B, kv, n, G, bits):
    """The tail has 0.4 or 0.1 per cent of the weight."""
    Lm, hd = 131072, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 11 GB of device memory")
    c = sunk(B, kv, Lm, hd, fmt, 77)
    q = torch.zeros(B, n, kv * G, hd, dtype=BF, device="cuda")
    q[..., 0] = 8.0
    scale = bits * math.log(2) / 32
    got = c.attend(q, int32(*[Lm - n] * B), scale=scale)
    want, bound = expected(c, n, Lm - n, 8.0, scale)
    check(got, *(x[None, :, None].expand(B, n, kv * G, hd) for x in (want, bound)))
    assert L.kernel_error() == 0
