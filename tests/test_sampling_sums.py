"""Verification and sampling where sums decide: large vocabularies whose terms
all round alike, numbers next to the border of a decision."""
import math

import pytest
import torch

from cdq_lrr_b200 import sampling
from test_sampling import BF, drawn, softmax

pytestmark = pytest.mark.gpu


def around(border, count, width):
    """`count` float32 numbers spread over border * (1 -+ width), none nearer to it than 64-bit sums tell apart."""
    e = torch.linspace(-width, width, count, dtype=torch.float64)
    u = (border * (1 + e)).float()
    return u[((u.double() / border - 1).abs() > 1e-9) & (u < 1)]


def outliers(V, low, dtype):
    """1,024 logits of 0 in front, the others `low`."""
    row = torch.full((V,), low)
    row[:1024] = 0
    return row.to(dtype)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [152064, 262144, 1 << 20, (1 << 22) - 5, 1 << 22])
@pytest.mark.parametrize("low", [-16.75, -10.8, -9.6, -3.0])
def test_kept_drafts_of_large_vocabularies(dtype, V, low):
    """u_accept on both sides of p(x) (drafts chosen greedily), many sequences of the same logits."""
    row = outliers(V, low, dtype).cuda()
    p = float(softmax(row, 1.0)[7])
    ua = around(p, 400, 3e-4)
    B = len(ua)
    t = row[None, None].expand(B, 2, V)
    d = torch.full((B, 1), 7, device="cuda")
    us = torch.zeros(B, device="cuda")
    _, kept = sampling.verify_drafts(t, d, None, ua[:, None].contiguous().cuda(), us)
    assert torch.equal(kept.cpu() == 1, ua.double() < p)


@pytest.mark.parametrize("V", [152064, 1 << 20, 1 << 22])
@pytest.mark.parametrize("rise", [1e-3, 1.0, 12.0, -12.0])
def test_kept_drafts_of_sloping_logits(V, rise):
    """Logits that rise, or fall, over the whole vocabulary: the maximum moves with every load. u_accept on both sides
    of p(x) / q(x), the other row flat."""
    slope = torch.linspace(0, rise, V, dtype=torch.float64).float().cuda()
    flat = torch.zeros(V, device="cuda")
    x = int(V * 0.45)
    p, q = float(softmax(slope, 1.0)[x]), 1 / V
    rows = (slope, flat) if p < q else (flat, slope)
    border = min(p / q, q / p)
    ua = around(border, 400, 3e-4)
    B = len(ua)
    t = rows[0][None, None].expand(B, 2, V)
    dl = rows[1][None, None].expand(B, 1, V)
    d = torch.full((B, 1), x, device="cuda")
    _, kept = sampling.verify_drafts(t, d, dl, ua[:, None].contiguous().cuda(), torch.zeros(B, device="cuda"))
    assert torch.equal(kept.cpu() == 1, ua.double() < border)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [262144, 1 << 22])
def test_sampled_tokens_of_large_vocabularies(dtype, V):
    """u on both sides of running sums' borders in a flat tail, and at both ends of [0, 1)."""
    row = outliers(V, -6.0, dtype).cuda()
    p = softmax(row, 0.9)
    c = torch.cumsum(p, 0)
    pick = torch.randint(0, V - 1, (40,), generator=torch.Generator().manual_seed(V)).cuda()
    us = c[pick].float()
    us = torch.cat([us, (us.view(torch.int32) - 1).view(torch.float32), (us.view(torch.int32) + 1).view(torch.float32),
                    torch.tensor([0.0, 1 - 2.0 ** -24], device="cuda")]).clamp(0, 1 - 2.0 ** -24)
    want = [drawn(p, float(u)) for u in us]
    assert sampling.sample_tokens(row.expand(len(us), V), us, 0.9).tolist() == want


@pytest.mark.parametrize("V", [4096, 50021, 262144, 1 << 20])
@pytest.mark.parametrize("ulps", [(0, 1), (-1, 1), (0, 2), (-3, 3)])
@pytest.mark.parametrize("heavy", [0.03, 0.3])
def test_draws_where_most_tokens_are_nearly_alike(V, ulps, heavy):
    """Draft and target share all but a few float32 steps of every logit, except for one token each that the other
    does not favour: max(p - q, 0) is the target's token and a sum of 10^-7 of the rest. u around the border of the
    two. The drawn token's interval of running sums holds u, to 1e-10 of the total: exponentials to 1.3e-12 of
    p + q <= 2, divided by a total of 0.029 at least."""
    g = torch.Generator().manual_seed(V + ulps[1])
    steps = torch.randint(0, 2, (V,), generator=g) * (ulps[1] - ulps[0]) + ulps[0]
    t = torch.ones(V)
    q = (t.view(torch.int32) + steps.int()).view(torch.float32)
    rise = math.log(V * heavy / (1 - 2 * heavy))
    t[V // 2] += rise
    q[V // 3] += rise
    w = (softmax(t, 1.0) - softmax(q, 1.0)).clamp(min=0)
    c = torch.cumsum(w, 0) / w.sum()
    # the tokens in front of the target's have 0 .. 10^-7 of the total, those behind it too
    us = torch.cat([torch.arange(1, 65) * 2.0 ** -28, 1 - torch.arange(1, 65) * 2.0 ** -24,
                    torch.rand(40, generator=g), torch.zeros(1)])
    B = len(us)
    d = torch.full((B, 1), V // 3)
    got, kept = sampling.verify_drafts(t.cuda()[None, None].expand(B, 2, V), d.cuda(), q.cuda()[None, None].expand(B, 1, V),
                                       torch.full((B, 1), 1 - 2.0 ** -24).cuda(), us.cuda())
    assert not kept.any()
    x = got[:, 0].cpu()
    u = us.double()
    assert bool((w[x] > 0).all())
    assert bool((c[x] > u - 1e-10).all()) and bool(((c - w / w.sum())[x] <= u + 1e-10).all())
