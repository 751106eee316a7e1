"""Verification of drafted tokens and sampling against the definition in 64
bits, and their refusals."""
import math

import pytest
import torch

from cdq_lrr_b200 import _lib as L
from cdq_lrr_b200 import sampling

gpu = pytest.mark.gpu
BF = torch.bfloat16


def softmax(row, T):
    z = row.double() / T
    if torch.isnan(z).any() or (z == math.inf).any() or (z == -math.inf).all():
        return None
    return torch.softmax(z, 0)


def drawn(w, u):
    c = torch.cumsum(w, 0)
    over = (c > u * float(c[-1])) & (w > 0)
    return int(over.nonzero()[0]) if over.any() else int((w > 0).nonzero()[-1])


def verify(target, drafts, draft, ua, us, T):
    """The definition, one sequence at a time, 64 bits."""
    B, k = drafts.shape
    V = target.shape[-1]
    tokens, kept = torch.full((B, k + 1), -1), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        a = 0
        while True:
            p = softmax(target[b, a], T)
            x = int(drafts[b, a]) if a < k else -1
            q = None
            if p is None:
                break
            if x < 0:
                tokens[b, a] = drawn(p, float(us[b]))
                break
            if draft is not None:
                q = softmax(draft[b, a], T)
                if q is None:
                    break
            px = float(p[x]) if x < V else 0.0
            qx = 1.0 if q is None else float(q[x]) if x < V else 0.0
            if not float(ua[b, a]) * qx < px:
                w = (p - q).clamp(min=0) if q is not None else p.clone()
                if q is None and x < V:
                    w[x] = 0
                tokens[b, a] = drawn(w if w.sum() > 0 else p, float(us[b]))
                break
            tokens[b, a] = x
            a += 1
        kept[b] = a
    return tokens, kept


def inputs(seed, B, k, V, dtype, spread=0.7, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(B, k + 1, V, generator=g) * scale
    draft = (base[:, :k] + spread * torch.randn(B, k, V, generator=g)).to(dtype)
    drafts = torch.multinomial(torch.softmax(draft.float(), -1).reshape(B * k, V), 1, generator=g).reshape(B, k) \
        if k else torch.zeros(B, 0, dtype=torch.long)
    return base.to(dtype), drafts, draft, torch.rand(B, k, generator=g), torch.rand(B, generator=g)


def run(target, drafts, draft, ua, us, T):
    t, n = sampling.verify_drafts(target.cuda(), drafts.cuda(), None if draft is None else draft.cuda(), ua.cuda(),
                                  us.cuda(), T)
    return t.cpu(), n.cpu()


def same(got, want):
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    assert torch.equal(got[0], want[0]), (got[0], want[0])


# ---------------------------------------------------------------- refusals (no GPU)


def test_refusals():
    x = torch.zeros(1, 3, 8, dtype=BF)
    d, u, s = torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 2), torch.zeros(1)
    with pytest.raises(RuntimeError):
        sampling.verify_drafts(x, d, None, u, s)
    with pytest.raises(RuntimeError):
        sampling.sample_tokens(x[0], torch.zeros(3))
    with pytest.raises(ValueError):
        sampling.verify_drafts(x[0], d, None, u, s)
    with pytest.raises(ValueError):
        sampling.sample_tokens(x, torch.zeros(1))
    with pytest.raises(ValueError):
        sampling.sample_tokens(x[0, :, :0], torch.zeros(3))


def test_c_abi_refusals():
    f = L.lib().cdq_verify_drafts

    def call(target=4096, dtype=0, drafts=4096, ua=4096, us=4096, batch=1, k=1, vocab=8, T=1.0, tokens=4096, row=8,
             ws=4096, ws_bytes=1 << 20):
        return f(target, 16, row, None, 0, 0, dtype, drafts, ua, us, batch, k, vocab, T, tokens, None, ws, ws_bytes,
                 None)

    assert call(dtype=2) == 8
    assert call(ws=None) == 7 and call(ws=4104) == 7 and call(ws_bytes=8) == 7
    for bad in (dict(target=None), dict(target=4097), dict(us=None), dict(tokens=None), dict(batch=0), dict(k=-1),
                dict(k=65), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(drafts=None), dict(ua=None), dict(T=0.0),
                dict(T=-1.0), dict(T=math.nan), dict(T=math.inf), dict(row=-8), dict(T=9e-31), dict(T=1.1e30),
                dict(drafts=4100), dict(tokens=4100), dict(ua=4098), dict(us=4098)):
        assert call(**bad) == 3, bad


@gpu
def test_python_refusals():
    t, d, q, ua, us = (x.cuda() for x in inputs(1, 2, 2, 16, BF))
    f = sampling.verify_drafts
    for err, call in ((TypeError, lambda: f(t.half(), d, q.half(), ua, us)),
                      (ValueError, lambda: f(t, d, q.float(), ua, us)),
                      (ValueError, lambda: f(t, d[:, :1], q, ua, us)),
                      (ValueError, lambda: f(t, d.int(), q, ua, us)),
                      (ValueError, lambda: f(t, d.cpu(), q, ua, us)),
                      (ValueError, lambda: f(t, d, q[:, :1], ua, us)),
                      (ValueError, lambda: f(t, d, q, ua.double(), us)),
                      (ValueError, lambda: f(t, d, q, ua, us[:1])),
                      (ValueError, lambda: f(t, d, q, ua, us, 0.0)),
                      (ValueError, lambda: f(t, d, q, ua, us, -2.0)),
                      (ValueError, lambda: f(t, d, q, ua, us, math.nan)),
                      (ValueError, lambda: f(t, d, q, ua, us, 1e-31)),
                      (ValueError, lambda: f(t, d, q, ua, us, math.inf)),
                      (ValueError, lambda: sampling.sample_tokens(t[:, 0], ua)),
                      (ValueError, lambda: sampling.sample_tokens(t[:, 0], us, out=us)),):
        with pytest.raises(err):
            call()
    with pytest.raises(L.CdqError):
        big = torch.zeros(1, 66, 8, dtype=BF, device="cuda")
        f(big, torch.zeros(1, 65, dtype=torch.long, device="cuda"), None, torch.zeros(1, 65, device="cuda"), us[:1])


# ---------------------------------------------------------------- results


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,k,V,T", [(1, 0, 1, 1.0), (2, 1, 2, 0.7), (5, 3, 7, 1.0), (3, 2, 255, 2.0),
                                     (4, 4, 1001, 0.5), (2, 8, 4096, 1.0), (9, 1, 5003, 1.3), (40, 2, 777, 1.0),
                                     (2, 64, 130, 1.0), (1, 3, 151936, 0.8), (3, 1, 152063, 1.0)])
def test_verify(dtype, B, k, V, T):
    a = inputs(B * 1000 + V + k, B, k, V, dtype)
    same(run(*a, T), verify(*a, T))


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,k,V", [(3, 2, 500), (9, 4, 50021)])     # the second: more logits than are summed twice
@pytest.mark.parametrize("T", [1e-30, 1e-8, 1e8, 1e30])
def test_extreme_temperatures(dtype, B, k, V, T):
    """Towards the argmax and towards the uniform distribution, with tokens of probability 0 and the types' largest and
    lowest values."""
    t, d, q, ua, us = inputs(31, B, k, V, dtype)
    t[0, :, 5:60] = -math.inf
    q[1, :, 7] = -math.inf
    t[2, 0, 11], t[2, 1, 12] = torch.finfo(dtype).min, torch.finfo(dtype).max
    same(run(t, d, q, ua, us, T), verify(t, d, q, ua, us, T))
    got = sampling.sample_tokens(t[:, 0].cuda(), us.cuda(), T)
    assert got.tolist() == [drawn(softmax(t[b, 0], T), float(us[b])) for b in range(B)]


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("T", [1.0, 1.5, 2.0 ** 0.5])
def test_masks_of_every_size(dtype, T):
    """Logits below the others by amounts from 100 to the type's range, in steps of about a factor 1.1, and by powers
    of two in units of log2: none has any weight."""
    e = torch.arange(7, 127, 0.125, dtype=torch.float64)
    low = torch.cat([-torch.exp2(e), -torch.exp2(torch.arange(7, 60).double()) * T * math.log(2)]).to(dtype)
    row = torch.cat([torch.tensor([0.0, 1.0], dtype=dtype), low])
    t = row[None, None].repeat(7, 1, 1)
    us = torch.tensor([0.0, 0.2, 0.5, 0.9, 0.99, 1 - 2.0 ** -24, 1 - 2.0 ** -23])
    got = sampling.sample_tokens(t[:, 0].cuda(), us.cuda(), T)
    assert got.tolist() == [drawn(softmax(row, T), float(u)) for u in us]
    d = torch.ones(7, 1, dtype=torch.long)
    t = t.repeat(1, 2, 1)
    q = t[:, :1].flip(-1).contiguous()
    same(run(t, d, q, us[:, None], us, T), verify(t, d, q, us[:, None], us, T))


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_verify_greedy_drafts_and_short_ones(dtype):
    t, d, q, ua, us = inputs(5, 12, 4, 333, dtype)
    d = q.float().argmax(-1)
    d[3, 1], d[4, 0], d[5, 3], d[6, :] = -1, -7, -1, -1
    d[7, 0] = 333                                # beyond the vocabulary: never kept
    d[8, 1] = 2 ** 40
    same(run(t, d, None, ua, us, 1.0), verify(t, d, None, ua, us, 1.0))
    same(run(t, d, q, ua, us, 0.9), verify(t, d, q, ua, us, 0.9))


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_equal_distributions_keep_every_draft(dtype):
    t, d, q, ua, us = inputs(6, 6, 5, 2000, dtype)
    q = t[:, :5].clone()
    ua[:] = 1 - 2.0 ** -24                       # the largest number below 1
    got = run(t, d, q, ua, us, 1.0)
    assert got[1].tolist() == [5] * 6 and torch.equal(got[0][:, :5], d)
    ua[:, 2] = 1.0                               # not below 1: refused, and nothing is left of p - q: drawn from p
    got = run(t, d, q, ua, us, 1.0)
    assert got[1].tolist() == [2] * 6
    same(got, verify(t, d, q, ua, us, 1.0))


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("spread", [2.0, 0.1, 1e-2, 1e-4, 1e-6])
def test_near_distributions_of_large_batches(dtype, spread):
    """More logits than are summed twice, target and draft closer and closer (bf16 rounds the closest to the same, or
    to a few tokens apart); the last sequences: a shifted copy, and a copy with one token changed. Numbers that refuse
    whatever can be refused."""
    B, k, V = 9, 3, 60013
    t, _, q, ua, us = inputs(37, B, k, V, dtype, spread=spread)
    g = torch.Generator().manual_seed(41)
    d = torch.randint(0, V, (B, k), generator=g)
    ua[:] = 1 - 2.0 ** -24
    q[7] = t[7, :k] + 4
    t[7, :k] = q[7] - 4
    q[8] = t[8, :k]
    q[8, :, 17] += 3
    d[8, 0] = 17
    same(run(t, d, q, ua, us, 1.0), verify(t, d, q, ua, us, 1.0))


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_masked_and_broken_rows(dtype):
    t, d, q, ua, us = inputs(8, 10, 2, 600, dtype)
    ua[:] = 0                                    # whatever has any probability is kept
    t[0, :, 17:] = -math.inf                     # d is not among the 17: refused although u is 0
    t[1, 0, int(d[1, 0])] = -math.inf
    t[2, 1] = -math.inf                          # no distribution
    t[3, 0, 5] = math.nan
    t[4, 2, 599] = math.inf
    q[5, 1, 0] = math.nan
    q[6, 0] = -math.inf
    t[7] = torch.finfo(dtype).min                # the type's lowest value is a number like another
    t[8, :, 1:] = -math.inf
    q[8] = t[8, :2]
    d[8] = 0
    q[9, 0, 300:] = -math.inf
    got, want = run(t, d, q, ua, us, 1.0), verify(t, d, q, ua, us, 1.0)
    same(got, want)
    assert got[0][2].tolist() == [int(d[2, 0]), -1, -1] and got[0][3].tolist() == [-1, -1, -1]
    assert got[0][8].tolist() == [0, 0, 0]


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [3, 600, 20011])
def test_sample_borders(dtype, V):
    """u on both sides of a running sum's border, and at both ends of [0, 1)."""
    g = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=g).to(dtype)
    p = torch.softmax(row.double() / 0.9, 0)
    c = torch.cumsum(p, 0)
    pick = torch.randint(0, V - 1, (60,), generator=g)
    us = torch.cat([c[pick].float(), torch.tensor([0.0, 1 - 2.0 ** -24])])
    for e in (-2, -1, 1, 2):                     # neighbouring float32 numbers
        us = torch.cat([us, (c[pick].float().view(torch.int32) + e).view(torch.float32)])
    us = us.clamp(0, 1 - 2.0 ** -24)
    want = [drawn(p, float(u)) for u in us]
    x = row.expand(len(us), V).cuda()
    assert sampling.sample_tokens(x, us.cuda(), 0.9).tolist() == want
    assert sampling.sample_tokens(x.contiguous(), us.cuda(), 0.9).tolist() == want


@gpu
def test_strided_logits_and_out():
    t, d, q, ua, us = inputs(9, 3, 2, 500, BF)
    want = verify(t, d, q, ua, us, 1.0)
    wide = torch.full((3, 3, 523), 7.0, dtype=BF)
    wide[:, :, 5:505] = t
    wq = torch.full((2, 3, 501), 7.0, dtype=BF).transpose(0, 1)
    wq[:, :, 1:] = q
    a, b = wide.cuda()[:, :, 5:505], wq.cuda()[:, :, 1:]
    got = sampling.verify_drafts(a, d.cuda(), b, ua.cuda(), us.cuda())
    same((got[0].cpu(), got[1].cpu()), want)
    got = sampling.verify_drafts(t.transpose(1, 2).contiguous().transpose(1, 2).cuda(), d.cuda(), b, ua.cuda(), us.cuda())
    same((got[0].cpu(), got[1].cpu()), want)
    out = torch.zeros(3, dtype=torch.long, device="cuda")
    assert sampling.sample_tokens(a[:, 1], us.cuda(), out=out) is out
    assert out.tolist() == [drawn(softmax(t[i, 1], 1.0), float(us[i])) for i in range(3)]


@gpu
def test_streams_and_graphs():
    """Captured and replayed on new numbers; two graphs at once."""
    sets = []
    for seed in (11, 12):
        a = [x.cuda() for x in inputs(seed, 2, 3, 30000, BF)]
        sets.append(dict(a=a, g=torch.cuda.CUDAGraph(), s=torch.cuda.Stream()))
        sampling.verify_drafts(*a)
    torch.cuda.synchronize()
    for x in sets:
        with torch.cuda.graph(x["g"]):
            x["out"] = sampling.verify_drafts(*x["a"])
    for r in range(3):
        for x in sets:
            x["a"][4].copy_(torch.rand(2, generator=torch.Generator().manual_seed(r)))
        torch.cuda.synchronize()
        for x in sets:
            with torch.cuda.stream(x["s"]):
                x["g"].replay()
        torch.cuda.synchronize()
        for x in sets:
            same([t.cpu() for t in x["out"]], verify(*[t.cpu() for t in x["a"]], 1.0))


@gpu
def test_frequencies():
    """Verified tokens follow the target's distribution: 20000 draws over 5 tokens, each count within 5 standard
    deviations of its expectation."""
    N, V = 20000, 5
    g = torch.Generator().manual_seed(3)
    t = torch.randn(1, 2, V, generator=g).expand(N, 2, V).contiguous()
    q = torch.randn(1, 1, V, generator=g).expand(N, 1, V).contiguous()
    d = torch.multinomial(torch.softmax(q[:, 0], -1), 1, generator=g)
    tokens, _ = run(t, d, q, torch.rand(N, 1, generator=g), torch.rand(N, generator=g), 1.0)
    p = torch.softmax(t[0, 0].double(), -1)
    count = torch.bincount(tokens[:, 0], minlength=V).double()
    assert bool(((count - N * p).abs() < 5 * (N * p * (1 - p)).sqrt()).all())
