"""The quantised key/value cache against plain 64-bit implementations of its
formats and of attention, and its refusals."""
import ctypes as C
import math

import pytest
import torch

from cdq_lrr_b200 import _lib as L
from cdq_lrr_b200.kvcache import QuantKVCache

gpu = pytest.mark.gpu
BF = torch.bfloat16

# ---------------------------------------------------------------- plain forms, 64 bits


def grid_of(fmt):
    if fmt == "e2m1":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quantise(x, fmt):
    """x float64 [..., hd] (CPU) -> (values of the codes, bf16 scales), nearest code, ties to the even one."""
    grid = grid_of(fmt)
    size = x.shape[-1] if fmt == "e4m3" else 32
    g = x.reshape(*x.shape[:-1], -1, size)
    amax = g.abs().amax(-1)
    s = (amax.float().clamp(min=2.0 ** -100) / (448.0 if fmt == "e4m3" else 6.0)).to(BF)
    s = torch.where(torch.isfinite(amax), s, torch.full_like(s, math.nan))
    y = (g.float() / s.float()[..., None]).double()
    y = torch.where(torch.isfinite(y), y, torch.zeros_like(y))
    a = y.abs().clamp(max=grid[-1])
    hi = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    v = grid[torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)] * torch.sign(y)
    return v.reshape(x.shape), s.squeeze(-1) if fmt == "e4m3" else s


def values(cache):
    """What a cache holds, float64 on the CPU: k, v [batch, kv_heads, max_len, hd]."""
    out = []
    for codes, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes, s = codes.cpu(), s.cpu().double()
        if cache.fmt == "e4m3":
            out.append(codes.double() * s[..., None])
        else:
            c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
            vals = torch.cat([grid_of("e2m1"), -grid_of("e2m1")])[c]
            out.append(vals * s.repeat_interleave(32, -1))
    return out


def rotate(x, cos, sin):
    """x float64 [..., hd], tables [..., hd]."""
    h = x.shape[-1] // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * cos.double() + turned * sin.double()


def tables(n, hd, device="cuda"):
    inv = 1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    a = torch.cat([a, a], -1)
    return a.cos().to(BF).to(device), a.sin().to(BF).to(device)


def attention(q, pos, cache, rope, rope_pos, scale, prefix=None, P=0):
    """(out, bound) in 64 bits; bound: how far a result in the kernel's steps may be off.

    The kernel rounds a rotated query element to half (relative 2^-11, or 2^-25 of its row's largest), which
    moves a score by at most d = 2^-11 * |scale| * sum |q k| (an error of a product scaled by a negative number is as
    large as by its magnitude; twice that for the small elements' floor), and so a
    probability by a factor within e^(2 d), numerator and denominator; it rounds a weight to half (2^-11, and
    2^-25 of the row's largest contribution, absolute); sums, ex2 and the float32 scales add less than 2^-13 in
    all at these lengths; the result is rounded to bf16 (2^-8). All but the last act on sum p |v|."""
    K, V = values(cache)
    B, n, H, hd = q.shape
    G = H // cache.kv_heads
    q = q.cpu().double()
    out = torch.zeros(B, n, H, hd, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(B):
        p0 = int(pos[b])
        if p0 < 0:
            continue
        for i in range(n):
            if p0 + i >= cache.max_len:
                out[b, i] = math.nan
                continue
            for h in range(H):
                k, v = K[b, h // G, :p0 + i + 1], V[b, h // G, :p0 + i + 1]
                if prefix is not None:
                    k = torch.cat([prefix[0][0, h // G, :P], k])
                    v = torch.cat([prefix[1][0, h // G, :P], v])
                x = q[b, i, h]
                if rope is not None:
                    t = (p0 if rope_pos is None else int(rope_pos[b])) + i
                    x = rotate(x, rope[0][t].cpu(), rope[1][t].cpu())
                s = k @ x * scale
                p = torch.softmax(s, 0)
                out[b, i, h] = p @ v
                d = float(((k.abs() @ x.abs()) * abs(scale)).max()) * (2 * 2.0 ** -11 if rope is not None else 2.0 ** -20)
                top = (p[:, None] * v.abs()).max()
                bound[b, i, h] = (p @ v.abs()) * (math.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -13) \
                    + top * 2.0 ** -22 * len(p) ** 0.5 + out[b, i, h].abs() * 2.0 ** -8
    return out, bound


def check(got, want, bound):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs() - bound - 1e-30
    off = off[~torch.isnan(off)]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def normal(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(BF).cuda()


def int32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def filled(seed, B, kv, L_, hd, fmt, scale=1.0):
    c = QuantKVCache(B, kv, L_, hd, fmt)
    c.append(normal(seed, B, L_, kv, hd, scale=scale), normal(seed + 1, B, L_, kv, hd, scale=scale),
             int32(*[0] * B))
    return c


# ---------------------------------------------------------------- refusals (no GPU)


def test_constructor_refusals():
    for bad in (dict(fmt="int8"), dict(head_dim=96), dict(batch=0), dict(max_len=0), dict(kv_heads=0)):
        a = dict(batch=1, kv_heads=2, max_len=8, head_dim=64, fmt="e4m3", device="cpu") | bad
        with pytest.raises(ValueError):
            QuantKVCache(**a)
    k = torch.zeros(1, 2, 8, 64, dtype=torch.uint8)
    s = torch.zeros(1, 2, 8, 4, dtype=BF)
    assert QuantKVCache.from_buffers(k, k.clone(), s, s.clone()).head_dim == 128
    with pytest.raises(ValueError):
        QuantKVCache.from_buffers(k, k.clone(), s[..., :2], s)
    with pytest.raises(TypeError):
        QuantKVCache.from_buffers(k.float(), k.float(), s, s)
    with pytest.raises(TypeError):
        QuantKVCache.from_buffers(k, k.clone(), s.float(), s.float())
    with pytest.raises(ValueError):
        QuantKVCache.from_buffers(k.transpose(1, 2), k.transpose(1, 2), s, s)
    with pytest.raises(ValueError):
        QuantKVCache.from_buffers(k, torch.zeros(1, 2, 9, 64, dtype=torch.uint8), s, s)


def test_cpu_tensors_are_refused():
    c = QuantKVCache(1, 2, 8, 64, device="cpu")
    x = torch.zeros(1, 1, 2, 64, dtype=BF)
    p = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: c.append(x, x, p), lambda: c.attend(x, p), lambda: c.read(p, 1)):
        with pytest.raises(RuntimeError):
            call()


def test_c_abi_refusals():
    """Arguments that are refused before anything is launched."""
    lib = L.lib()
    ok = dict(k=4096, v=8192, k_scale=64, v_scale=128, batch=1, kv_heads=2, max_len=8, head_dim=64, format=0)

    def cache(**kw):
        s = L.cdq_kv_cache()
        for name, v in (ok | kw).items():
            setattr(s, name, v)
        return C.byref(s)

    def append(c, k=4096, seq=128, tok=128, pos=4096, n=1, cos=None, sin=None, rows=0):
        return lib.cdq_kv_append(c, k, seq, tok, 4096, 128, 128, pos, n, cos, sin, rows, None, None)

    assert append(None) == 3
    assert append(cache(format=2)) == 8
    assert append(cache(head_dim=80)) == 8
    assert append(cache(batch=0)) == 1
    assert append(cache(max_len=0)) == 1
    assert append(cache(k=4100)) == 3
    assert append(cache(v_scale=130)) == 3
    assert append(cache(), k=4104) == 3      # rows not 16-byte aligned
    assert append(cache(), tok=132) == 3     # nor their stride
    assert append(cache(), seq=-128) == 3
    assert append(cache(), pos=None) == 3
    assert append(cache(), n=0) == 3
    assert append(cache(), cos=4096, rows=4) == 3            # a cosine table without a sine table
    assert append(cache(), cos=4096, sin=4096) == 3          # empty tables
    assert append(cache(), cos=4096, sin=4104, rows=4) == 3
    assert lib.cdq_kv_read(cache(), None, 1, 4096, None, None) == 3
    b = C.c_int64()
    ws = lib.cdq_kv_attend_workspace
    assert ws(cache(), 3, 1, None, C.byref(b)) == 3                  # heads over kv heads
    assert ws(cache(), 4, 0, None, C.byref(b)) == 3
    assert ws(cache(), 4, L.KV_MAX_NEW + 1, None, C.byref(b)) == 3
    assert ws(cache(), 4, 1, None, None) == 3
    for out in (None, 1 << 20 | 2, 4096 + 64, 4096 - 64):   # not 16-byte aligned; over the queries at 4096
        assert lib.cdq_kv_attend(cache(), 4096, 128, 128, 2, 1, 4096, None, None, 0, None, 0.125, None, None, out,
                                 None, 0, None) == 3


@gpu
def test_python_refusals():
    c = QuantKVCache(2, 2, 8, 64)
    x, p = normal(1, 2, 1, 2, 64), int32(0, 0)
    cos, sin = tables(8, 64)
    one = QuantKVCache(1, 2, 8, 64)
    for err, call in (
            (TypeError, lambda: c.append(x.float(), x, p)),
            (ValueError, lambda: c.append(x[:1], x[:1], p)),
            (ValueError, lambda: c.append(x, x.repeat(1, 2, 1, 1), p)),
            (ValueError, lambda: c.append(x, x, p.long())),
            (ValueError, lambda: c.append(x, x, p.cpu())),
            (ValueError, lambda: c.append(x, x, int32(0))),
            (ValueError, lambda: c.append(x, x, p, rope=(cos.float(), sin.float()))),
            (ValueError, lambda: c.append(x, x, p, rope=(cos, sin[:4]))),
            (ValueError, lambda: c.append(x, x, p, rope_pos=p)),
            (ValueError, lambda: c.attend(normal(1, 2, 1, 3, 64), p)),
            (ValueError, lambda: c.attend(normal(1, 2, 65, 2, 64), p)),
            (ValueError, lambda: c.attend(x[:, :0], p)),
            (ValueError, lambda: c.attend(x, p, prefix=one)),
            (ValueError, lambda: c.attend(x, p, prefix_len=int32(3))),
            (ValueError, lambda: c.attend(x, p, prefix=c, prefix_len=int32(3))),
            (ValueError, lambda: c.attend(x, p, prefix=QuantKVCache(1, 2, 8, 64, "e2m1"), prefix_len=int32(3))),
            (ValueError, lambda: c.attend(x, p, out=torch.empty(2, 1, 2, 64, device="cuda"))),
            (ValueError, lambda: c.attend(x, p, out=torch.empty(257, dtype=BF, device="cuda")[1:].view(2, 1, 2, 64))),
            (ValueError, lambda: c.attend(x, p, out=x)),
            (ValueError, lambda: c.read(p, -1)),
    ):
        with pytest.raises(err):
            call()
    both = normal(2, 1, 2, 2, 64)     # two rows: queries in the first, results in the second are apart
    assert torch.equal(one.attend(both[:, :1], int32(0), out=both[:, 1:]), torch.zeros_like(both[:, 1:]))
    with pytest.raises(ValueError):
        one.attend(both[:, :1], int32(0), out=both.view(-1)[64:192].view(1, 1, 2, 64))
    c.append(x[:, :0], x[:, :0], p)   # nothing to write
    assert c.read(p, 0)[0].shape == (2, 0, 2, 64)


# ---------------------------------------------------------------- writing and reading back


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd,kv,n", [(64, 2, 1), (128, 4, 3), (64, 3, 37), (128, 1, 130)])
@pytest.mark.parametrize("rope", [False, True])
def test_append_and_read(fmt, hd, kv, n, rope):
    """Scales and codes of every written element against the formats' definitions (v: to the bit; k: a rotated
    element is a float32 sum, off by 2^-24 of it, which can move a code on a border by one step: at most 1 in 10^4
    does), untouched positions as they were, and the values read back."""
    B, Lm = 3, n + 9
    c = QuantKVCache(B, kv, Lm, hd, fmt)
    k, v = normal(3, B, n, kv, hd), normal(4, B, n, kv, hd)
    k[0, 0, 0, :8] *= 50                                    # an outlier
    v[B - 1, n - 1, kv - 1] = 0                             # a row of zeros
    pos = int32(2, 0, 9)
    cos, sin = tables(Lm + 40, hd)
    at = int32(5, 31, 0)
    c.append(k, v, pos, rope=(cos, sin) if rope else None, rope_pos=at if rope else None)
    got_k, got_v = values(c)
    rk, rv = c.read(pos, n)
    for b in range(B):
        p = int(pos[b])
        kk = k[b].cpu().double()
        if rope:
            t = int(at[b])
            kk = rotate(kk, cos[t:t + n, None].cpu(), sin[t:t + n, None].cpu())
            kk = kk.float().double()
        for x, held, scales, back in ((kk, got_k, c.k_scale, rk), (v[b].cpu().double(), got_v, c.v_scale, rv)):
            want, s = quantise(x, fmt)
            assert torch.equal(scales[b, :, p:p + n].cpu().transpose(0, 1), s)
            sf = s.double()[..., None] if fmt == "e4m3" else s.double().repeat_interleave(32, -1)
            mine = held[b, :, p:p + n].transpose(0, 1)
            wrong = mine != want * sf
            assert wrong.float().mean() <= (1e-4 if rope and x is kk else 0)
            assert torch.equal(back[b].cpu(), mine.to(BF))
            assert not held[b, :, :p].any() and not held[b, :, p + n:].any()


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_ties_and_extremes(fmt):
    """Elements on the border between two codes, the largest and smallest magnitudes, and rows that cannot be held."""
    hd, c = 64, QuantKVCache(1, 1, 8, 64, fmt)
    grid = grid_of(fmt)
    mids = ((grid[1:] + grid[:-1]) / 2)[-40:]
    rows = torch.zeros(8, hd, dtype=torch.float64)
    rows[0, :len(mids)] = mids
    rows[0, 40:40 + min(24, len(mids))] = -mids[:24]
    rows[0, 31] = rows[0, 63] = grid[-1]                     # the scale is 1
    rows[1] = 3.38e38
    rows[2] = 1e-38                                          # below the scale's floor: zeros
    rows[3] = torch.linspace(-1, 1, hd) * 2.0 ** -60
    rows[4] = 1.0
    rows[4, 5] = math.nan
    rows[5] = 1.0
    rows[5, 40] = -math.inf
    rows[6, 7] = 5e-39                                       # a subnormal
    x = rows.to(BF).reshape(1, 8, 1, hd).cuda()
    c.append(x, x, int32(0))
    want, s = quantise(x[0, :, 0].cpu().double(), fmt)
    sf = s.double()[:, None] if fmt == "e4m3" else s.double().repeat_interleave(32, -1)
    for held in values(c):
        assert torch.allclose(held[0, 0], want * sf, rtol=0, atol=0, equal_nan=True)
    k, v = c.read(None, 8)
    assert torch.isnan(k[0, 4, 0, 5]) and torch.isnan(k[0, 5, 0, 40])
    assert bool(torch.isnan(k[0, 4, 0, 63])) == (fmt == "e4m3")  # the other group of 32 is whole
    assert torch.equal(k.isnan(), v.isnan())


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_positions_that_do_not_fit(fmt):
    c = filled(5, 3, 2, 10, 64, fmt)
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    x = normal(6, 3, 4, 2, 64)
    c.append(x, x, int32(-1, 8, 2 ** 31 - 2))
    for t, old in zip((c.k, c.v, c.k_scale, c.v_scale), before):
        t, old = t.view(torch.uint8), old.view(torch.uint8)
        assert torch.equal(t[0], old[0]) and torch.equal(t[2], old[2])
        assert torch.equal(t[1, :, :8], old[1, :, :8]) and not torch.equal(t[1, :, 8:], old[1, :, 8:])
    k, v = c.read(int32(-5, 7, 10), 4)
    assert not k[0].any() and not k[2].any() and not k[1, 3].any() and k[1, :3].any()
    # a rotary position outside the tables
    c.append(x, x, int32(0, 0, 0), rope=tables(6, 64), rope_pos=int32(3, -1, 0))
    k, v = c.read(None, 4)
    bad = torch.isnan(k).all(-1).all(-1).cpu()
    assert bad.tolist() == [[False, False, False, True], [True, False, False, False], [False] * 4]
    assert not torch.isnan(v).any()


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_strided_inputs(fmt):
    """k, v and q as slices of one fused projection output, and a layout that has to be copied."""
    B, n, H, kv, hd = 2, 3, 6, 2, 64
    fused = normal(7, B, n, H + 2 * kv, hd)
    q, k, v = fused[:, :, :H], fused[:, :, H:H + kv], fused[:, :, H + kv:]
    a, b, d = (QuantKVCache(B, kv, 12, hd, fmt) for _ in range(3))
    pos = int32(0, 5)
    a.append(k, v, pos)
    b.append(k.contiguous(), v.contiguous(), pos)
    d.append(k.transpose(2, 3).contiguous().transpose(2, 3), v.transpose(0, 1).contiguous().transpose(0, 1), pos)
    for t, u, w in zip((a.k, a.v, a.k_scale, a.v_scale), (b.k, b.v, b.k_scale, b.v_scale),
                       (d.k, d.v, d.k_scale, d.v_scale)):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    assert torch.equal(a.attend(q, pos), a.attend(q.contiguous(), pos))
    assert torch.equal(a.attend(q, pos), a.attend(q.transpose(2, 3).contiguous().transpose(2, 3), pos))
    one = q[:1, :1].expand(B, n, H, hd)
    assert torch.equal(a.attend(one, pos), a.attend(one.contiguous(), pos))


# ---------------------------------------------------------------- attention


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,H,kv,pos", [
    (1, 14, 2, (0, 1, 15, 16, 17, 63, 64, 299)),
    (1, 8, 8, (130, -1, 5)),
    (5, 14, 2, (0, 250, 59)),
    (3, 5, 1, (7,)),
    (2, 24, 2, (100, 33)),
    (64, 4, 2, (0, 200)),
    (7, 20, 1, (122,)),
])
def test_attend(fmt, hd, n, H, kv, pos):
    B, Lm = len(pos), 333
    c = filled(11, B, kv, Lm, hd, fmt)
    q = normal(13, B, n, H, hd, scale=2.0)
    rope = tables(Lm, hd)
    out = c.attend(q, int32(*pos), rope=rope)
    check(out, *attention(q, pos, c, rope, None, hd ** -0.5))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("B,H,kv,hd,pos", [(1, 7, 1, 64, 9000), (1, 16, 2, 128, 5003), (2, 3, 1, 128, 6001)])
def test_attend_split_positions(fmt, B, H, kv, hd, pos):
    """A long axis split over CTAs and joined, against the same in 64 bits; more than one call gives the same bits."""
    c = filled(17, B, kv, 9100, hd, fmt)
    q = normal(19, B, 1, H, hd, scale=3.0)
    p = [pos - 11 * b for b in range(B)]
    out = c.attend(q, int32(*p), scale=0.2)
    check(out, *attention(q, p, c, None, None, 0.2))
    assert torch.equal(out, c.attend(q, int32(*p), scale=0.2))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,H,kv,Lm,pos", [
    (1, 14, 2, 1100, (0, 126, 127, 128, 255, 256, 1024, 1099)),      # nine units over eight CTAs
    (1, 7, 1, 2048, (2047, -1, 1151, 1152)),
    (3, 6, 2, 1000, (997, 998, 126, 640)),                          # past the end; both sides of a unit in one call
    (9, 10, 1, 257, (250, 0)),
])
def test_attend_in_clusters(fmt, hd, n, H, kv, Lm, pos):
    """Caches of 2 to 16 units, whose segments a cluster of CTAs joins without a workspace."""
    c = filled(183, len(pos), kv, Lm, hd, fmt)
    q = normal(191, len(pos), n, H, hd, scale=2.0)
    rope = tables(Lm + n, hd)
    need = C.c_int64()
    L.check(L.lib().cdq_kv_attend_workspace(c._ref, H, n, None, C.byref(need)), "workspace")
    assert need.value == 0
    out = c.attend(q, int32(*pos), rope=rope)
    check(out, *attention(q, pos, c, rope, None, hd ** -0.5))
    assert torch.equal(out.view(torch.int16), c.attend(q, int32(*pos), rope=rope).view(torch.int16))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("B,n,H,kv,hd,P,pos", [
    (2, 1, 14, 2, 64, 100, (0, 40)),
    (5, 2, 8, 2, 128, 257, (0, 3, -1, 64, 17)),
    (3, 1, 4, 4, 64, 1, (0, 1, 2)),
    (2, 4, 6, 1, 64, 0, (9, 30)),
    (9, 3, 7, 1, 128, 1030, tuple(range(9))),
])
def test_attend_prefix(fmt, B, n, H, kv, hd, P, pos):
    c = filled(23, B, kv, 80, hd, fmt)
    pre = filled(29, 1, kv, 1100, hd, fmt)
    q = normal(31, B, n, H, hd, scale=2.0)
    rope = tables(P + 80, hd)
    rp = [P + x for x in pos]
    out = c.attend(q, int32(*pos), rope=rope, rope_pos=int32(*rp), prefix=pre, prefix_len=int32(P))
    check(out, *attention(q, pos, c, rope, rp, hd ** -0.5, values(pre), P))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_prefix_lengths_that_do_not_fit(fmt):
    c, pre = filled(23, 2, 1, 8, 64, fmt), filled(29, 1, 1, 20, 64, fmt)
    q = normal(31, 2, 1, 2, 64)
    got = c.attend(q, int32(3, -1), prefix=pre, prefix_len=int32(21))
    assert torch.isnan(got[0]).all() and not got[1].any()
    got = c.attend(q, int32(3, 0), prefix=pre, prefix_len=int32(-4))
    assert torch.equal(got, c.attend(q, int32(3, 0), prefix=pre, prefix_len=int32(0)))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_what_is_hidden_does_not_matter(fmt):
    """NaN in every position behind a sequence's last, in later new positions, in another sequence and in the idle
    sequence's query; positions past the cache give NaN and no more."""
    B, kv, Lm, hd, n, H = 4, 2, 96, 64, 3, 6
    pos = (40, 94, -1, 10)
    c, clean = filled(37, B, kv, Lm, hd, fmt), filled(37, B, kv, Lm, hd, fmt)
    q = normal(41, B, n, H, hd)
    want = clean.attend(q, int32(*pos))
    for codes in (c.k, c.v):
        codes.view(torch.uint8)[0, :, 43:] = 0x7F            # e4m3: the code of NaN
        codes.view(torch.uint8)[2] = 0x7F
    bad = normal(43, B, Lm, kv, hd)
    bad[:] = math.nan
    keep = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    c.append(bad[:, :1], bad[:, :1], int32(42, -1, 5, 12))   # the newest position of sequences 0 and 3
    q2 = q.clone()
    q2[2] = math.nan
    got = c.attend(q2, int32(*pos))
    for b, n_ok in ((0, 2), (1, 2), (3, 2)):
        assert torch.equal(got[b, :n_ok], want[b, :n_ok]), b
    assert torch.isnan(got[0, 2]).all() and torch.isnan(got[3, 2]).all()
    assert torch.isnan(got[1, 2]).all() and torch.isnan(want[1, 2]).all()   # position 96 of 96
    assert not got[2].any()
    del keep
    q3 = q.clone()
    q3[0, 1, 4] = math.inf                                    # one head's query is broken: that row alone
    got = clean.attend(q3, int32(*pos))
    same = torch.isnan(got) == torch.isnan(want)
    assert torch.isnan(got[0, 1, 4]).all() and int((~same).sum()) == hd
    q3[0, 1, 4] = q[0, 1, 4]
    assert torch.equal(clean.attend(q3, int32(*pos))[0], want[0])


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
def test_value_scales_of_all_sizes(fmt, hd):
    """Values whose magnitudes differ by 10^6 between positions (and groups): the small ones count where the large
    ones have no weight. Position j's value is about 10^(j % 7 - 3), keys point away from the large ones."""
    kv, Lm = 1, 70
    k, v = normal(47, 1, Lm, kv, hd), normal(53, 1, Lm, kv, hd)
    mag = 10.0 ** (torch.arange(Lm, device="cuda") % 7 - 3).float()
    v = (v.float() * mag[None, :, None, None]).to(BF)
    v[..., 32:] = (v[..., 32:].float() * 1e-5).to(BF)
    q = normal(59, 1, 1, 3, hd, scale=4.0)
    k[0, mag > 5] = (-8 * q[0, 0, :1].float() / q[0, 0, :1].float().norm() * 4).to(BF)
    c = QuantKVCache(1, kv, Lm, hd, fmt)
    c.append(k, v, int32(0))
    want, bound = attention(q, (Lm - 1,), c, None, None, hd ** -0.5)
    got = c.attend(q, int32(Lm - 1))
    check(got, want, bound)


@gpu
def test_large_and_small_queries():
    """A query row's magnitude has no say in its precision: powers of two scale the scores exactly."""
    c = filled(61, 1, 2, 50, 64, "e4m3")
    q = normal(67, 1, 2, 4, 64)
    want = c.attend(q, int32(48), scale=0.125)
    for e in (-100, -30, 30, 100):
        got = c.attend((q.float() * 2.0 ** e).to(BF), int32(48), scale=0.125 * 2.0 ** -e)
        assert torch.equal(got, want), e
    q[:] = 0   # the mean of the values, every row alike
    got = c.attend(q, int32(48))
    assert torch.equal(got[0, 0, 0], got[0, 0, 1])


@gpu
def test_long_cache_offsets():
    """Byte offsets past 2^31 within one head's keys."""
    Lm, hd = (1 << 24) + 70000, 128
    if torch.cuda.mem_get_info()[0] < 6 * Lm * hd:
        pytest.skip("needs 13 GB of device memory")
    c = QuantKVCache(1, 1, Lm, hd, "e4m3")
    n = 64
    k, v = normal(71, 1, n, 1, hd), normal(73, 1, n, 1, hd)
    pos = int32(Lm - n)
    c.append(k, v, pos)
    k2, v2 = c.read(pos, n)
    small = QuantKVCache(1, 1, n, hd, "e4m3")
    small.append(k, v, int32(0))
    ks, vs = small.read(int32(0), n)
    assert torch.equal(k2, ks) and torch.equal(v2, vs)
    assert not c.read(int32(0), 3)[0].any()
    # all but the last positions are zero keys and zero values: weight e^0 each
    q = (k[:, -1:] * 8).expand(1, 1, 2, hd).contiguous()
    K, V = (x[0, 0] for x in values(small))
    x = q[0, 0, 0].cpu().double()
    s = K @ x * hd ** -0.5
    e = torch.exp(s - s.max())
    p = e / (e.sum() + (Lm - n) * torch.exp(-s.max()))
    d = float((K.abs() @ x.abs()).max()) * hd ** -0.5 * 2.0 ** -20
    want = p @ V
    bound = (p @ V.abs()) * (math.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -13) + want.abs() * 2.0 ** -8 \
        + float((p[:, None] * V.abs()).max()) * 2.0 ** -22 * 8
    for h in range(2):
        check(c.attend(q, int32(Lm - 1))[0, 0, h], want, bound)


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_other_streams_and_graphs(fmt):
    """append + attend captured and replayed at new positions, two graphs at once on two streams, each with the
    same results as eager calls."""
    B, kv, H, hd, Lm = 2, 2, 14, 64, 700
    rope = tables(Lm, hd)
    sets = []
    for seed in (79, 83):
        c = filled(seed, B, kv, Lm, hd, fmt)
        sets.append(dict(c=c, q=normal(seed + 2, B, 1, H, hd), k=normal(seed + 3, B, 1, kv, hd),
                         v=normal(seed + 4, B, 1, kv, hd), pos=int32(600, 20)))

    def step(s):
        s["c"].append(s["k"], s["v"], s["pos"], rope=rope)
        return s["c"].attend(s["q"], s["pos"], rope=rope)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            s["eager"] = step(s)
    torch.cuda.current_stream().wait_stream(side)
    for s in sets:
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = step(s)
    streams = [torch.cuda.Stream() for _ in sets]
    for shift in (0, 1, 2):
        for s, st in zip(sets, streams):
            s["pos"].copy_(int32(600 + shift, 20 + shift))
        torch.cuda.synchronize()
        for _ in range(5):
            for s, st in zip(sets, streams):
                with torch.cuda.stream(st):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            got = s["out"].clone()
            assert torch.equal(got, step(s)), shift
            if shift == 0:
                assert torch.equal(got, s["eager"])


@gpu
def test_batch_rows_do_not_depend_on_each_other():
    """A sequence's output is the same alone and in a batch up to the order of its split sums (two bf16 roundings
    and 2^-13 of sum p |v| apart at most: the bound of either side)."""
    c = filled(89, 4, 2, 400, 64, "e4m3")
    q = normal(97, 4, 2, 8, 64)
    pos = (5, 390, 77, 200)
    got = c.attend(q, int32(*pos))
    for b in range(4):
        one = QuantKVCache.from_buffers(*(t[b:b + 1].clone() for t in (c.k, c.v, c.k_scale, c.v_scale)))
        want, bound = attention(q[b:b + 1], pos[b:b + 1], one, None, None, 0.125)
        check(one.attend(q[b:b + 1], int32(pos[b])), want, bound)
        check(got[b:b + 1], want, bound)


# ---------------------------------------------------------------- many rows (e4m3: the tensor-memory kernel)


def roomy(c, n_rows, spare=5):
    """A cache with c's contents and room for so many positions that `n_rows` rows of a pass over it are a matter for
    the tensor-memory kernel (8 units of 128 positions and 128 rows a multiprocessor)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = -(-n_rows // 128)
    per = -(-8 * sms // (c.batch * c.kv_heads * tiles))
    big = QuantKVCache(c.batch, c.kv_heads, max(128 * per - spare, c.max_len), c.head_dim, c.fmt)
    for a, b in ((big.k, c.k), (big.v, c.v)):
        a.view(torch.uint8)[:, :, :c.max_len] = b.view(torch.uint8)
    big.k_scale[:, :, :c.max_len] = c.k_scale
    big.v_scale[:, :, :c.max_len] = c.v_scale
    return big


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,H,kv,Lm,pos,scale", [
    (64, 4, 2, 333, (5, 269), None),                   # a whole tile; the last positions of the cache
    (33, 6, 2, 260, (0, 100, 127), -0.1),              # 99 rows; a scale below zero
    (64, 8, 1, 513, (-1, 0, 480, 513, 400), 0.3),      # 512 rows, four tiles; idle, past the end from the middle on
    (17, 16, 4, 300, tuple((37 * b) % 290 - 1 for b in range(20)), None),  # more segments than CTAs
    (65 - 32, 2, 1, 1, (0, -1), 0.0),                  # one position; no weight differs
    (41, 2, 1, 130, (0, 89), 0.0),
])
@pytest.mark.parametrize("rope", [True, False])
def test_attend_many_rows(fmt, hd, n, H, kv, Lm, pos, scale, rope):
    B = len(pos)
    c = filled(101, B, kv, Lm, hd, fmt)
    q = normal(103, B, n, H, hd, scale=2.0)
    t = tables(Lm + n, hd) if rope else None
    out = c.attend(q, int32(*pos), rope=t, scale=scale)
    want, bound = attention(q, pos, c, t, None, hd ** -0.5 if scale is None else scale)
    check(out, want, bound)
    big = roomy(c, n * H // kv)
    got = big.attend(q, int32(*pos), rope=t, scale=scale)
    in_c = (torch.tensor(pos)[:, None] + torch.arange(n) < Lm).cuda()
    check(torch.where(in_c[..., None, None], got, out), want, bound)
    for x, y in ((out, c), (got, big)):
        assert torch.equal(x.view(torch.int16), y.attend(q, int32(*pos), rope=t, scale=scale).view(torch.int16))
    assert L.kernel_error() == 0


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_at_the_end_of_a_long_cache(hd):
    """The last positions of a cache of many units: split over every multiprocessor and joined; rows past the end."""
    c = roomy(QuantKVCache(1, 1, 8, hd), 81, spare=41)
    Lm, n, H = c.max_len, 27, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(1, Lm, 1, hd, device="cuda", generator=g).to(BF) for _ in range(2))
    c.append(k, v, int32(0))
    q = normal(181, 1, n, H, hd, scale=2.0)
    for pos in (Lm - n, Lm - 9, Lm // 2 + 77):
        check(c.attend(q, int32(pos)), *attention(q, (pos,), c, None, None, hd ** -0.5))
    assert L.kernel_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd,B,n,H,kv,P", [(64, 34, 1, 4, 2, 1500), (128, 23, 3, 2, 1, 129), (128, 5, 16, 4, 4, 6000)])
def test_prefix_many_rows(fmt, hd, B, n, H, kv, P):
    c, pre = filled(107, B, kv, 70, hd, fmt), filled(109, 1, kv, P + 3, hd, fmt)
    pos = [(13 * b) % 50 - 1 for b in range(B)]
    q = normal(113, B, n, H, hd, scale=2.0)
    got = c.attend(q, int32(*pos), prefix=pre, prefix_len=int32(P))
    check(got, *attention(q, pos, c, None, None, hd ** -0.5, values(pre), P))
    big = roomy(pre, B * n * H // kv)
    for short in (0, 1, 128, P):
        want, bound = attention(q, pos, c, None, None, hd ** -0.5, values(pre), short)
        for p in (pre, big):
            check(c.attend(q, int32(*pos), prefix=p, prefix_len=int32(short)), want, bound)
    for p in (pre, big):
        got = c.attend(q, int32(*pos), prefix=p, prefix_len=int32(p.max_len + 1))
        for b in range(B):
            assert (torch.isnan(got[b]).all() if pos[b] >= 0 else not got[b].any()), b
    assert L.kernel_error() == 0


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("order", [1, -1])
def test_many_rows_value_scales_of_all_sizes(fmt, hd, order):
    """Positions' values from 2^-60 to 2^60, rising or falling along the axis (rising: the largest contribution moves
    with nearly every position), and scores against them, so that every size has some weight."""
    n, H, Lm = 45, 2, 400
    k, v = normal(127, 1, Lm, 1, hd), normal(131, 1, Lm, 1, hd)
    e = (torch.arange(Lm, device="cuda") - Lm // 2).float() * (0.3 * order)
    v = (v.float() * torch.exp2(e)[None, :, None, None]).to(BF)
    k[..., 0] = (-e * 0.5).to(BF)[None, :, None]
    q = normal(137, 1, n, H, hd, scale=0.5)
    q[..., 0] = 8.0
    c = QuantKVCache(1, 1, Lm, hd, fmt)
    c.append(k, v, int32(0))
    # e4m3 keys: the row's scale follows its largest element, the others are coarse; the plain form sees the codes
    want, bound = attention(q, (Lm - n,), c, None, None, 0.12)
    for x in (c, roomy(c, n * H)):
        check(x.attend(q, int32(Lm - n), scale=0.12), want, bound)
    assert L.kernel_error() == 0


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("room", [False, True])
def test_many_rows_hidden_positions(hd, room):
    """NaN codes and scales behind every sequence's last position and in an idle sequence; NaN in newer positions
    reaches the rows that see them and no others; an infinite query element its own row alone."""
    B, kv, Lm, n, H = 3, 1, 400, 50, 2
    pos = (100, -1, 250)
    c = roomy(filled(139, B, kv, Lm, hd, "e4m3"), n * H) if room else filled(139, B, kv, Lm, hd, "e4m3")
    q = normal(149, B, n, H, hd)
    for t in (c.k, c.v):
        t.view(torch.uint8)[0, :, 150:] = 0x7F
        t.view(torch.uint8)[1] = 0x7F
    c.k_scale[0, :, 150:] = math.nan
    c.v_scale[0, :, 150:] = math.nan
    q2 = q.clone()
    q2[1] = math.nan
    got = c.attend(q2, int32(*pos))
    check(got, *attention(q2, pos, c, None, None, hd ** -0.5))
    assert not torch.isnan(got).any()
    nan = torch.full((B, 1, kv, hd), math.nan, dtype=BF, device="cuda")
    c.append(nan, nan, int32(130, -1, 299))
    q2[2, 7, 1, 3] = math.inf
    got = c.attend(q2, int32(*pos))
    check(got, *attention(q2, pos, c, None, None, hd ** -0.5))
    bad = torch.isnan(got).all(-1)
    assert int(bad.sum()) == (20 + 1) * H + 1 and bad[0, 30:].all() and bad[2, 49].all() and bad[2, 7, 1]
    assert L.kernel_error() == 0


@gpu
def test_many_rows_on_two_streams():
    """Two graphs of the tensor-memory kernel and its join at once, each with a prefix, against eager calls."""
    B, kv, H, hd, n = 3, 2, 8, 128, 20
    sets = []
    for seed in (151, 157):
        s = dict(c=roomy(filled(seed, B, kv, 500, hd, "e4m3"), n * H // kv),
                 pre=roomy(filled(seed + 1, 1, kv, 2100, hd, "e4m3"), B * n * H // kv),
                 q=normal(seed + 2, B, n, H, hd), pos=int32(0, 300, 479), len=int32(2100))
        s["run"] = lambda s=s: s["c"].attend(s["q"], s["pos"], prefix=s["pre"], prefix_len=s["len"])
        s["want"] = [s["run"]()]
        sets.append(s)
    torch.cuda.synchronize()
    for s in sets:
        s["graph"], s["stream"] = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(s["graph"]):
            s["out"] = s["run"]()
    for ln in (2100, 700, 0):
        for s in sets:
            s["len"].fill_(ln)
        torch.cuda.synchronize()
        for _ in range(4):
            for s in sets:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            assert torch.equal(s["out"], s["run"]()), ln
            if ln == 2100:
                assert torch.equal(s["out"], s["want"][0])
    assert L.kernel_error() == 0


@gpu
def test_direct_entry_and_general_path_agree(monkeypatch):
    """The C++ entry and the Python path behind it: the same bits, the same refusals."""
    c, pre = filled(163, 2, 2, 90, 64, "e4m3"), filled(167, 1, 2, 50, 64, "e4m3")
    q, pos, t = normal(173, 2, 3, 4, 64), int32(40, 7), tables(200, 64)
    wide = normal(179, 2, 3, 5, 64)[:, :, 1:, :]                 # heads contiguous, rows strided

    def run():
        out = torch.zeros_like(q)
        c.append(q[:, :, :2], q[:, :, 2:], pos, rope=t)           # heads strided by the wider tensor's positions
        return [c.attend(q, pos), c.attend(q, pos, rope=t, rope_pos=int32(90, 57), prefix=pre, prefix_len=int32(50)),
                c.attend(wide, pos, out=out), out, c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), pos),
                c.attend(q, pos, scale=1), *c.read(pos, 5)]

    a = run()

    class Nothing:
        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(L, "direct", lambda: Nothing())
    b = run()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
