"""The decode paths that use the quantised cache, sampling and draft
verification together: every step's attention and tokens against the 64-bit
forms of the operators on the step's own buffers."""
import pytest
import torch

from test_kvcache import attention, check, values
from test_sampling import drawn, softmax, verify

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def models():
    from cdq_lrr_b200 import decode
    from cdq_lrr_b200.quant import CAMKII_LATTICE_16
    a, b = decode.build_model(seed=0, layers=1), decode.build_model(seed=0, layers=1)
    decode.patch_cdq(a)
    decode.patch_cdq(b, lattice=CAMKII_LATTICE_16)
    return a, b


def _prompt(n, seed=1):
    return torch.randint(0, 151936, (1, n), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_step_with_a_quantised_cache(models, fmt):
    """Prefill, then greedy steps: the cache holds the model's rotated keys, the step's attention is the operator's."""
    from cdq_lrr_b200 import decode
    fd = decode.FusedDecoder(models[0], 60, kv_format=fmt)
    tok = fd.prefill(_prompt(37))
    assert int(tok) == int(fd.logits[0].argmax())
    for i in range(4):
        fd._step()
        torch.cuda.synchronize()
        q = fd.q.view(1, 1, fd.n_heads, fd.hd)
        want = attention(q, (37 + i,), fd.kv[0], (fd.cos, fd.sin), None, fd.hd ** -0.5)
        check(fd.att.view(1, 1, fd.n_heads, fd.hd), *want)
        assert int(fd.ids) == int(fd.logits[0].argmax()) and int(fd.pos) == 38 + i
    held = values(fd.kv[0])[0][0, 0].abs().sum(-1)
    assert bool((held[:41] > 0).all()) and not held[41:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_prefilled_cache_is_the_models(models, fmt):
    """The prompt's keys and values in the quantised cache are the bf16 cache's, within half a code step."""
    from cdq_lrr_b200 import decode
    from cdq_lrr_b200.quant import CAMKII_LATTICE_16
    a, b = decode.FusedDecoder(models[0], 40, kv_format=fmt), decode.FusedDecoder(models[0], 40)
    a.prefill(_prompt(30))
    b.prefill(_prompt(30))
    cl = b.cache.layers[0]
    for got, want, scale in ((values(a.kv[0])[0], cl.keys, a.kv[0].k_scale), (values(a.kv[0])[1], cl.values, a.kv[0].v_scale)):
        x, s = want[:, :, :30].cpu().double(), scale[:, :, :30].cpu().double()
        s = s[..., None] if fmt == "e4m3" else s.repeat_interleave(32, -1)
        # e4m3: half a step is 2^-4 of the value, 2^-10 of the scale below 2^-6; the largest may lose 2^-9 to the
        # scale's rounding. e2m1: steps of 0.5, 1 and 2: a quarter of the value, or of the scale below 1
        half = (x.abs() * 2.0 ** -4).clamp(min=s * 2.0 ** -10) if fmt == "e4m3" else (x.abs() / 4).clamp(min=s / 4)
        assert bool(((got[:, :, :30] - x).abs() <= half * (1 + 2.0 ** -7)).all())


@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_sampled_step(models, fmt):
    """A sampled step's token is the draw of its own logits; graph replays repeat eager steps."""
    from cdq_lrr_b200 import decode
    fd = decode.FusedDecoder(models[0], 40, kv_format=fmt, temperature=0.7)
    fd.prefill(_prompt(20))
    fd.uniforms[:5] = torch.tensor([0.1, 0.9, 0.5, 0.0, 0.99])
    for i in range(5):
        fd._step()
        torch.cuda.synchronize()
        p = softmax(fd.logits[0].cpu(), 0.7)
        assert int(fd.tokens[i]) == drawn(p, float(fd.uniforms[i]))
    eager = decode.fused_sample_decode(models[0], _prompt(20), 12, 0.7, seed=5, kv_format=fmt, use_graph=False)
    graph = decode.fused_sample_decode(models[0], _prompt(20), 12, 0.7, seed=5, kv_format=fmt)
    assert torch.equal(eager["tokens"], graph["tokens"])
    other = decode.fused_sample_decode(models[0], _prompt(20), 12, 0.7, seed=6, kv_format=fmt)
    assert not torch.equal(other["tokens"], graph["tokens"])


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_verify_pass_with_a_quantised_cache(models, fmt):
    from cdq_lrr_b200 import decode, sampling
    fd = decode.FusedDecoder(models[0], 60, kv_format=fmt)
    fd.prefill(_prompt(33))
    ver = decode.VerifyStep(fd, 4, keep_logits=True)
    ver.ids.copy_(_prompt(4, seed=9)[0])
    ver._run()
    torch.cuda.synchronize()
    want = attention(ver.q.view(1, 4, fd.n_heads, fd.hd), (33,), fd.kv[0], (fd.cos, fd.sin), None, fd.hd ** -0.5)
    check(ver.att.view(1, 4, fd.n_heads, fd.hd), *want)
    d = torch.tensor([[5, 1000, 150000]], device="cuda")
    ua, us = torch.tensor([[0.0, 0.5, 0.2]], device="cuda"), torch.tensor([0.4], device="cuda")
    got = sampling.verify_drafts(ver.logits[None], d, None, ua, us, 0.9)
    ref = verify(ver.logits[None].cpu(), d.cpu(), None, ua.cpu(), us.cpu(), 0.9)
    assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu(), ref[1])


@pytest.mark.parametrize("fmt", [None, "e4m3", "e2m1"])
def test_speculative_sampling_runs(models, fmt):
    from cdq_lrr_b200 import decode
    r = decode.speculative_sample_decode(models[0], models[1], _prompt(25), 30, k=3, temperature=0.9, kv_format=fmt)
    t = r["tokens"]
    assert t.shape == (1, 30) and bool(((t >= 0) & (t < 151936)).all())
    assert 1 <= r["tokens_per_verify"] <= 4
    again = decode.speculative_sample_decode(models[0], models[1], _prompt(25), 30, k=3, temperature=0.9, kv_format=fmt,
                                             use_graph=False)
    assert torch.equal(again["tokens"], t)
    # the same model drafting for itself: its distributions agree up to rounding, most drafts are kept
    own = decode.speculative_sample_decode(models[0], models[0], _prompt(25), 30, k=3, temperature=0.9, kv_format=fmt)
    assert own["tokens_per_verify"] > 2


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_samples_of_one_prompt(models, fmt):
    """n continuations: attention over the shared prompt and each one's own cache, tokens drawn from their logits."""
    from cdq_lrr_b200 import decode
    n, P = 5, 29
    fd = decode.FusedDecoder(models[0], 60, kv_format=fmt)
    fd.prefill(_prompt(P))
    step = decode.SamplesStep(fd, n, 16, 0.8)
    step.uniforms[:3] = torch.rand(3, n, generator=torch.Generator().manual_seed(2))
    step.begin(_prompt(n, seed=4)[0], P)
    for i in range(3):
        step._run()
        torch.cuda.synchronize()
        want = attention(step.q.view(n, 1, fd.n_heads, fd.hd), (i,) * n, step.own[0], (fd.cos, fd.sin), (P + i,) * n,
                         fd.hd ** -0.5, values(fd.kv[0]), P)
        check(step.att.view(n, 1, fd.n_heads, fd.hd), *want)
        for b in range(n):
            assert int(step.ids[b]) == drawn(softmax(step.logits[b].cpu(), 0.8), float(step.uniforms[i, b]))
    a = decode.parallel_sample_decode(models[0], _prompt(P), n, 12, 0.8, seed=3, kv_format=fmt, use_graph=False)
    b = decode.parallel_sample_decode(models[0], _prompt(P), n, 12, 0.8, seed=3, kv_format=fmt)
    assert torch.equal(a["tokens"], b["tokens"]) and a["tokens"].shape == (n, 12)


def test_refusals(models):
    from cdq_lrr_b200 import decode
    with pytest.raises(ValueError):
        decode.FusedDecoder(models[0], 20, persistent=True, kv_format="e4m3")
    with pytest.raises(ValueError):
        decode.FusedDecoder(models[0], 20, persistent=True, temperature=1.0)
    with pytest.raises(ValueError):
        decode.FusedDecoder(models[0], 20, kv_format="int4")
    with pytest.raises(ValueError):
        decode.SamplesStep(decode.FusedDecoder(models[0], 20), 2, 8, 1.0)
    fd = decode.FusedDecoder(models[0], 20, kv_format="e4m3")
    with pytest.raises(ValueError):
        decode.SamplesStep(fd, 9, 8, 1.0)
    with pytest.raises(ValueError):
        decode.speculative_sample_decode(models[0], models[1], _prompt(5), 4, k=8)
