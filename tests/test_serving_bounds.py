"""What the decode paths that sample do at and past their capacity, on the
CPU: the steps run on stand-ins for the model and the kernels."""
from types import SimpleNamespace

import pytest
import torch

from cdq_lrr_b200 import decode, sampling


@pytest.fixture
def draws(monkeypatch):
    """The random numbers that the steps hand to the sampler."""
    seen = []

    def sample(logits, u, temperature, out):
        seen.append(u.clone())

    monkeypatch.setattr(sampling, "sample_tokens", sample)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: SimpleNamespace(cuda_stream=0))
    return seen


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_sampled_step_past_its_capacity(draws):
    """A step reads the random number of its count, and one past max_len the last (never out of range)."""
    t, cap = torch.zeros(1), 5
    fd = SimpleNamespace(persistent=False, layers=[], dev="cpu", h=t, dn=t, norm_w=t, eps=0.0, xn=t, H=1, lm_w=t, vocab=1,
                         logits=t, best=t, next=t, ids=t, tokens=t, pos=t, max_len=cap, temperature=1.0,
                         uniforms=torch.arange(cap) / 8, uniform=torch.zeros(1), count=_i32(0), row=_i32(0),
                         _call=lambda *a: None)
    for count in (0, 3, 4, 5, 6, 4000, 2 ** 31 - 1):
        fd.count.fill_(count)
        decode.FusedDecoder._step(fd)
        assert int(fd.count) == count
    assert torch.cat(draws).tolist() == [0.0, 0.375, 0.5, 0.5, 0.5, 0.5, 0.5]


def test_samples_step_past_its_capacity(draws):
    n, cap = 3, 4
    u = torch.arange(cap * n).view(cap, n) / 16
    st = SimpleNamespace(logits=torch.zeros(n, 8), temperature=1.0, uniforms=u, uniform=torch.zeros(1, n), count=_i32(0),
                         row=_i32(0), next=torch.zeros(n), ids=torch.zeros(n), pos=_i32(*[0] * n),
                         rope_pos=_i32(*[7] * n))
    for _ in range(cap + 3):
        decode.SamplesStep._finish(st)
    assert torch.equal(torch.stack(draws), torch.cat([u, u[-1:].expand(3, n)]))
    assert st.pos.tolist() == [cap + 3] * n and int(st.count) == cap + 3


class _Model:
    """Stands in for a model that must not be run."""

    def __call__(self, **kw):
        raise AssertionError("the prompt was run")


@pytest.mark.parametrize("kv", [None, "e4m3"])
@pytest.mark.parametrize("n", [0, 9, 4000])
def test_prompts_that_do_not_fit(kv, n):
    """A prompt longer than the cache would be written past its end (bf16) or cut off without a word (quantised)."""
    fd = SimpleNamespace(max_len=8, dev="cpu", kv_format=kv, cache=None if kv else object(),
                         model=_Model())
    fd.model.config = None
    with pytest.raises(ValueError, match="1 to 8 tokens"):
        decode.FusedDecoder.prefill(fd, torch.zeros(1, n, dtype=torch.long))


@pytest.mark.parametrize("prefix", [-1, 9])
def test_prefixes_that_do_not_fit(prefix):
    st = SimpleNamespace(fd=SimpleNamespace(max_len=8), ids=torch.zeros(2, dtype=torch.long), pos=_i32(0, 0),
                         rope_pos=_i32(0, 0), prefix_len=_i32(0), count=_i32(0))
    with pytest.raises(ValueError, match="prefix"):
        decode.SamplesStep.begin(st, torch.zeros(2, dtype=torch.long), prefix)
    decode.SamplesStep.begin(st, torch.ones(2, dtype=torch.long), 8)
    assert int(st.prefix_len) == 8 and st.rope_pos.tolist() == [8, 8]


@pytest.mark.parametrize("new", [0, -3])
def test_no_new_tokens(new):
    """Refused before a model is looked at."""
    p = torch.zeros(1, 4, dtype=torch.long)
    for call in (lambda: decode.fused_sample_decode(None, p, new), lambda: decode.parallel_sample_decode(None, p, 2, new),
                 lambda: decode.speculative_sample_decode(None, None, p, new)):
        with pytest.raises(ValueError, match="new_tokens"):
            call()
