"""Sampling from a model's logits, and verification of drafted tokens, from
given random numbers.

The reference decodes greedily (code/cdq_lrr_qwen05.py:335-340). Speculative
sampling keeps the target model's distribution exactly: draft token x_i of the
draft's distribution q_i is kept with probability min(1, p_i(x_i) / q_i(x_i)),
and the first one that is not is replaced by a draw from max(p_i - q_i, 0),
normalised. The random numbers are arguments, so a result can be repeated.
"""
from __future__ import annotations

import torch

from . import _lib as L

_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


def _logits(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: must be bf16 or float32")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: expected a CUDA tensor (the sampling kernels have no CPU path)")
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _floats(x: torch.Tensor, shape: tuple, dev, what: str) -> int:
    if x.dtype is not torch.float32 or x.shape != shape or x.device != dev or not x.is_contiguous():
        raise ValueError(f"{what}: must be contiguous float32 {list(shape)} on the logits' device")
    return x.data_ptr()


def _temperature(t: float) -> float:
    t = float(t)
    if not 1e-30 <= t <= 1e30:
        raise ValueError(f"temperature must be in [1e-30, 1e30], got {t} (greedy decoding takes the argmax)")
    return t


def _call(target, draft, tokens_in, u_accept, u_sample, batch, k, vocab, temperature, out, n_acc) -> None:
    dev = target.device
    ds, dr = (0, 0) if draft is None else draft.stride()[:2]
    ws, need = None, 0
    if k:
        need = batch * (2 * k + 1 if draft is not None else k + 1) * L.VERIFY_ROW_BYTES
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with L.on_device(dev):
        L.check(L.lib().cdq_verify_drafts(
            target.data_ptr(), target.stride(0), target.stride(1) if k else 0,
            None if draft is None else draft.data_ptr(), ds, dr, _DTYPES[target.dtype], tokens_in, u_accept, u_sample,
            batch, k, vocab, temperature, out.data_ptr(), None if n_acc is None else n_acc.data_ptr(),
            ws.data_ptr() if k else None, need, L.raw_stream(dev)), "cdq_verify_drafts")


def verify_drafts(target_logits: torch.Tensor, draft_tokens: torch.Tensor, draft_logits: torch.Tensor | None,
                  u_accept: torch.Tensor, u_sample: torch.Tensor,
                  temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Checks k drafted tokens of every sequence against the target.

    target_logits [batch, k + 1, vocab] and draft_logits [batch, k, vocab]
    (None: drafts chosen greedily, a distribution with one token), both bf16
    or both float32; draft_tokens int64 [batch, k], a negative token ending a
    sequence's drafts; u_accept [batch, k] and u_sample [batch] float32 in
    [0, 1); temperature in [1e-30, 1e30]. Returns tokens int64 [batch, k + 1] (the kept drafts, the token
    drawn after them, then -1) and the number of kept drafts, int32 [batch].
    A row without a distribution (a NaN, +inf or nothing but -inf) ends its
    sequence with the token -1."""
    r = L.direct().verify_drafts(target_logits, draft_tokens, draft_logits, u_accept, u_sample, temperature)
    if r is not None:
        return r if isinstance(r, tuple) else L.check(r, "cdq_verify_drafts")
    if target_logits.dim() != 3:
        raise ValueError(f"verify_drafts: target logits must be [batch, k + 1, vocab], got {list(target_logits.shape)}")
    batch, rows, vocab = target_logits.shape
    k, dev = rows - 1, target_logits.device
    if batch < 1 or rows < 1 or vocab < 1:
        raise ValueError("verify_drafts: empty target logits")
    target = _logits(target_logits, "verify_drafts: target logits")
    if tuple(draft_tokens.shape) != (batch, k) or draft_tokens.dtype != torch.int64 or draft_tokens.device != dev or \
            not draft_tokens.is_contiguous():
        raise ValueError(f"verify_drafts: drafts must be contiguous int64 [{batch}, {k}] on the logits' device")
    draft = None
    if draft_logits is not None:
        if tuple(draft_logits.shape) != (batch, k, vocab) or draft_logits.dtype != target.dtype or \
                draft_logits.device != dev:
            raise ValueError(f"verify_drafts: draft logits must be [{batch}, {k}, {vocab}] of the target logits' type "
                             "on their device")
        draft = _logits(draft_logits, "verify_drafts: draft logits") if k else None
    ua, us = _floats(u_accept, (batch, k), dev, "u_accept"), _floats(u_sample, (batch,), dev, "u_sample")
    t = _temperature(temperature)
    tokens = torch.empty(batch, k + 1, dtype=torch.int64, device=dev)
    n_acc = torch.empty(batch, dtype=torch.int32, device=dev)
    _call(target, draft, draft_tokens.data_ptr(), ua, us, batch, k, vocab, t, tokens, n_acc)
    return tokens, n_acc


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: float = 1.0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of softmax(logits / temperature) a sequence: logits [batch,
    vocab] bf16 or float32, u float32 [batch] in [0, 1); the smallest token
    whose cumulative probability exceeds u. Returns int64 [batch] (in `out` if
    given); -1 for a row without a distribution."""
    r = L.direct().sample_tokens(logits, u, temperature, out)
    if r is not None:
        return r if isinstance(r, torch.Tensor) else L.check(r, "cdq_verify_drafts")
    if logits.dim() != 2:
        raise ValueError(f"sample_tokens: logits must be [batch, vocab], got {list(logits.shape)}")
    batch, vocab = logits.shape
    if batch < 1 or vocab < 1:
        raise ValueError("sample_tokens: empty logits")
    x = _logits(logits, "sample_tokens: logits")
    us, t = _floats(u, (batch,), x.device, "u"), _temperature(temperature)
    if out is None:
        out = torch.empty(batch, dtype=torch.int64, device=x.device)
    elif tuple(out.shape) != (batch,) or out.dtype != torch.int64 or out.device != x.device or not out.is_contiguous():
        raise ValueError(f"sample_tokens: out must be contiguous int64 [{batch}] on the logits' device")
    _call(x, None, None, None, us, batch, 0, vocab, t, out, None)
    return out
