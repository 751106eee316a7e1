"""Quantised key/value cache of a batch of sequences, and attention over it.

The reference keeps HF's bf16 cache (code/cdq_lrr_qwen05.py:335-340). Here the
keys and values of every (sequence, kv head, position) are rows of 8-bit
("e4m3", one bf16 scale a row) or 4-bit codes ("e2m1", one bf16 scale per 32
elements); the formats are those of include/cdq.h. Writing rotates and
quantises in one pass, attention reads the codes as they are and never
dequantises them to memory.

    cache = QuantKVCache(batch, kv_heads, max_len, head_dim, "e4m3")
    cache.append(k, v, pos, rope=(cos, sin))          # [batch, n, kv_heads, head_dim]
    out = cache.attend(q, pos, rope=(cos, sin))       # [batch, n, heads, head_dim]

Positions are device tensors, so a captured step replays with new ones. The
host cannot see them, so a position that does not fit is not an error of the
call: `append` does not write it, `read` gives zeros for it and `attend` NaN.
A sequence with a negative position is idle: nothing is written and its
outputs are zeros.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

GROUP = 32  # e2m1 elements per scale
_DTYPES = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}


def _rows(x: torch.Tensor) -> tuple:
    """x [batch, n, heads, head_dim] as (tensor, pointer, sequence stride, position stride) with contiguous heads
    and 16-byte rows (copied if it has none)."""
    sb, sn, sh, sd = x.stride()
    p = x.data_ptr()
    if sd != 1 or sh != x.shape[3] or (sb | sn | p) % 8 or p % 16 or sb < 0 or sn < 0:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        sb, sn, _, _ = x.stride()
        p = x.data_ptr()
    return x, p, sb, sn


def _overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether the address ranges of x and y meet."""
    def ends(t):
        p = t.data_ptr()
        return p, p + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    (a, b), (c, d) = ends(x), ends(y)
    return a < d and c < b


class QuantKVCache:
    """Codes k, v [batch, kv_heads, max_len, head_dim] (e2m1: head_dim / 2
    bytes) and bf16 scales [batch, kv_heads, max_len] (e2m1: [..., head_dim /
    32]), zero-filled. The buffers belong to the cache; calls on one cache must
    be ordered by their stream like any use of a tensor, and need no
    workspace of the caller's: `attend` takes its scratch from torch's
    allocator, so calls on several streams and captured graphs share none."""

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, fmt: str = "e4m3", device="cuda"):
        if fmt not in L.KV_FORMATS:
            raise ValueError(f"QuantKVCache: unknown format {fmt!r} (e4m3 or e2m1)")
        if head_dim not in (64, 128):
            raise ValueError(f"QuantKVCache: head_dim must be 64 or 128, got {head_dim}")
        if batch < 1 or kv_heads < 1 or max_len < 1:
            raise ValueError("QuantKVCache: batch, kv_heads and max_len must be positive")
        lead, dev = (batch, kv_heads, max_len), torch.device(device)
        width = head_dim if fmt == "e4m3" else head_dim // 2
        groups = lead if fmt == "e4m3" else (*lead, head_dim // GROUP)
        # (a zero byte is the code 0 of both formats)
        codes = [torch.zeros(*lead, width, dtype=torch.uint8, device=dev).view(_DTYPES[fmt]) for _ in range(2)]
        scales = [torch.zeros(groups, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        self._bind(codes[0], codes[1], scales[0], scales[1])

    @classmethod
    def from_buffers(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor) -> "QuantKVCache":
        """A cache over existing buffers of the layout above (float8_e4m3fn
        codes: e4m3, uint8: e2m1), which it uses in place. The codes are
        trusted to be finite, as those that `append` writes are."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        fmt = {d: f for f, d in _DTYPES.items()}.get(k.dtype)
        if fmt is None or v.dtype != k.dtype:
            raise TypeError("QuantKVCache: codes must be float8_e4m3fn (e4m3) or uint8 (e2m1)")
        if k_scale.dtype != torch.bfloat16 or v_scale.dtype != torch.bfloat16:
            raise TypeError("QuantKVCache: scales must be bf16")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("QuantKVCache: codes must be [batch, kv_heads, max_len, row bytes]")
        lead = tuple(k.shape[:3])
        hd = k.shape[3] * (1 if fmt == "e4m3" else 2)
        want = lead if fmt == "e4m3" else (*lead, hd // GROUP)
        if hd not in (64, 128):
            raise ValueError(f"QuantKVCache: head_dim must be 64 or 128, got {hd}")
        if tuple(k_scale.shape) != want or tuple(v_scale.shape) != want:
            raise ValueError(f"QuantKVCache: scales must be {list(want)}")
        parts = (k, v, k_scale, v_scale)
        if not all(t.is_contiguous() and t.device == k.device for t in parts):
            raise ValueError("QuantKVCache: buffers must be contiguous and on one device")
        if any(t.data_ptr() % a for t, a in zip(parts, (16, 16, 8, 8))):
            raise ValueError("QuantKVCache: buffers must be aligned (codes 16 bytes, scales 8)")
        self.k, self.v, self.k_scale, self.v_scale, self.fmt = k, v, k_scale, v_scale, fmt
        self.device = k.device
        self.batch, self.kv_heads, self.max_len = lead
        self.head_dim = hd
        s = L.cdq_kv_cache()
        s.k, s.v, s.k_scale, s.v_scale = (t.data_ptr() for t in parts)
        s.batch, s.kv_heads, s.max_len, s.head_dim = *lead, hd
        s.format = L.KV_FORMATS[fmt]
        self._struct = s
        self._ref = C.byref(s)
        self._address = C.addressof(s)
        self._index = k.device.index if k.device.type == "cuda" else -1
        self._ws_bytes: dict = {}

    def nbytes(self) -> int:
        """Bytes of the codes and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    # ---- argument checks ----
    def _check_rows(self, x: torch.Tensor, heads: int | None, what: str) -> torch.Size:
        shape = x.shape
        if x.dtype is not torch.bfloat16:
            raise TypeError(f"{what}: must be bf16")
        if x.device != self.device:
            if not x.is_cuda:
                raise RuntimeError(f"{what}: expected a CUDA tensor (the cache kernels have no CPU path)")
            raise ValueError(f"{what}: on another device than the cache")
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != self.head_dim or (heads and shape[2] != heads):
            raise ValueError(f"{what}: must be [{self.batch}, n, {heads or 'heads'}, {self.head_dim}], "
                             f"got {list(shape)}")
        return shape

    def _like(self, cache: "QuantKVCache") -> bool:
        """Whether this cache can be a prefix of `cache`."""
        return self.batch == 1 and self.kv_heads == cache.kv_heads and self.head_dim == cache.head_dim and \
            self.fmt == cache.fmt and self.device == cache.device

    def _check_cuda(self, what: str) -> None:
        if self.device.type != "cuda":
            raise RuntimeError(f"{what}: expected a CUDA cache (the cache kernels have no CPU path)")

    def _check_index(self, t: torch.Tensor, n: int, what: str) -> int:
        if t.dtype is not torch.int32 or t.device != self.device or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{what}: must be contiguous int32 [{n}] on the cache's device")
        return t.data_ptr()

    def _rope(self, rope, rope_pos) -> tuple:
        """(cos, sin, rows, row of the first new position) of the C calls."""
        if rope is None:
            if rope_pos is not None:
                raise ValueError("rope_pos without rotary tables")
            return None, None, 0, None
        cos, sin = rope
        shape = cos.shape
        pc, ps = cos.data_ptr(), sin.data_ptr()
        if len(shape) != 2 or shape[1] != self.head_dim or not shape[0] or sin.shape != shape:
            raise ValueError(f"rope: cos and sin tables must be [positions, {self.head_dim}] alike")
        if cos.dtype is not torch.bfloat16 or sin.dtype is not torch.bfloat16 or cos.device != self.device or \
                sin.device != self.device or (pc | ps) % 16 or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError("rope: tables must be contiguous bf16 on the cache's device, 16-byte aligned")
        return pc, ps, shape[0], None if rope_pos is None else self._check_index(rope_pos, self.batch, "rope_pos")

    # ---- operators ----
    def append(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, rope=None, rope_pos=None) -> None:
        """Quantises k, v bf16 [batch, n, kv_heads, head_dim] into positions
        pos[b] .. pos[b] + n - 1 (pos: device int32 [batch]). rope: bf16
        (cos, sin) tables [positions, head_dim], by which keys are rotated
        first; rope_pos: the table row of each sequence's first new position
        where that is not pos (a cache behind a shared prefix)."""
        st = L.direct().kv_append(self._address, self._index, k, v, pos, rope, rope_pos)
        if st is not None:
            return L.check(st, "cdq_kv_append")
        self._check_cuda("append")
        n = self._check_rows(k, self.kv_heads, "append: k")[1]
        if self._check_rows(v, self.kv_heads, "append: v")[1] != n:
            raise ValueError("append: k and v differ in shape")
        cos, sin, rows, rpos = self._rope(rope, rope_pos)
        pp = self._check_index(pos, self.batch, "append: pos")
        if n == 0:
            return
        k, kp, kb, kn = _rows(k)
        v, vp, vb, vn = _rows(v)
        with L.on_device(self.device):
            L.check(L.lib().cdq_kv_append(self._ref, kp, kb, kn, vp, vb, vn, pp, n, cos, sin, rows, rpos,
                                          L.raw_stream(self.device)), "cdq_kv_append")

    def read(self, pos: torch.Tensor | None, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of positions pos[b] .. pos[b] + n - 1 (pos None: from 0)
        as bf16 k, v [batch, n, kv_heads, head_dim]."""
        r = L.direct().kv_read(self._address, self._index, pos, n)
        if r is not None:
            return r if isinstance(r, tuple) else L.check(r, "cdq_kv_read")
        self._check_cuda("read")
        pp = None if pos is None else self._check_index(pos, self.batch, "read: pos")
        if n < 0:
            raise ValueError("read: n must not be negative")
        shape = (self.batch, n, self.kv_heads, self.head_dim)
        k, v = torch.empty((2, *shape), dtype=torch.bfloat16, device=self.device)
        if n:
            with L.on_device(self.device):
                L.check(L.lib().cdq_kv_read(self._ref, pp, n, k.data_ptr(), v.data_ptr(), L.raw_stream(self.device)),
                        "cdq_kv_read")
        return k, v

    def attend(self, q: torch.Tensor, pos: torch.Tensor, rope=None, rope_pos=None, scale: float | None = None,
               prefix: "QuantKVCache | None" = None, prefix_len: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Grouped-query attention of q bf16 [batch, n, heads, head_dim], the
        n <= 64 newest positions pos[b] .. pos[b] + n - 1 of every sequence
        (their keys and values appended already), over the cache: position p
        attends to 0 .. p. prefix: a cache of batch 1 whose positions 0 ..
        prefix_len[0] - 1 (device int32 [1]) every sequence attends to as
        well; it is read once for the whole batch. scale defaults to
        head_dim ** -0.5. Returns bf16 like q (contiguous), in `out` if given
        (16-byte aligned, not over q). Inference only: no gradients."""
        if prefix is None or prefix._like(self):
            r = L.direct().kv_attend(self._address, self._index, q, pos, rope, rope_pos, scale,
                                     None if prefix is None else prefix._address, prefix_len, out)
            if r is not None:
                return r if isinstance(r, torch.Tensor) else L.check(r, "cdq_kv_attend")
        self._check_cuda("attend")
        shape = self._check_rows(q, None, "attend: q")
        _, n, heads, _ = shape
        if not 1 <= n <= L.KV_MAX_NEW:
            raise ValueError(f"attend: 1 to {L.KV_MAX_NEW} new positions, got {n}")
        if heads < self.kv_heads or heads % self.kv_heads:
            raise ValueError(f"attend: {heads} heads over {self.kv_heads} kv heads")
        cos, sin, rows, rpos = self._rope(rope, rope_pos)
        pp = self._check_index(pos, self.batch, "attend: pos")
        pref = plen = None
        if prefix is not None:
            if not prefix._like(self):
                raise ValueError("attend: the prefix must be a cache of batch 1 with the same heads, format and device")
            if prefix_len is None:
                raise ValueError("attend: a prefix needs prefix_len")
            pref, plen = prefix._ref, self._check_index(prefix_len, 1, "attend: prefix_len")
        elif prefix_len is not None:
            raise ValueError("attend: prefix_len without a prefix")
        if out is None:
            out = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        elif out.shape != shape or out.dtype is not torch.bfloat16 or out.device != self.device or \
                not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("attend: out must be contiguous bf16 of q's shape on the cache's device, 16-byte aligned")
        elif _overlap(q, out):
            raise ValueError("attend: out overlaps q")
        q, qp, qb, qn = _rows(q)
        with L.on_device(self.device):
            key = (heads, n, prefix.max_len if prefix is not None else 0)
            need = self._ws_bytes.get(key)
            if need is None:
                b = C.c_int64()
                L.check(L.lib().cdq_kv_attend_workspace(self._ref, heads, n, pref, C.byref(b)),
                        "cdq_kv_attend_workspace")
                need = self._ws_bytes[key] = b.value
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            L.check(L.lib().cdq_kv_attend(self._ref, qp, qb, qn, heads, n, pp, cos, sin, rows, rpos,
                                          self.head_dim ** -0.5 if scale is None else float(scale), pref, plen,
                                          out.data_ptr(), ws.data_ptr() if need else None, need,
                                          L.raw_stream(self.device)), "cdq_kv_attend")
        return out
