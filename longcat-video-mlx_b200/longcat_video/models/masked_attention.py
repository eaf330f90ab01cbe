"""Dense attention over key intervals: document, prefix, causal and padding masks, scores capped by a tanh.

The dense side of the attention hook on the engine's own kernels.  A mask is a key interval [lo, hi) for each
query row (:class:`AttentionMask`), built once for a batch and used by every layer; no Sq x Sk tensor exists.
``masked_attention`` is differentiable; its gradients are computed without atomics, so two runs give the same
bits.
"""

from __future__ import annotations

import math
from typing import Optional, Union

import torch

from .. import _dense

__all__ = ["AttentionMask", "masked_attention"]


class AttentionMask:
    """Which keys each query row sees: ``ranges`` [batch or 1, Sq, 2] int32 and the kernels' tile ``table``.

    Build one with :meth:`build` or, from intervals of one's own, with :meth:`from_ranges`."""

    def __init__(self, buffer, ranges: int, table: int, batch: int, Sq: int, Sk: int):
        # one device buffer, the addresses of its two parts, and their sizes (see _dense.attention_ranges)
        self._buffer, self._ranges, self._table = buffer, ranges, table
        self.batch, self.Sq, self.Sk = batch, Sq, Sk

    @property
    def ranges(self) -> torch.Tensor:
        return self._buffer[:self.batch * self.Sq * 2].view(self.batch, self.Sq, 2)

    @property
    def table(self) -> torch.Tensor:
        """[batch, tiles of 128 rows, 4]: lowest lo and highest hi of the rows that see a key, highest lo and lowest hi of
        all rows."""
        tiles = (self.Sq + 127) // 128
        return self._buffer[self._buffer.numel() - self.batch * tiles * 4:].view(self.batch, tiles, 4)

    @classmethod
    def build(cls, Sq: int, Sk: int, *, causal: bool = False, prefix: Union[int, torch.Tensor, None] = None,
              q_offsets: Optional[torch.Tensor] = None, k_offsets: Optional[torch.Tensor] = None,
              q_lengths: Optional[torch.Tensor] = None, k_lengths: Optional[torch.Tensor] = None,
              device=None) -> "AttentionMask":
        """The batch's rows as documents (``q_offsets``, ``k_offsets``: int32 [n + 1], ascending, shared by the
        batch), as padded entries (``q_lengths``, ``k_lengths``: int32 [B], each optional) or as one document.

        With a document of qn queries and kn keys, query i stands at key place a = i + kn - qn and sees a + 1 keys
        (``causal``) or all of them.  With a ``prefix`` (one number, or int32 for each document or entry) the rows
        at a < prefix see exactly the first ``prefix`` keys: conditioning tokens that attend to themselves, or a
        prompt in both directions in front of a causal continuation.  Rows outside every document or behind their
        length see nothing and come out as zeros."""
        if Sq < 0 or Sk < 0:
            raise ValueError("lengths must be >= 0")
        given = [t for t in (q_offsets, k_offsets, q_lengths, k_lengths) if t is not None]
        given += [prefix] if isinstance(prefix, torch.Tensor) else []
        if device is None:
            device = given[0].device if given else torch.device("cuda", torch.cuda.current_device())
        if (q_offsets is None) != (k_offsets is None):
            raise ValueError("q_offsets and k_offsets come together")
        if q_offsets is not None and (q_lengths is not None or k_lengths is not None):
            raise ValueError("give documents or lengths, not both")
        batch, n = 1, None
        if q_offsets is not None:
            if q_offsets.dim() != 1 or q_offsets.shape != k_offsets.shape or q_offsets.numel() < 2:
                raise ValueError("q_offsets and k_offsets must be [documents + 1]")
            n = q_offsets.numel() - 1
        for t, name in ((q_lengths, "q_lengths"), (k_lengths, "k_lengths")):
            if t is not None:
                if t.dim() != 1 or (n is not None and t.numel() != n):
                    raise ValueError(f"{name} must be [B]")
                batch = n = t.numel()
        prefixes = None
        if isinstance(prefix, torch.Tensor):
            if n is None:
                batch = n = prefix.numel()
            prefixes, prefix = _dense._i32(prefix, "prefix", (n,)), 0
        prefix = 0 if prefix is None else int(prefix)
        if prefix < 0:
            raise ValueError("prefix must be >= 0")
        parts = _dense.attention_ranges(
            batch, Sq, Sk, device=device, causal=causal, prefix=prefix, prefixes=prefixes,
            q_offsets=_dense._i32(q_offsets, "q_offsets"), k_offsets=_dense._i32(k_offsets, "k_offsets"),
            q_lengths=_dense._i32(q_lengths, "q_lengths"), k_lengths=_dense._i32(k_lengths, "k_lengths"))
        return cls(*parts, batch, Sq, Sk)

    @classmethod
    def from_ranges(cls, ranges: torch.Tensor, Sk: int) -> "AttentionMask":
        """From [batch or 1, Sq, 2] int32 intervals [lo, hi); they are clamped to [0, Sk]."""
        if ranges.dim() != 3 or ranges.shape[-1] != 2:
            raise ValueError("ranges must be [batch, Sq, 2]")
        given = _dense._i32(ranges, "ranges")
        if given.data_ptr() % 8:
            given = given.clone()
        batch, Sq = int(given.shape[0]), int(given.shape[1])
        return cls(*_dense.attention_ranges(batch, Sq, Sk, device=given.device, given=given), batch, Sq, int(Sk))


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, sm_scale, softcap):
        rest = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        out, lse = _dense.masked_attention(q, k, v, *_mask_args(mask), sm_scale, softcap, want_lse=True, rest=rest)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.mask = mask
        ctx.rest = (sm_scale, softcap)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 6
        q, k, v, out, rest, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv = _dense.masked_attention_backward(q, k, v, out, rest, lse, grad.to(q.dtype), *_mask_args(ctx.mask),
                                                      *ctx.rest, need[0], need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None


def _mask_args(mask):
    return (mask._ranges, mask._table, mask.batch) if mask is not None else (None, None, 1)


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[AttentionMask] = None, *,
                     sm_scale: Optional[float] = None, softcap: float = 0.0, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None):
    """softmax(z) v with z = sm_scale q k^T, or softcap * tanh(z / softcap), over the keys that ``mask`` shows.

    q [B, H, Sq, D], k and v [B, Hk, Sk, D] with H a multiple of Hk (query head h reads key head h // (H // Hk));
    bf16 or fp16 CUDA tensors, D a multiple of 8 up to 128, any strides (views that the kernels cannot read in place
    are copied once).  sm_scale defaults to 1 / sqrt(D).  Rows that see no key give zeros, and -inf in the
    log-sum-exp [B, H, Sq] (fp32, natural) that ``return_lse`` adds; it carries no gradient.  ``out``: a
    preallocated [B, H, Sq, D] result (not with gradients)."""
    _dense.check_qkv(q, k, v)
    scale = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else float(sm_scale)
    softcap = float(softcap)
    _dense.check_scale(scale, softcap)
    if mask is not None:
        if mask.Sq != q.shape[2] or mask.Sk != k.shape[2]:
            raise ValueError(f"the mask is for {mask.Sq} queries and {mask.Sk} keys, got {q.shape[2]} and {k.shape[2]}")
        if mask.batch != 1 and mask.batch != q.shape[0]:
            raise ValueError(f"the mask has {mask.batch} batch entries, q has {q.shape[0]}")
        _dense._same_place(q, mask._buffer)
    if out is not None:
        _dense._same_place(q, out)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out must have q's shape and dtype")
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if grad:
        if out is not None:
            raise ValueError("out= is for calls without gradients")
        o, lse = _MaskedAttention.apply(q, k, v, mask, scale, softcap)
        return (o, lse) if return_lse else o
    o, lse = _dense.masked_attention(q, k, v, *_mask_args(mask), scale, softcap, out=out, want_lse=return_lse)
    return (o, lse) if return_lse else o
