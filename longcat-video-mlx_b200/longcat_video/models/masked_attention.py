"""Dense attention over key intervals: document, prefix, causal and padding masks, scores capped by a tanh.

The dense side of the attention hook on the engine's own kernels.  A mask is a key interval [lo, hi) for each
query row (:class:`AttentionMask`), which one build (a small launch) makes for as many calls as share it; no Sq x Sk
tensor exists.
``masked_attention`` is differentiable, once (``create_graph=True`` is refused, and so is forward mode); its gradients
are computed without atomics, so two runs give the same bits.
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

    def __init__(self, buffer: torch.Tensor, batch: int, table_at: int, Sq: int, Sk: int):
        # one device buffer: the intervals, and the table from `table_at` on
        self._buffer, self._table_at = buffer, table_at
        self.batch, self.Sq, self.Sk = batch, Sq, Sk

    @property
    def ranges(self) -> torch.Tensor:
        return self._buffer[:self.batch * self.Sq * 2].view(self.batch, self.Sq, 2)

    @property
    def table(self) -> torch.Tensor:
        """[batch, tiles of 128 rows, 4]: lowest lo and highest hi of the rows that see a key, highest lo and lowest hi of
        all rows."""
        return self._buffer[self._table_at:].view(self.batch, (self.Sq + 127) // 128, 4)

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
        many = isinstance(prefix, torch.Tensor)
        parts = _dense.ops().attention_ranges(
            None if device is None else torch.device(device), Sq, Sk, 1, None, causal, 0 if many or prefix is None else prefix,
            prefix if many else None, q_offsets, k_offsets, q_lengths, k_lengths, 0)
        return cls(*parts, Sq, Sk)

    @classmethod
    def from_ranges(cls, ranges: torch.Tensor, Sk: int) -> "AttentionMask":
        """From [batch or 1, Sq, 2] int32 intervals [lo, hi); they are clamped to [0, Sk]."""
        if ranges.dim() != 3 or ranges.shape[-1] != 2:
            raise ValueError("ranges must be [batch, Sq, 2]")
        batch, Sq = int(ranges.shape[0]), int(ranges.shape[1])
        parts = _dense.ops().attention_ranges(ranges.device, Sq, Sk, batch, ranges, False, 0, None, None, None, None, None, 0)
        return cls(*parts, Sq, int(Sk))

    def _args(self):
        return self._buffer, self.batch, self._table_at, self.Sq, self.Sk


_NO_MASK = (None, 1, 0, 0, 0)


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[AttentionMask] = None, *,
                     sm_scale: Optional[float] = None, softcap: float = 0.0, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None):
    """softmax(z) v with z = sm_scale q k^T, or softcap * tanh(z / softcap), over the keys that ``mask`` shows.

    q [B, H, Sq, D], k and v [B, Hk, Sk, D] with H a multiple of Hk (query head h reads key head h // (H // Hk));
    bf16 or fp16 CUDA tensors, D a multiple of 8 up to 128, any strides (views that the kernels cannot read in place
    are copied once).  sm_scale defaults to 1 / sqrt(D).  Rows that see no key give zeros, and -inf in the
    log-sum-exp [B, H, Sq] (fp32, natural) that ``return_lse`` adds; it carries no gradient.  ``out``: a
    preallocated [B, H, Sq, D] result, which may be q; over another input, or itself, it is refused (so with gradients).

    What masked places hold does not matter, with limits for values that are infinite or NaN: in a row of v (for
    gradients, of k too) between the first and the last key that some row of the same 128 queries sees, they can reach all
    of those queries; in a row of q or of the output's gradient that sees a key, they can reach the gradients of all keys
    in the runs of 128 that some row of the same 128 queries sees.  Rows that see nothing may hold anything."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale
    args = _NO_MASK if mask is None else mask._args()
    o, lse = _dense.ops().masked_attention(q, k, v, *args, scale, softcap, out, return_lse)
    return (o, lse) if return_lse else o
