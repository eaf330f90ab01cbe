"""Key/value cache in 8 bits for the chunked continuation and for token-by-token decoding.

Keys and values are held as e4m3 codes with one power-of-two scale for each 64 tokens of a head: half of the
bf16 cache's memory and, where few rows attend, half of its traffic.  A floating-point code loses no precision
by a power-of-two scale, and decoding a code to 16 bits is exact within the type's range (in fp16 for scales of 2^-15
and above, where the block's largest value is above 0.0068; smaller ones fall into fp16's subnormals and are rounded).
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _dense

__all__ = ["KVCache8"]

BLOCK = _dense.CACHE_BLOCK

# Most rows (query heads of a key head x query tokens) that read the codes directly, 16 to a pass; above, the
# cache is unpacked to 16 bits once and the tile kernel runs.  On one B200, codes against unpacked: 1 x 8 heads x
# 4,096 tokens, 128 rows 29 and 46 us, 256 rows 48 and 45; 8 x 8 x 8,192, 128 rows 169 and 255, 256 rows 285 and 255.
FEW_ROWS = 128


class KVCache8:
    """Codes ``k_codes`` / ``v_codes`` [B, Hk, capacity, D] (e4m3), scales ``k_scale`` / ``v_scale``
    [B, Hk, capacity / 64] (fp32) and ``lengths`` [B] (int32: tokens held), all on one CUDA device.

    The lengths live on the device, so an append or a lookup can be captured into a CUDA graph and replayed.
    Calls on one cache are ordered by their stream, like any in-place update of a tensor."""

    def __init__(self, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
                 lengths: torch.Tensor):
        self._cache = _dense.ops().Cache(k_codes, k_scale, v_codes, v_scale, lengths)
        self.k_codes, self.k_scale, self.v_codes, self.v_scale, self.lengths = k_codes, k_scale, v_codes, v_scale, lengths

    @classmethod
    def allocate(cls, batch: int, heads: int, capacity: int, head_dim: int, device=None) -> "KVCache8":
        """An empty cache; the capacity is rounded up to whole blocks of 64 tokens."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        cap = -(-int(capacity) // BLOCK) * BLOCK
        codes = [torch.zeros((batch, heads, cap, head_dim), device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
                 for _ in range(2)]
        scale = [torch.zeros((batch, heads, cap // BLOCK), device=device, dtype=torch.float32) for _ in range(2)]
        return cls(codes[0], scale[0], codes[1], scale[1], torch.zeros((batch,), device=device, dtype=torch.int32))

    @classmethod
    def from_kv(cls, k: torch.Tensor, v: torch.Tensor, capacity: Optional[int] = None) -> "KVCache8":
        """A cache that holds k and v [B, Hk, S, D]."""
        B, Hk, S, D = k.shape
        cache = cls.allocate(B, Hk, max(S, 1) if capacity is None else capacity, D, k.device)
        cache.append(k, v)
        return cache

    @property
    def capacity(self) -> int:
        return int(self.k_codes.shape[2])

    def expand(self, batch: int) -> "KVCache8":
        """This cache, or a one-sequence cache repeated for a batch (a copy)."""
        B = self.k_codes.shape[0]
        if batch == B:
            return self
        if B != 1:
            raise ValueError(f"a cache of {B} sequences for a batch of {batch}")
        rep = lambda t: t.view(torch.uint8).repeat(batch, 1, 1, 1).view(t.dtype)  # noqa: E731
        return KVCache8(rep(self.k_codes), self.k_scale.repeat(batch, 1, 1), rep(self.v_codes),
                        self.v_scale.repeat(batch, 1, 1), self.lengths.repeat(batch))

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
        """Adds n tokens to every sequence (``counts`` int32 [B]: only the first counts[b] of them).

        A block whose largest value grows takes a larger scale, and its codes are rounded again at it.  Tokens that
        do not fit are dropped, and ``_native.device_error()`` then reports it; more tokens than the whole capacity
        are refused here.  Infinities are held as the block's largest code, NaN as NaN; neither sets a scale, but that a
        block with either has the smallest one (2^-126) at least.  What is held is constant to gradients."""
        self._cache.append(k, v, counts)

    def truncate(self, lengths: Union[int, torch.Tensor]) -> None:
        """Sets the lengths: a rejected draft, or the conditioning tokens before the next chunk.  Blocks keep their
        scales; a block that ends up without tokens takes a new one at the next append."""
        if isinstance(lengths, torch.Tensor):
            if lengths.shape != self.lengths.shape:
                raise ValueError(f"lengths must be {list(self.lengths.shape)}")
            self.lengths.copy_(lengths)
        else:
            if not 0 <= int(lengths) <= self.capacity:
                raise ValueError(f"length {lengths} is outside [0, {self.capacity}]")
            self.lengths.fill_(int(lengths))

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [B, Hk, capacity, D]: the held tokens, zeros behind them."""
        return self._cache.unpack(dtype)

    def attend(self, q: torch.Tensor, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None, *,
               causal: bool = False, sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [B, H, Sq, D] over the held tokens and, behind them, fresh keys and values k, v
        [B, Hk, n, D] that are not cached (the frames being denoised); H is a multiple of Hk.

        ``causal``: the last query sees every key (held, then fresh), the one before it one less, and so on.
        sm_scale defaults to 1 / sqrt(D).  Sequences without a key give zeros.  Few rows read the codes as they are;
        many rows, or fresh keys, unpack the cache into 16-bit scratch first.  What lies behind the held tokens does not
        matter; a value of NaN that is held, or infinite or NaN among the fresh ones, reaches the rows that see it and,
        with ``causal``, can reach earlier rows of the same pass: 16 of them, or 128 where the cache is unpacked."""
        return self._cache.attend(q, k, v, causal, sm_scale, out, FEW_ROWS)
