"""Bindings of the C ABI's dense side (include/bsa_b200.h): q/k norm with rotary positions, attention over key
intervals, and the 8-bit key/value cache.  Argument checks, allocation of outputs and scratch, and the
launch on the tensors' device and its current stream; the public functions are in ``models``."""

from __future__ import annotations

import contextlib
from typing import Optional, Sequence, Tuple

import torch

from . import _native

CACHE_BLOCK = 64  # tokens of a head that share a scale


def _on(t: torch.Tensor):
    """The tensor's device as the current one for a launch."""
    if torch.cuda.current_device() == t.device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _same_place(*tensors: Optional[torch.Tensor]) -> None:
    given = [t for t in tensors if t is not None]
    _native._require_cuda(*given)
    if any(t.device != given[0].device for t in given):
        raise ValueError("all tensors must be on one device")


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _readable(t: torch.Tensor) -> torch.Tensor:
    """A view the kernels read in place, else a contiguous copy.  In place: d contiguous, base and strides in
    multiples of 16 bytes; any order and gaps of batch, heads and tokens otherwise."""
    if t.stride(-1) != 1 or _native._misaligned(t) or any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _i32(t: Optional[torch.Tensor], name: str, shape: Optional[Tuple[int, ...]] = None) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t.contiguous()


# ------------------------------------------------------------------------------- q/k norm + rotary positions
def _rope_args(rope, start: int):
    if rope is None:
        return (None, 0, 0, 0, 0, 0, 0, 0)
    tables, dims, grid = rope.native_args() if hasattr(rope, "native_args") else rope
    if tables.dtype != torch.float32 or not tables.is_contiguous():
        raise ValueError("rope tables must be contiguous fp32")
    if tables.numel() != sum(int(n) * int(d) for n, d in zip(grid, dims)):
        raise ValueError(f"rope tables of {tables.numel()} values do not match grid {tuple(grid)} and dims {tuple(dims)}")
    return (tables.data_ptr(), *(int(d) for d in dims), *(int(g) for g in grid), int(start))


def _norm_rope_check(xs: Sequence[torch.Tensor], ws, rope):
    tables = (rope.native_args() if hasattr(rope, "native_args") else rope)[0] if rope is not None else None
    _same_place(*xs, *ws, tables)
    x = xs[0]
    for t in xs:
        if t.dim() != 4:
            raise ValueError("expected tensors of shape [B, H, S, D]")
        if t.dtype != x.dtype or t.shape[0] != x.shape[0] or t.shape[2:] != x.shape[2:]:
            raise ValueError("q and k must share dtype, batch, length and head_dim")
    _native._dtype_code(x)
    for w in ws:
        if w is not None and tuple(w.shape) != (x.shape[-1],):
            raise ValueError(f"norm weight must be [{x.shape[-1]}]")


def _weights(ws, x: torch.Tensor):
    """Contiguous weights of one type: fp32 or the input's are read as they are, others as fp32."""
    kinds = {w.dtype for w in ws if w is not None}
    if len(kinds) == 1 and kinds <= {torch.float32, x.dtype}:
        kind = kinds.pop()
        return [w.contiguous() if w is not None else None for w in ws], _native.DTYPE_CODES[kind]
    return [w.float().contiguous() if w is not None else None for w in ws], 0


def norm_rope(xs, ws, eps: float, rope, start: int):
    _norm_rope_check(xs, ws, rope)
    ra = _rope_args(rope, start)
    x = xs[0]
    B, _, S, D = x.shape
    ys = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in xs]
    if any(t.numel() == 0 for t in xs):
        return ys
    xs = [_readable(t) for t in xs]
    ws, wcode = _weights(ws, x)
    sides = []
    for t, w, y in zip(xs, ws, ys):
        sides += [t.data_ptr(), _native._strides(t), t.shape[1], _ptr(w), y.data_ptr()]
    if len(xs) == 1:
        sides += [None, None, 0, None, None]
    with _on(x):
        rc = _native.lib().bsa_norm_rope(*sides, _native._dtype_code(x), wcode, B, S, D, float(eps), *ra,
                                         _native._stream(x))
    _native._check(rc, "bsa_norm_rope")
    return ys


def norm_rope_backward(xs, gs, ws, eps: float, rope, start: int, want_dw):
    x = xs[0]
    B, _, S, D = x.shape
    dxs = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in xs]
    dws = [torch.zeros((D,), device=x.device, dtype=torch.float32) if want else None for want in want_dw]
    if any(t.numel() == 0 for t in xs):
        return dxs, dws
    xs, gs = [_readable(t) for t in xs], [_readable(g) for g in gs]
    ws, wcode = _weights(ws, x)
    sides = []
    for t, g, w, dx, dw in zip(xs, gs, ws, dxs, dws):
        sides += [t.data_ptr(), _native._strides(t), g.data_ptr(), _native._strides(g), t.shape[1], _ptr(w),
                  dx.data_ptr(), _ptr(dw)]
    if len(xs) == 1:
        sides += [None, None, None, None, 0, None, None, None]
    with _on(x):
        scratch = None
        if any(want_dw):
            n = int(_native.lib().bsa_norm_rope_backward_scratch_bytes(D))
            scratch = torch.empty((n,), device=x.device, dtype=torch.uint8)
        rc = _native.lib().bsa_norm_rope_backward(*sides, _native._dtype_code(x), wcode, B, S, D, float(eps),
                                                  *_rope_args(rope, start), _ptr(scratch), _native._stream(x))
    _native._check(rc, "bsa_norm_rope_backward")
    return dxs, dws


# ------------------------------------------------------------------------------------------- key intervals
def attention_ranges(batch: int, Sq: int, Sk: int, *, device, given=None, causal=False, prefix=0, prefixes=None,
                     q_offsets=None, k_offsets=None, q_lengths=None, k_lengths=None, k_add: int = 0):
    ranges = torch.empty((batch, Sq, 2), device=device, dtype=torch.int32)
    table = torch.empty((batch, (Sq + 127) // 128, 4), device=device, dtype=torch.int32)
    _same_place(ranges, given, prefixes, q_offsets, k_offsets, q_lengths, k_lengths)
    if Sq == 0 or batch == 0:
        return ranges, table
    with _on(ranges):
        rc = _native.lib().bsa_attention_ranges(
            ranges.data_ptr(), table.data_ptr(), batch, Sq, Sk, _ptr(given), int(bool(causal)), int(prefix),
            _ptr(prefixes), _ptr(q_offsets), _ptr(k_offsets), q_offsets.numel() - 1 if q_offsets is not None else 0,
            _ptr(q_lengths), _ptr(k_lengths), int(k_add), _native._stream(ranges))
    _native._check(rc, "bsa_attention_ranges")
    return ranges, table


# ------------------------------------------------------------------------------------------ dense attention
def check_qkv(q, k, v, names=("q", "k", "v")) -> None:
    _same_place(q, k, v)
    for t, n in zip((q, k, v), names):
        if t.dim() != 4:
            raise ValueError(f"{n} must be [B, H, S, D]")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError("q, k, v must share one dtype")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported dtype {q.dtype} (bf16 or fp16)")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("q and k must share batch and head_dim")
    D = q.shape[3]
    if D % 8 or not 0 < D <= 128:
        raise ValueError(f"head_dim D={D} must be a multiple of 8 and <= 128")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads are no multiple of {k.shape[1]} key heads")


def check_scale(sm_scale: float, softcap: float = 0.0) -> None:
    if not 0.0 < sm_scale < float("inf"):
        raise ValueError("sm_scale must be positive and finite")
    if not 0.0 <= softcap < float("inf"):
        raise ValueError("softcap must be finite and >= 0")


def masked_attention(q, k, v, ranges, table, sm_scale: float, softcap: float, out=None, want_lse: bool = False,
                     rest: Optional[torch.Tensor] = None):
    """(out, lse or None).  ranges / table: of attention_ranges, or None for every key.  ``rest`` (contiguous, like
    out) receives what out's rounding left over."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    lse = torch.empty((B, H, Sq), device=q.device, dtype=torch.float32) if want_lse else None
    target = out
    if out is None or _native._misaligned(out) or out.stride(-1) != 1:
        target = torch.empty((B, H, Sq, D), device=q.device, dtype=q.dtype)
    if B and H and Sq and Sk:
        q, k, v = _readable(q), _readable(k), _readable(v)
        with _on(q):
            n = int(_native.lib().bsa_masked_attention_scratch_bytes(B, H, Sq, Sk, D))
            scratch = torch.empty((n,), device=q.device, dtype=torch.uint8) if n else None
            rc = _native.lib().bsa_masked_attention(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _native._dtype_code(q), B, H, Hk, Sq, Sk, D,
                _native._strides(q), _native._strides(k), _native._strides(v), _ptr(ranges), _ptr(table),
                ranges.shape[0] if ranges is not None else 1, float(sm_scale), float(softcap), target.data_ptr(),
                _native._strides(target), _ptr(rest), _ptr(lse), _ptr(scratch), _native._stream(q))
        _native._check(rc, "bsa_masked_attention")
    else:  # no rows, or no keys: zeros
        target.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
    if out is not None and target is not out:
        out.copy_(target)
        target = out
    return target, lse


def masked_attention_backward(q, k, v, out, rest, lse, grad, ranges, table, sm_scale: float, softcap: float, want_q: bool,
                              want_kv: bool):
    """(dq, dk, dv), contiguous; None where not wanted."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    empty = not (B and H and Sq and Sk)
    new = torch.zeros if empty else torch.empty
    dq = new((B, H, Sq, D), device=q.device, dtype=q.dtype) if want_q else None
    dk, dv = (new((B, Hk, Sk, D), device=q.device, dtype=q.dtype) if want_kv else None for _ in range(2))
    if empty:
        return dq, dk, dv
    q, k, v, out, grad = (_readable(t) for t in (q, k, v, out, grad))
    bm = ranges.shape[0] if ranges is not None else 0
    with _on(q):
        n = int(_native.lib().bsa_masked_attention_backward_scratch_bytes(B, H, Sq, bm))
        scratch = torch.empty((n,), device=q.device, dtype=torch.uint8)
        rc = _native.lib().bsa_masked_attention_backward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rest.data_ptr(), grad.data_ptr(), lse.data_ptr(),
            _native._dtype_code(q), B, H, Hk, Sq, Sk, D, *(_native._strides(t) for t in (q, k, v, out, grad)),
            _ptr(ranges), _ptr(table), max(bm, 1), float(sm_scale), float(softcap), _ptr(dq), _ptr(dk), _ptr(dv),
            scratch.data_ptr(), _native._stream(q))
    _native._check(rc, "bsa_masked_attention_backward")
    return dq, dk, dv


# ---------------------------------------------------------------------------------------------- 8-bit cache
def _cache_args(c):
    B, Hk, cap, D = c.k_codes.shape
    return (c.k_codes.data_ptr(), c.k_scale.data_ptr(), c.v_codes.data_ptr(), c.v_scale.data_ptr(),
            c.lengths.data_ptr(), B, Hk, cap, D)


def cache_append(c, k, v, counts) -> None:
    k, v = _readable(k), _readable(v)
    with _on(k):
        rc = _native.lib().bsa_kv8_append(*_cache_args(c), k.data_ptr(), v.data_ptr(), _native._dtype_code(k),
                                          k.shape[2], _native._strides(k), _native._strides(v), _ptr(counts),
                                          _native._stream(k))
    _native._check(rc, "bsa_kv8_append")


def cache_unpack(c, dtype, k=None, v=None, rows: Optional[int] = None):
    B, Hk, cap, D = c.k_codes.shape
    n = k.shape[2] if k is not None else 0
    rows = cap + n if rows is None else rows
    ko, vo = (torch.empty((B, Hk, rows, D), device=c.k_codes.device, dtype=dtype) for _ in range(2))
    ks = vs = None
    if n:
        k, v = _readable(k), _readable(v)
        ks, vs = _native._strides(k), _native._strides(v)
    with _on(ko):
        rc = _native.lib().bsa_kv8_unpack(*_cache_args(c), _ptr(k) if n else None, _ptr(v) if n else None,
                                          _native.DTYPE_CODES[dtype], n, ks, vs, ko.data_ptr(), vo.data_ptr(), rows,
                                          _native._stream(ko))
    _native._check(rc, "bsa_kv8_unpack")
    return ko, vo


def cache_attention(c, q, causal: bool, sm_scale: float, out: torch.Tensor) -> torch.Tensor:
    B, H, Sq, D = q.shape
    Hk, cap = c.k_codes.shape[1], c.k_codes.shape[2]
    q = _readable(q)
    target = out
    if _native._misaligned(out) or out.stride(-1) != 1:
        target = torch.empty((B, H, Sq, D), device=q.device, dtype=q.dtype)
    with _on(q):
        n = int(_native.lib().bsa_kv8_attention_scratch_bytes(B, H, Hk, Sq, cap, D))
        scratch = torch.empty((n,), device=q.device, dtype=torch.uint8) if n else None
        rc = _native.lib().bsa_kv8_attention(
            q.data_ptr(), _native._dtype_code(q), B, H, Sq, _native._strides(q), c.k_codes.data_ptr(),
            c.k_scale.data_ptr(), c.v_codes.data_ptr(), c.v_scale.data_ptr(), c.lengths.data_ptr(), Hk, cap, D,
            int(bool(causal)), float(sm_scale), target.data_ptr(), _native._strides(target), _ptr(scratch),
            _native._stream(q))
    _native._check(rc, "bsa_kv8_attention")
    if target is not out:
        out.copy_(target)
    return out
