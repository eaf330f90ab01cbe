"""Bindings of the C ABI's dense side (include/bsa_b200.h): q/k norm with rotary positions, attention over key
intervals, and the 8-bit key/value cache.  Argument checks, allocation of outputs and scratch, and the
launch on the tensors' device and its current stream; the public functions are in ``models``."""

from __future__ import annotations

import functools
import struct
from typing import Optional, Tuple

import torch

from . import _native

CACHE_BLOCK = 64  # tokens of a head that share a scale


_pack3 = struct.Struct("3q").pack  # the strides of one tensor, as the C ABI reads them
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _call(name: str, device: int, *args) -> None:
    """One C entry on ``device`` and its current stream (the entry's last argument)."""
    fn = getattr(_native.lib(), name)
    if _current_device() == device:
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        _native._check(rc, name)


def _same_place(*tensors: Optional[torch.Tensor]) -> None:
    device = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected torch tensors")
        d = t.get_device()
        if d < 0:
            raise ValueError("BSA engine inputs must be CUDA tensors (there is no CPU path)")
        if device is None:
            device = d
        elif d != device:
            raise ValueError("all tensors must be on one device")


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _view(t: torch.Tensor) -> Tuple[torch.Tensor, int, bytes]:
    """(tensor to keep alive, address, strides) of a [B, H, S, D] tensor that the kernels can read in place, else of a
    contiguous copy.  In place: d contiguous, base and strides in multiples of 16 bytes, nothing broadcast; any
    order and gaps of batch, heads and tokens otherwise."""
    sb, sh, ss, sd = t.stride()
    p = t.data_ptr()
    if sd != 1 or p & 15 or (sb | sh | ss) & (16 // t.element_size() - 1) or not (sb and sh and ss):
        # an axis of one element may have any stride, which the kernels do not use
        sizes = t.shape
        sb, sh, ss = (st if n > 1 else 8 * sizes[3] for st, n in zip((sb, sh, ss), sizes))
        if sd != 1 or p & 15 or (sb | sh | ss) & (16 // t.element_size() - 1) or not (sb and sh and ss):
            t = t.clone(memory_format=torch.contiguous_format)
            sb, sh, ss, _ = t.stride()
            p = t.data_ptr()
    return t, p, _pack3(sb, sh, ss)


def _out_view(t: torch.Tensor) -> Optional[Tuple[int, bytes]]:
    """(address, strides) of an output that the kernels can write in place, else None."""
    sb, sh, ss, sd = t.stride()
    p = t.data_ptr()
    if sd != 1 or p & 15 or (sb | sh | ss) & (16 // t.element_size() - 1):
        return None
    return p, _pack3(sb, sh, ss)


def _i32(t: Optional[torch.Tensor], name: str, shape: Optional[Tuple[int, ...]] = None) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t.contiguous()


# ------------------------------------------------------------------------------- q/k norm + rotary positions
@functools.lru_cache(maxsize=1024)
def _scratch(name: str, device: int, *sizes: int) -> int:
    """Scratch bytes of a call of these sizes (a function of them and of the device's SM count)."""
    with torch.cuda.device(device):
        return int(getattr(_native.lib(), name)(*sizes))


def _rope_args(rope, start: int):
    if rope is None:
        return (None, 0, 0, 0, 0, 0, 0, 0)
    tables, (dt, dh, dw), (T, H, W) = rope
    if tables.dtype is not torch.float32 or not tables.is_contiguous():
        raise ValueError("rope tables must be contiguous fp32")
    if tables.numel() != T * dt + H * dh + W * dw:
        raise ValueError(f"rope tables of {tables.numel()} values do not match grid {(T, H, W)} and dims {(dt, dh, dw)}")
    return (tables.data_ptr(), dt, dh, dw, T, H, W, start)


def _norm_rope_check(xs, ws, rope):
    _same_place(*xs, *ws, rope[0] if rope is not None else None)
    x = xs[0]
    shape, dt = x.shape, x.dtype
    if dt not in _native.DTYPE_CODES:
        raise ValueError(f"unsupported dtype {dt}")
    if len(shape) != 4:
        raise ValueError("expected tensors of shape [B, H, S, D]")
    for t in xs[1:]:
        st = t.shape
        if t.dtype is not dt or len(st) != 4 or st[0] != shape[0] or st[2] != shape[2] or st[3] != shape[3]:
            raise ValueError("q and k must share dtype, batch, length and head_dim")
    for w in ws:
        if w is not None and (w.dim() != 1 or w.shape[0] != shape[3]):
            raise ValueError(f"norm weight must be [{shape[3]}]")


def _weights(ws, x: torch.Tensor):
    """Contiguous weights of one type: fp32 or the input's are read as they are, others as fp32."""
    kind = None
    for w in ws:
        if w is not None:
            if not w.is_contiguous() or (w.dtype is not torch.float32 and w.dtype is not x.dtype) or \
                    (kind is not None and w.dtype is not kind):
                return [u.float().contiguous() if u is not None else None for u in ws], 0
            kind = w.dtype
    return ws, _native.DTYPE_CODES[kind] if kind is not None else 0


def norm_rope(xs, ws, eps: float, rope, start: int):
    _norm_rope_check(xs, ws, rope)
    x = xs[0]
    B, _, S, D = x.shape
    ys = [t.new_empty(t.shape) for t in xs]
    for t in xs:
        if t.numel() == 0:
            return ys
    views = [_view(t) for t in xs]
    ws, wcode = _weights(ws, x)
    sides = []
    for (t, p, st), w, y in zip(views, ws, ys):
        sides += (p, st, t.shape[1], _ptr(w), y.data_ptr())
    if len(xs) == 1:
        sides += (None, None, 0, None, None)
    _call("bsa_norm_rope", x.get_device(), *sides, _native.DTYPE_CODES[x.dtype], wcode, B, S, D, eps,
          *_rope_args(rope, start))
    return ys


def norm_rope_backward(xs, gs, ws, eps: float, rope, start: int, want_dw):
    x = xs[0]
    B, _, S, D = x.shape
    dxs = [t.new_empty(t.shape) for t in xs]
    if any(t.numel() == 0 for t in xs):
        return dxs, [torch.zeros((D,), device=x.device) if want else None for want in want_dw]
    dws = [x.new_empty((D,), dtype=torch.float32) if want else None for want in want_dw]
    xv, gv = [_view(t) for t in xs], [_view(g) for g in gs]
    ws, wcode = _weights(ws, x)
    sides = []
    for (t, p, st), (_, gp, gst), w, dx, dw in zip(xv, gv, ws, dxs, dws):
        sides += (p, st, gp, gst, t.shape[1], _ptr(w), dx.data_ptr(), _ptr(dw))
    if len(xs) == 1:
        sides += (None, None, None, None, 0, None, None, None)
    scratch = None
    if any(want_dw):
        scratch = x.new_empty((_scratch("bsa_norm_rope_backward_scratch_bytes", x.get_device(), x.shape[1],
                                       xs[1].shape[1] if len(xs) > 1 else 0, D),), dtype=torch.uint8)
    _call("bsa_norm_rope_backward", x.get_device(), *sides, _native.DTYPE_CODES[x.dtype], wcode, B, S, D, eps,
          *_rope_args(rope, start), _ptr(scratch))
    return dxs, dws


# ------------------------------------------------------------------------------------------- key intervals
def attention_ranges(batch: int, Sq: int, Sk: int, *, device, given=None, causal=False, prefix=0, prefixes=None,
                     q_offsets=None, k_offsets=None, q_lengths=None, k_lengths=None, k_add: int = 0):
    """The intervals and their tile table in one allocation: (buffer, address of ranges, address of table)."""
    n = batch * Sq * 2
    at = (n + 3) & ~3  # the table starts on 16 bytes
    buf = torch.empty((at + batch * ((Sq + 127) // 128) * 4,), device=device, dtype=torch.int32)
    _same_place(buf, given, prefixes, q_offsets, k_offsets, q_lengths, k_lengths)
    ranges = buf.data_ptr()
    table = ranges + 4 * at
    if n:
        _call("bsa_attention_ranges", buf.get_device(), ranges, table, batch, Sq, Sk, _ptr(given), 1 if causal else 0,
              prefix, _ptr(prefixes), _ptr(q_offsets), _ptr(k_offsets),
              q_offsets.numel() - 1 if q_offsets is not None else 0, _ptr(q_lengths), _ptr(k_lengths), k_add)
    return buf, ranges, table


# ------------------------------------------------------------------------------------------ dense attention
def check_qkv(q, k, v) -> None:
    _same_place(q, k, v)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError("q, k and v must be [B, H, S, D]")
    if ks != v.shape:
        raise ValueError("k and v must have the same shape")
    dt = q.dtype
    if dt != k.dtype or dt != v.dtype:
        raise ValueError("q, k, v must share one dtype")
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise ValueError(f"unsupported dtype {dt} (bf16 or fp16)")
    if qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError("q and k must share batch and head_dim")
    if qs[3] % 8 or not 0 < qs[3] <= 128:
        raise ValueError(f"head_dim D={qs[3]} must be a multiple of 8 and <= 128")
    if ks[1] == 0 or qs[1] % ks[1]:
        raise ValueError(f"{qs[1]} query heads are no multiple of {ks[1]} key heads")


def check_scale(sm_scale: float, softcap: float = 0.0) -> None:
    if not 0.0 < sm_scale < float("inf"):
        raise ValueError("sm_scale must be positive and finite")
    if not 0.0 <= softcap < float("inf"):
        raise ValueError("softcap must be finite and >= 0")


def masked_attention(q, k, v, ranges, table, batch: int, sm_scale: float, softcap: float, out=None,
                     want_lse: bool = False, rest: Optional[torch.Tensor] = None):
    """(out, lse or None).  ranges / table: addresses of attention_ranges with ``batch`` entries, or None for every key.
    ``rest`` (contiguous, like out) receives what out's rounding left over."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    lse = q.new_empty((B, H, Sq), dtype=torch.float32) if want_lse else None
    target, tv = out, None
    if out is not None:
        tv = _out_view(out)
    if tv is None:
        target = q.new_empty((B, H, Sq, D))
        tv = target.data_ptr(), _pack3(H * Sq * D, Sq * D, D)
    if B and H and Sq and Sk:
        (q, qp, qst), (k, kp, kst), (v, vp, vst) = _view(q), _view(k), _view(v)
        device = q.get_device()
        n = _scratch("bsa_masked_attention_scratch_bytes", device, B, H, Sq, Sk, D)
        scratch = q.new_empty((n,), dtype=torch.uint8) if n else None
        _call("bsa_masked_attention", device, qp, kp, vp, _native.DTYPE_CODES[q.dtype], B, H, Hk, Sq, Sk, D, qst, kst,
              vst, ranges, table, batch, sm_scale, softcap, tv[0], tv[1], _ptr(rest), _ptr(lse), _ptr(scratch))
    else:  # no rows, or no keys: zeros
        target.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
    if out is not None and target is not out:
        out.copy_(target)
        target = out
    return target, lse


def masked_attention_backward(q, k, v, out, rest, lse, grad, ranges, table, batch: int, sm_scale: float,
                              softcap: float, want_q: bool, want_kv: bool):
    """(dq, dk, dv), contiguous; None where not wanted."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    empty = not (B and H and Sq and Sk)
    new = q.new_zeros if empty else q.new_empty
    dq = new((B, H, Sq, D)) if want_q else None
    dk, dv = (new((B, Hk, Sk, D)) if want_kv else None for _ in range(2))
    if empty:
        return dq, dk, dv
    (q, qp, qst), (k, kp, kst), (v, vp, vst) = _view(q), _view(k), _view(v)
    (out, op, ost), (grad, gp, gst) = _view(out), _view(grad)
    device = q.get_device()
    n = _scratch("bsa_masked_attention_backward_scratch_bytes", device, B, H, Sq, batch if ranges else 0)
    scratch = q.new_empty((n,), dtype=torch.uint8)
    _call("bsa_masked_attention_backward", device, qp, kp, vp, op, rest.data_ptr(), gp, lse.data_ptr(),
          _native.DTYPE_CODES[q.dtype], B, H, Hk, Sq, Sk, D, qst, kst, vst, ost, gst, ranges, table, batch, sm_scale,
          softcap, _ptr(dq), _ptr(dk), _ptr(dv), scratch.data_ptr())
    return dq, dk, dv


# ---------------------------------------------------------------------------------------------- 8-bit cache
def _cache_args(c):
    return (c.k_codes.data_ptr(), c.k_scale.data_ptr(), c.v_codes.data_ptr(), c.v_scale.data_ptr(),
            c.lengths.data_ptr(), *c.k_codes.shape)


def cache_append(c, k, v, counts) -> None:
    (k, kp, kst), (v, vp, vst) = _view(k), _view(v)
    _call("bsa_kv8_append", k.get_device(), *_cache_args(c), kp, vp, _native.DTYPE_CODES[k.dtype], k.shape[2], kst, vst,
          _ptr(counts))


def cache_unpack(c, dtype, k=None, v=None):
    """(k, v) in 16 bits: the held tokens, the fresh ones k, v, zeros up to capacity + fresh."""
    B, Hk, cap, D = c.k_codes.shape
    n, kp, vp, kst, vst = 0, None, None, None, None
    if k is not None:
        n = k.shape[2]
        (k, kp, kst), (v, vp, vst) = _view(k), _view(v)
    ko, vo = (c.k_codes.new_empty((B, Hk, cap + n, D), dtype=dtype) for _ in range(2))
    _call("bsa_kv8_unpack", ko.get_device(), *_cache_args(c), kp, vp, _native.DTYPE_CODES[dtype], n, kst, vst,
          ko.data_ptr(), vo.data_ptr(), cap + n)
    return ko, vo


def cache_attention(c, q, causal: bool, sm_scale: float, out: torch.Tensor) -> torch.Tensor:
    B, H, Sq, D = q.shape
    _, Hk, cap, _ = c.k_codes.shape
    q, qp, qst = _view(q)
    target, tv = out, _out_view(out)
    if tv is None:
        target = q.new_empty((B, H, Sq, D))
        tv = target.data_ptr(), _pack3(H * Sq * D, Sq * D, D)
    device = q.get_device()
    n = _scratch("bsa_kv8_attention_scratch_bytes", device, B, H, Hk, Sq, cap, D)
    scratch = q.new_empty((n,), dtype=torch.uint8) if n else None
    _call("bsa_kv8_attention", device, qp, _native.DTYPE_CODES[q.dtype], B, H, Sq, qst, c.k_codes.data_ptr(),
          c.k_scale.data_ptr(), c.v_codes.data_ptr(), c.v_scale.data_ptr(), c.lengths.data_ptr(), Hk, cap, D,
          1 if causal else 0, sm_scale, tv[0], tv[1], _ptr(scratch))
    if target is not out:
        out.copy_(target)
    return out
