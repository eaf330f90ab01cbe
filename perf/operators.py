"""Work of the dense side of the attention hook: q/k norm + 3-axis rotary positions, masked dense attention
with its gradient, and attention over an 8-bit key/value cache.

`listed()` names the cases, `run()` makes one pass: in plain torch where `own` is false, through the
framework's operators where it is true.  Layouts are the framework's: q [B, H, S, D], k and v
[B, Hk, S, D] with H a multiple of Hk; cache codes [B, Hk, capacity, D] e4m3 with one fp32 power-of-two
scale for each 64 tokens of a head, [B, Hk, capacity / 64].
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 64  # cache tokens that share a scale
EPS = 1e-6


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one latent frame of a small preview: a few hundred tokens, where the launch counts
        dict(name="norm_rope_frame", op="norm_rope", B=1, H=32, Hk=32, T=1, h=15, w=26, D=128, start=0,
             dtype="bf16", train=False),
        # 480p training step of one layer: six latent frames, norm and rotation with their gradients
        dict(name="norm_rope_train", op="norm_rope", B=1, H=32, Hk=32, T=6, h=30, w=52, D=128, start=0,
             dtype="bf16", train=True),
        # the 720p refinement's whole latent grid, half of the heads (two ranks)
        dict(name="norm_rope_720p", op="norm_rope", B=1, H=16, Hk=16, T=24, h=45, w=80, D=128, start=0,
             dtype="bf16", train=False),
        # a padded batch of short queries over longer keys
        dict(name="attn_padded", op="attention", B=2, H=8, Hk=8, Sq=77, Sk=1001, D=128, docs=0, padded=True,
             causal=False, prefix=0, softcap=0.0, dtype="bf16", train=False),
        # packed documents of a text tower: shared key heads, narrow heads, capped scores, a padded tail
        dict(name="attn_documents", op="attention", B=1, H=12, Hk=4, Sq=4096, Sk=4096, D=64, docs=7, padded=False,
             causal=True, prefix=0, softcap=50.0, dtype="fp16", train=False),
        # 480p continuation: 4 conditioning frames of 13, which see only themselves; heads of one of 4 ranks
        dict(name="attn_cond_480p", op="attention", B=1, H=8, Hk=8, Sq=20280, Sk=20280, D=128, docs=0, padded=False,
             causal=False, prefix=6240, softcap=0.0, dtype="bf16", train=False),
        # training on packed clips and captions with shared key heads
        dict(name="attn_train_documents", op="attention", B=1, H=16, Hk=4, Sq=4680, Sk=4680, D=128, docs=9,
             padded=False, causal=True, prefix=64, softcap=30.0, dtype="bf16", train=True),
        # training with conditioning frames at 480p
        dict(name="attn_train_cond", op="attention", B=1, H=8, Hk=8, Sq=9360, Sk=9360, D=128, docs=0, padded=False,
             causal=False, prefix=1560, softcap=0.0, dtype="bf16", train=True),
        # filling the cache with the conditioning frames
        dict(name="cache_append_prompt", op="append", B=1, Hk=32, D=128, cap=8192, filled=0, n=6240, dtype="bf16"),
        # one more token of every sequence
        dict(name="cache_append_token", op="append", B=16, Hk=8, D=128, cap=4096, filled=3001, n=1, dtype="bf16"),
        # one token of every sequence over a long ragged cache
        dict(name="cache_token", op="attend", B=8, H=32, Hk=8, D=128, cap=32768, filled=32001, Sq=1, fresh=False,
             causal=True, dtype="bf16"),
        # the denoising frames of a continuation over the cached conditioning frames and themselves
        dict(name="cache_continuation", op="attend", B=1, H=8, Hk=8, D=128, cap=6272, filled=6240, Sq=14040,
             fresh=True, causal=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "attention", "attention", "train", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([128, 128, 64, 80, 40])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    if op == "norm_rope":
        T, h, w = rng.randint(1, 16), rng.randint(1, 45), rng.randint(1, 80)
        return dict(op=op, B=rng.choice([1, 1, 2]), H=H, Hk=Hk, T=T, h=h, w=w, D=D, start=rng.choice([0, h * w]),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), train=rng.random() < 0.5)
    if op in ("attention", "train"):
        train = op == "train"
        most = 6.0e8 if train else 2.4e9  # B * H * Sq * Sk
        B = rng.choice([1, 1, 2, 4])
        docs = rng.choice([0, 0, 3, 8, 21])
        Sk = _log(rng, 5, 12000)
        Sq = Sk if docs or train or rng.random() < 0.6 else _log(rng, 1, 6000)
        while B * H * Sq * Sk > most:
            Sq, Sk = (Sq * 2 + 2) // 3, (Sk * 2 + 2) // 3
        prefix = rng.choice([0, 0, Sk // 3])
        return dict(op="attention", B=B, H=H, Hk=Hk, Sq=Sq, Sk=Sk, D=D, docs=docs,
                    padded=not docs and rng.random() < 0.4, causal=rng.random() < 0.5,
                    prefix=prefix, softcap=rng.choice([0.0, 0.0, 30.0]), dtype=dtype, train=train)
    if op == "append":
        filled, n = rng.choice([0, rng.randint(1, 4000)]), _log(rng, 1, 6000)
        B = rng.choice([1, 2, 8])
        return dict(op=op, B=B, Hk=Hk, D=D, cap=-(-(filled + n) // BLOCK) * BLOCK + BLOCK * rng.randint(0, 9),
                    filled=filled, n=n, dtype=dtype)
    filled, fresh = _log(rng, 1, 20000), rng.random() < 0.4
    B = 1 if fresh else rng.choice([1, 2, 8])
    Sq = _log(rng, 64, 6000) if fresh else min(filled, rng.choice([1, 1, 2, 5, 16, 100]))
    while B * H * Sq * (filled + Sq) > 2.4e9:
        Sq, filled = (Sq * 2 + 2) // 3, (filled * 2 + 2) // 3
    return dict(op=op, B=B, H=H, Hk=Hk, D=D, cap=-(-filled // BLOCK) * BLOCK + BLOCK * rng.randint(0, 3),
                filled=filled, Sq=Sq, fresh=fresh, causal=fresh or rng.random() < 0.7, dtype=dtype)


# -------------------------------------------------------------------- what a case says about its layout
def _offsets(total, docs, salt):
    """Document borders 0 = o[0] <= ... <= o[docs] <= total: ragged, with a padded tail behind the last."""
    r = random.Random(1000 * docs + salt)
    end = total - total // 50
    return [0] + sorted(r.randint(0, end) for _ in range(docs - 1)) + [end]


def _lengths(B, most, salt):
    """Ragged lengths of a batch, the first one full."""
    r = random.Random(77 + salt)
    return [most] + [r.randint((most + 1) // 2, most) for _ in range(B - 1)]


def _visible(c):
    """[B, Sq, 2] numpy: the keys [lo, hi) that each query row sees."""
    B, Sq, Sk, prefix = c["B"], c["Sq"], c["Sk"], c["prefix"]
    lo, hi = np.zeros((B, Sq), np.int64), np.zeros((B, Sq), np.int64)
    for b in range(B):
        if c["docs"]:
            o = _offsets(Sq, c["docs"], 0)
            parts = [(s, e, s, e) for s, e in zip(o, o[1:])]
        else:
            parts = [(0, Sq, 0, _lengths(B, Sk, 1)[b] if c["padded"] else Sk)]
        for qs, qe, ks, ke in parts:
            n = ke - ks
            at = np.arange(qe - qs) + n - (qe - qs)  # a query's place among the keys: the last ones line up
            seen = at + 1 if c["causal"] else np.full_like(at, n)
            seen = np.where(at < prefix, prefix if prefix else seen, seen) if prefix else seen
            lo[b, qs:qe], hi[b, qs:qe] = ks, ks + np.clip(seen, 0, n)
    return np.stack([lo, hi], -1)


def _grid(c):
    """The rotary grid: `start` tokens (whole frames) lie before the first token."""
    return (c["T"] + c["start"] // (c["h"] * c["w"]), c["h"], c["w"])


def _axis_dims(D):
    d6 = D // 6
    return (D - 4 * d6, 2 * d6, 2 * d6)


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "norm_rope":
        n = c["B"] * (c["H"] + c["Hk"]) * c["T"] * c["h"] * c["w"] * c["D"]
        return {"bytes": n * e * (5 if c["train"] else 2), "flops": n * (30 if c["train"] else 10)}
    if c["op"] == "attention":
        r = _visible(c)
        pairs = float((r[..., 1] - r[..., 0]).sum()) * c["H"]
        q, kv = c["B"] * c["H"] * c["Sq"] * c["D"], c["B"] * c["Hk"] * c["Sk"] * c["D"]
        # forward: q, k, v in, out out; backward: those and dout in, dq, dk, dv out
        return {"bytes": e * ((2 * q + 2 * kv) + (4 * q + 4 * kv if c["train"] else 0)),
                "flops": pairs * c["D"] * (14 if c["train"] else 4)}
    if c["op"] == "append":
        n = c["B"] * c["Hk"] * c["n"] * c["D"]
        return {"bytes": 2 * n * 3, "flops": 4 * n}
    held = sum(_lengths(c["B"], c["filled"], 2))
    keys = held * c["Sq"] - (c["B"] * c["Sq"] * (c["Sq"] - 1) // 2 if c["causal"] and not c["fresh"] else 0)
    if c["fresh"]:
        keys += c["B"] * (c["Sq"] * (c["Sq"] + 1) // 2 if c["causal"] else c["Sq"] * c["Sq"])
    q = c["B"] * c["H"] * c["Sq"] * c["D"]
    fresh = 2 * e * c["B"] * c["Hk"] * c["Sq"] * c["D"] if c["fresh"] else 0
    return {"bytes": 2 * held * c["Hk"] * c["D"] + 2 * q * e + fresh, "flops": 4.0 * keys * c["H"] * c["D"]}


# ------------------------------------------------------------------------------------------ inputs
def _to8(x, scale):
    """Codes of x / scale (a power of two: exact), rounded to nearest even."""
    inv = torch.where(scale > 0, 1.0 / torch.where(scale > 0, scale, 1.0), 0.0)
    return (x * inv).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _scale_of(amax):
    """The smallest power of two s with amax / s <= 448 (0 for 0)."""
    m, e = torch.frexp(amax)  # m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).to(e.dtype))
    return torch.where(amax > 0, s.clamp(min=2.0 ** -126), torch.zeros_like(s))


def _filled_cache(c, gen, dt, dev):
    B, Hk, cap, D = c["B"], c["Hk"], c["cap"], c["D"]
    lengths = torch.tensor(_lengths(B, c["filled"], 2) if c["filled"] else [0] * B, dtype=torch.int32, device=dev)
    held = (torch.arange(cap, device=dev)[None] < lengths[:, None])[:, None, :, None]
    parts = []
    for _ in range(2):
        x = torch.randn((B, Hk, cap, D), generator=gen, device=dev, dtype=torch.float32).to(dt)
        x = torch.where(held, x, torch.zeros_like(x)).float()
        s = _scale_of(x.view(B, Hk, cap // BLOCK, BLOCK * D).abs().amax(-1))
        parts += [_to8(x.view(B, Hk, cap // BLOCK, BLOCK, D), s[..., None, None]).view(B, Hk, cap, D), s]
        del x
    return dict(k_codes=parts[0], k_scale=parts[1], v_codes=parts[2], v_scale=parts[3], lengths=lengths)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dt)

    st = dict(case=c)
    B, D = c["B"], c["D"]
    if c["op"] == "norm_rope":
        # q and k as the projection leaves them: views of [B, N, heads, D]
        N, H, Hk = c["T"] * c["h"] * c["w"], c["H"], c["Hk"]
        qkv = rand(B, N, H + 2 * Hk, D)
        st["q"], st["k"] = qkv[:, :, :H].transpose(1, 2), qkv[:, :, H:H + Hk].transpose(1, 2)
        st["wq"] = 1.0 + 0.2 * torch.randn(D, generator=gen, device=dev)
        st["wk"] = 1.0 + 0.2 * torch.randn(D, generator=gen, device=dev)
        if c["train"]:
            st["gq"], st["gk"] = rand(B, H, N, D), rand(B, Hk, N, D)
        flat = []  # cos_t | sin_t | cos_h | sin_h | cos_w | sin_w, one angle for each rotated pair
        for n, dim in zip(_grid(c), _axis_dims(D)):
            freq = 10000.0 ** (-np.arange(0, dim, 2, dtype=np.float64) / max(dim, 1))
            ang = np.arange(n)[:, None] * freq[None]
            flat += [np.cos(ang).ravel(), np.sin(ang).ravel()]
        st["tables"] = torch.from_numpy(np.concatenate(flat).astype(np.float32)).to(dev)
    elif c["op"] == "attention":
        # capped scores matter where they are large
        st["q"] = rand(B, c["H"], c["Sq"], D, scale=4.0 if c["softcap"] else 1.0)
        st["k"], st["v"] = rand(B, c["Hk"], c["Sk"], D), rand(B, c["Hk"], c["Sk"], D)
        if c["train"]:
            st["g"] = rand(B, c["H"], c["Sq"], D)
        i32 = dict(dtype=torch.int32, device=dev)
        st["offsets"] = torch.tensor(_offsets(c["Sq"], c["docs"], 0), **i32) if c["docs"] else None
        st["k_lengths"] = torch.tensor(_lengths(B, c["Sk"], 1), **i32) if c["padded"] else None
    elif c["op"] == "append":
        st.update(_filled_cache(c, gen, dt, dev))
        st["start"] = st["lengths"].clone()
        st["k"], st["v"] = rand(B, c["Hk"], c["n"], D, scale=1.5), rand(B, c["Hk"], c["n"], D)
    else:
        st.update(_filled_cache(c, gen, dt, dev))
        st["q"] = rand(B, c["H"], c["Sq"], D)
        if c["fresh"]:
            st["k"], st["v"] = rand(B, c["Hk"], c["Sq"], D), rand(B, c["Hk"], c["Sq"], D)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _plain_angles(c, tables):
    """[N, D / 2] cos and sin of the case's tokens from the per-axis tables."""
    T, h, w = _grid(c)
    at, cos, sin = 0, [], []
    s = torch.arange(c["start"], c["start"] + c["T"] * c["h"] * c["w"], device=tables.device)
    t0, h0, w0 = _axis_dims(c["D"])
    nt, nh, nw = t0 // 2, h0 // 2, w0 // 2
    ct, tt = tables[:T * nt].view(T, nt), tables[T * nt:2 * T * nt].view(T, nt)
    at = 2 * T * nt
    ch, th = tables[at:at + h * nh].view(h, nh), tables[at + h * nh:at + 2 * h * nh].view(h, nh)
    at += 2 * h * nh
    cw, tw = tables[at:at + w * nw].view(w, nw), tables[at + w * nw:at + 2 * w * nw].view(w, nw)
    cos = torch.cat([ct[s // (h * w)], ch[(s // w) % h], cw[s % w]], -1)
    sin = torch.cat([tt[s // (h * w)], th[(s // w) % h], tw[s % w]], -1)
    return cos, sin


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _plain_norm_rope(x, weight, cos, sin, grad=None):
    xf = x.float()
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    out = _rotate(xf * r * weight, cos, sin).to(x.dtype)
    if grad is None:
        return out, None, None
    dz = _rotate(grad.float(), cos, -sin)
    dw = (dz * xf * r).sum((0, 1, 2))
    g = dz * weight
    dx = r * g - xf * (r * r * r) * (g * xf).mean(-1, keepdim=True)
    return out, dx.to(x.dtype), dw


def _plain_mask(c, offsets, k_lengths, dev):
    """[B or 1, 1, 1, Sq, Sk] truth values."""
    i, j = torch.arange(c["Sq"], device=dev)[:, None], torch.arange(c["Sk"], device=dev)[None]
    if offsets is not None:
        last = offsets.numel() - 1
        dq = torch.searchsorted(offsets.long(), i[:, 0].contiguous(), right=True)[:, None]
        dk = torch.searchsorted(offsets.long(), j[0].contiguous(), right=True)[None]
        first = torch.cat([offsets[:1], offsets]).long()[dq]
        ok = (dq == dk) & (dq <= last)
        at, kj = i - first, j - first
    else:
        n = (k_lengths.long() if k_lengths is not None else torch.tensor([c["Sk"]], device=dev))[:, None, None]
        ok, at, kj = j[None] < n, i[None] + n - c["Sq"], j[None]
    seen = kj <= at if c["causal"] else torch.ones_like(kj <= at)
    if c["prefix"]:
        # the prefix sees itself whole and nothing else; the rest sees it whole
        head = kj < c["prefix"]
        seen = torch.where(at < c["prefix"], head, head | seen)
    ok = ok & seen
    return ok.view(-1, 1, 1, c["Sq"], c["Sk"])


def _plain_attention(q, k, v, ok, softcap, grad=None):
    B, H, Sq, D = q.shape
    Hk = k.shape[1]
    qf, kf, vf = q.float().view(B, Hk, H // Hk, Sq, D), k.float()[:, :, None], v.float()[:, :, None]
    scale = 1.0 / math.sqrt(D)
    s = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale)
    t = None
    if softcap:
        t = torch.tanh(s / softcap)
        s = t * softcap
    s = s.masked_fill_(~ok, -math.inf) if ok is not None else s
    m = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)))
    l = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(l > 0, l, torch.ones_like(l)))
    of = torch.matmul(p, vf)
    out = of.view(B, H, Sq, D).to(q.dtype)
    if grad is None:
        return out
    gf = grad.float().view(B, Hk, H // Hk, Sq, D)
    dv = torch.matmul(p.transpose(-1, -2), gf).sum(2)
    ds = torch.matmul(gf, vf.transpose(-1, -2)).sub_((gf * of).sum(-1, keepdim=True)).mul_(p)
    if softcap:
        ds.mul_(1 - t * t)
    dq = torch.matmul(ds, kf).mul_(scale).view(B, H, Sq, D)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2).mul_(scale)
    return out, dq.to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def _plain_append(codes, scale, lengths, x):
    B, Hk, cap, D = codes.shape
    n, nb = x.shape[2], cap // BLOCK
    pos = torch.arange(cap, device=x.device)[None] - lengths.long()[:, None]  # place among the new tokens
    new = ((pos >= 0) & (pos < n))[:, None, :, None]
    xf = torch.gather(x.float(), 2, pos.clamp(0, n - 1)[:, None, :, None].expand(B, Hk, cap, D))
    xf = torch.where(new, xf, torch.zeros_like(xf))
    need = _scale_of(xf.view(B, Hk, nb, BLOCK * D).abs().amax(-1))
    touched = new.view(B, 1, nb, BLOCK).any(-1)
    raised = torch.where(touched, torch.maximum(scale, need), scale)
    each, was = raised.repeat_interleave(BLOCK, 2)[..., None], scale.repeat_interleave(BLOCK, 2)[..., None]
    old = _to8(codes.float() * was, each)
    keep = ((pos < 0)[:, None, :, None]) & touched.repeat_interleave(BLOCK, 2)[..., None]
    u8 = torch.where(new, _to8(xf, each).view(torch.uint8),
                     torch.where(keep, old.view(torch.uint8), codes.view(torch.uint8)))
    return u8.view(torch.float8_e4m3fn), raised


def _plain_attend(st):
    c = st["case"]
    q = st["q"]
    k = st["k_codes"].float() * st["k_scale"].repeat_interleave(BLOCK, 2)[..., None]
    v = st["v_codes"].float() * st["v_scale"].repeat_interleave(BLOCK, 2)[..., None]
    cap, Sq, dev = c["cap"], c["Sq"], q.device
    n = st["lengths"].long()[:, None, None]
    i, j = torch.arange(Sq, device=dev)[None, :, None], torch.arange(cap, device=dev)[None, None]
    if c["fresh"]:
        ok = (j < n).expand(-1, Sq, -1)
        jf = torch.arange(Sq, device=dev)[None, None]
        fresh_ok = (jf <= i) if c["causal"] else torch.ones((1, Sq, Sq), dtype=torch.bool, device=dev)
        ok = torch.cat([ok, fresh_ok.expand(ok.shape[0], -1, -1)], -1)
        k, v = torch.cat([k, st["k"].float()], 2), torch.cat([v, st["v"].float()], 2)
    else:
        ok = (j < n) & (j <= n - Sq + i) if c["causal"] else (j < n).expand(-1, Sq, -1)
    return _plain_attention(q, k, v, ok[:, None, None], 0.0)


# --------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(st):
    c = st["case"]
    if c["op"] == "norm_rope":
        cos, sin = _plain_angles(c, st["tables"])
        q, dq, dwq = _plain_norm_rope(st["q"], st["wq"], cos, sin, st.get("gq"))
        k, dk, dwk = _plain_norm_rope(st["k"], st["wk"], cos, sin, st.get("gk"))
        return dict(q=q, k=k, dq=dq, dk=dk, dwq=dwq, dwk=dwk) if c["train"] else dict(q=q, k=k)
    if c["op"] == "attention":
        masked = c["docs"] or c["padded"] or c["causal"] or c["prefix"]
        ok = _plain_mask(c, st["offsets"], st["k_lengths"], st["q"].device) if masked else None
        r = _plain_attention(st["q"], st["k"], st["v"], ok, c["softcap"], st.get("g"))
        return dict(out=r[0], dq=r[1], dk=r[2], dv=r[3]) if c["train"] else dict(out=r)
    if c["op"] == "append":
        kc, ks = _plain_append(st["k_codes"], st["k_scale"], st["start"], st["k"])
        vc, vs = _plain_append(st["v_codes"], st["v_scale"], st["start"], st["v"])
        return dict(k_codes=kc, k_scale=ks, v_codes=vc, v_scale=vs, lengths=st["start"] + c["n"])
    return dict(out=_plain_attend(st))


def _package():
    import sys
    from pathlib import Path

    here = str(Path(__file__).resolve().parent.parent / "longcat-video-mlx_b200")
    if here not in sys.path:
        sys.path.insert(0, here)


def _run_own(st):
    c = st["case"]
    _package()
    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import AttentionMask, masked_attention
    from longcat_video.models.rope_3d import qk_norm_rope

    if c["op"] == "norm_rope":
        rope = (st["tables"], _axis_dims(c["D"]), _grid(c))
        if not c["train"]:
            q, k = qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], EPS, rope=rope, start=c["start"])
            return dict(q=q, k=k)
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
        q, k = qk_norm_rope(*leaves, EPS, rope=rope, start=c["start"])
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (st["gq"], st["gk"]))
        return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    if c["op"] == "attention":
        mask = None
        if c["docs"] or c["padded"] or c["causal"] or c["prefix"]:
            mask = AttentionMask.build(c["Sq"], c["Sk"], causal=c["causal"], prefix=c["prefix"],
                                       q_offsets=st["offsets"], k_offsets=st["offsets"],
                                       k_lengths=st["k_lengths"], device=st["q"].device)
        if not c["train"]:
            return dict(out=masked_attention(st["q"], st["k"], st["v"], mask, softcap=c["softcap"]))
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "v")]
        out = masked_attention(*leaves, mask, softcap=c["softcap"])
        dq, dk, dv = torch.autograd.grad(out, leaves, st["g"])
        return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)
    cache = KVCache8(st["k_codes"], st["k_scale"], st["v_codes"], st["v_scale"], st["lengths"])
    if c["op"] == "append":
        cache.truncate(st["start"])
        cache.append(st["k"], st["v"])
        return dict(k_codes=cache.k_codes, k_scale=cache.k_scale, v_codes=cache.v_codes, v_scale=cache.v_scale,
                    lengths=cache.lengths)
    if c["fresh"]:
        return dict(out=cache.attend(st["q"], st["k"], st["v"], causal=c["causal"]))
    return dict(out=cache.attend(st["q"], causal=c["causal"]))


# ------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    c = case
    st = prepare(case, seed)
    dev = st["lengths"].device if "lengths" in st else st["q"].device
    if c["op"] == "norm_rope":
        return _exact_norm_rope(c, st)
    if c["op"] == "append":
        return _exact_append(c, st)
    if c["op"] == "attention":
        r = torch.from_numpy(_visible(c)).to(dev)
        return _exact_attention(c, st["q"], st["k"].double(), st["v"].double(), r[..., 0], r[..., 1], c["softcap"],
                                st.get("g"))
    out = []
    for b in range(c["B"]):  # keys held, then the fresh ones: one run of keys for each sequence
        n, Sq = int(st["lengths"][b]), c["Sq"]
        k, v = [(st[x + "_codes"][b, :, :n].double() * st[x + "_scale"][b].double().repeat_interleave(BLOCK, 1)[:, :n, None])
                for x in ("k", "v")]
        first = n - Sq
        if c["fresh"]:
            k, v, first = torch.cat([k, st["k"][b].double()], 1), torch.cat([v, st["v"][b].double()], 1), n
        total = k.shape[1]
        hi = (torch.arange(Sq, device=dev) + first + 1).clamp(0, total) if c["causal"] else torch.full((Sq,), total, device=dev)
        out.append(_exact_attention(c, st["q"][b:b + 1], k[None], v[None], torch.zeros_like(hi)[None], hi[None], 0.0, None)["out"])
    return dict(out=torch.cat(out))


def _exact_append(c, st):
    """Sequence by sequence and block by block of tokens; a code is the nearest of 8 * 2^e / 8 .. 15 * 2^e / 8."""
    def code(v):
        e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(-6, 8)
        return torch.round(v * torch.exp2(3 - e)) * torch.exp2(e - 3)

    res = dict(lengths=None)
    for x in ("k", "v"):
        codes, scale, new = st[x + "_codes"].double(), st[x + "_scale"].double(), st[x].double()
        for b in range(c["B"]):
            n0 = int(st["start"][b])
            n1 = n0 + c["n"]
            for t in range(n0 // BLOCK, (n1 - 1) // BLOCK + 1):
                i0, i1 = max(t * BLOCK, n0), min(t * BLOCK + BLOCK, n1)
                part = new[b, :, i0 - n0:i1 - n0]
                most = part.abs().amax((1, 2))
                s = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
                s = torch.where(most > 448.0 * s, 2 * s, torch.where(most <= 224.0 * s, s / 2, s))
                s = torch.maximum(torch.where(most > 0, s, torch.zeros_like(s)), scale[b, :, t])
                inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))[:, None, None]
                held = codes[b, :, t * BLOCK:i0] * scale[b, :, t, None, None]
                codes[b, :, t * BLOCK:i0] = code(held * inv)
                codes[b, :, i0:i1] = code(part * inv)
                scale[b, :, t] = s
        res[x + "_codes"], res[x + "_scale"] = codes, scale
    return res


def _exact_norm_rope(c, st):
    T, h, w = _grid(c)
    dev = st["q"].device
    s = torch.arange(c["T"] * c["h"] * c["w"], device=dev) + c["start"]
    place = [torch.div(s, h * w, rounding_mode="floor"), torch.div(s, w, rounding_mode="floor") % h, s % w]
    turn, at = [], 0
    for x, n, dim in zip(place, (T, h, w), _axis_dims(c["D"])):  # unit complex numbers from the tables given
        m = n * (dim // 2)
        tab = torch.complex(st["tables"][at:at + m].double(), st["tables"][at + m:at + 2 * m].double())
        turn.append(tab.view(n, dim // 2)[x])
        at += 2 * m
    turn = torch.cat(turn, -1)
    res = {}
    for n in ("q", "k"):
        x, wt = st[n].double(), st["w" + n].double()
        rms = ((x ** 2).mean(-1, keepdim=True) + EPS).sqrt()
        y = x / rms * wt
        z = torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous()) * turn
        res[n] = torch.view_as_real(z).flatten(-2)
        if c["train"]:
            g = torch.view_as_complex(st["g" + n].double().unflatten(-1, (-1, 2)).contiguous()) * turn.conj()
            g = torch.view_as_real(g).flatten(-2)
            u = x / rms
            res["dw" + n] = (g * u).sum((0, 1, 2))
            gw = g * wt
            res["d" + n] = (gw - u * (gw * u).mean(-1, keepdim=True)) / rms
    return res


def _exact_attention(c, q, k, v, lo, hi, softcap, grad):
    """Head by head, in row pieces, in 64 bits; k and v are in 64 bits already."""
    B, H, Sq, D = q.shape
    G = H // k.shape[1]
    names = ("out",) if grad is None else ("out", "dq", "dk", "dv")
    res = dict(out=torch.zeros(q.shape, dtype=torch.float64, device=q.device))
    if grad is not None:
        res.update(dq=torch.zeros_like(res["out"]), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    j = torch.arange(k.shape[2], device=q.device)
    step = max(1, int(2.5e8) // max(1, k.shape[2]))
    for b in range(B):
        for i0 in range(0, Sq, step):
            rows = slice(i0, min(Sq, i0 + step))
            see = (j[None] >= lo[b, rows, None]) & (j[None] < hi[b, rows, None])
            some = see.any(-1, keepdim=True)
            for h in range(H):
                qh = q[b, h, rows].double() / math.sqrt(D)
                kh, vh = k[b, h // G], v[b, h // G]
                z = qh @ kh.T
                th = torch.tanh(z / softcap) if softcap else None
                z = softcap * th if softcap else z
                w = torch.softmax(z.masked_fill(~see & some, -math.inf), -1) * some
                o = w @ vh
                res["out"][b, h, rows] = o
                if grad is not None:
                    gh = grad[b, h, rows].double()
                    res["dv"][b, h // G] += w.T @ gh
                    dz = w * (gh @ vh.T - (gh * o).sum(-1, keepdim=True))
                    dz = dz * (1 - th ** 2) if softcap else dz
                    res["dq"][b, h, rows] = dz @ kh / math.sqrt(D)
                    res["dk"][b, h // G] += dz.T @ qh
    return {n: res[n] for n in names}
