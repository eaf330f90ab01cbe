"""The dense side of the attention hook against its definitions in 64 bits: q/k norm with rotary positions,
attention over key intervals, and the 8-bit key/value cache.

Tolerances count roundings.  A rounding to type t is off by at most half a step, u = finfo(t).eps / 2 of the
value.  fp32 arithmetic adds a little: sums of at most a few thousand terms in fp32 are off by less than
2^-14 of the sum of the terms' sizes (n * 2^-24 for n <= 1024 in the worst order; the orders used are far
better), which the bounds below give as SLACK.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SLACK = 2.0 ** -14


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rand(shape, dtype, seed, device, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def check(got, ref, bound):
    """|got - ref| <= bound everywhere (all in 64 bits)."""
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    over = (got - ref).abs() - bound
    assert bool((over <= 0).all()), f"worst excess {over.max().item():.3e} of bound at {over.argmax().item()}"


# ------------------------------------------------------------------------------- q/k norm + rotary positions
def rope_of(grid, D, device):
    from longcat_video.models.rope_3d import RopeTables

    return RopeTables(grid, D, device)


def turns(rope, start, S):
    """[S, D / 2] complex turns of the tokens, in 64 bits, from the fp32 tables."""
    tables, dims, (T, H, W) = rope.native_args()
    t = tables.double()
    s = torch.arange(start, start + S, device=t.device)
    place = (s // (H * W), (s // W) % H, s % W)
    out, at = [], 0
    for x, n, d in zip(place, (T, H, W), dims):
        m = n * (d // 2)
        out.append(torch.complex(t[at:at + m], t[at + m:at + 2 * m]).view(n, d // 2)[x])
        at += 2 * m
    return torch.cat(out, -1)


def ref_norm_rope(x, w, eps, turn):
    y = x
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w
    if turn is not None:
        y = torch.view_as_real(torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    return y


NORM_ROPE = [  # B, H, Hk, grid, start, S, D
    (1, 1, 1, (1, 1, 1), 0, 1, 128),
    (2, 5, 5, (2, 3, 7), 0, 42, 64),
    (1, 6, 2, (3, 5, 9), 45, 90, 128),
    (2, 3, 1, (2, 4, 8), 7, 33, 40),
    (1, 2, 2, (4, 6, 10), 0, 240, 80),
    (1, 9, 3, (1, 13, 17), 0, 221, 8),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,grid,start,S,D", NORM_ROPE)
def test_norm_rope(cuda, dtype, B, H, Hk, grid, start, S, D):
    from longcat_video.models.rope_3d import qk_norm_rope

    qkv = rand((B, S, H + 2 * Hk, D), dtype, 1, cuda)
    q, k = qkv[:, :, :H].transpose(1, 2), qkv[:, :, H:H + Hk].transpose(1, 2)
    wq, wk = 1 + 0.2 * rand((D,), torch.float32, 2, cuda), 1 + 0.2 * rand((D,), torch.float32, 3, cuda)
    rope = rope_of(grid, D, cuda)
    turn = turns(rope, start, S)
    for use_w, use_r in ((True, True), (True, False), (False, True)):
        a, b = (wq, wk) if use_w else (None, None)
        got = qk_norm_rope(q, k, a, b, 1e-6, rope=rope if use_r else None, start=start)
        for g, x, w in zip(got, (q, k), (a, b)):
            ref = ref_norm_rope(x.double(), w.double() if use_w else None, 1e-6, turn if use_r else None)
            # one rounding, and a few fp32 steps on the pair's larger value
            big = ref.abs().amax(-1, keepdim=True)
            check(g, ref, unit(dtype) * ref.abs() + 2.0 ** -20 * big + 2.0 ** -24 * (dtype == torch.float16))
    alone = qk_norm_rope(q, None, wq, rope=rope, start=start)
    assert torch.equal(alone, qk_norm_rope(q, k, wq, wk, rope=rope, start=start)[0])


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_norm_rope_weight_types(cuda, wdtype):
    from longcat_video.models.rope_3d import qk_norm_rope

    q, k = rand((1, 2, 9, 64), torch.bfloat16, 1, cuda), rand((1, 1, 9, 64), torch.bfloat16, 2, cuda)
    wq, wk = rand((64,), wdtype, 3, cuda), rand((64,), torch.float32, 4, cuda)  # one type, and two
    for ws in ((wq, wk), (wq, wk.to(wdtype))):
        for g, x, w in zip(qk_norm_rope(q, k, *ws), (q, k), ws):
            ref = ref_norm_rope(x.double(), w.double(), 1e-6, None)
            check(g, ref, unit(torch.bfloat16) * ref.abs() + 2.0 ** -20 * ref.abs().amax())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,grid,start,S,D", NORM_ROPE)
def test_norm_rope_gradients(cuda, dtype, B, H, Hk, grid, start, S, D):
    from longcat_video.models.rope_3d import qk_norm_rope

    x = [rand((B, S, n, D), dtype, 1 + i, cuda).transpose(1, 2).requires_grad_() for i, n in enumerate((H, Hk))]
    w = [(1 + 0.2 * rand((D,), torch.float32, 3 + i, cuda)).requires_grad_() for i in range(2)]
    g = [rand((B, n, S, D), dtype, 5 + i, cuda) for i, n in enumerate((H, Hk))]
    rope = rope_of(grid, D, cuda)
    out = qk_norm_rope(*x, *w, 1e-6, rope=rope, start=start)
    got = torch.autograd.grad(out, (*x, *w), g)
    turn = turns(rope, start, S)
    xd = [t.detach().double().requires_grad_() for t in x]
    wd = [t.detach().double().requires_grad_() for t in w]
    ref = torch.autograd.grad([ref_norm_rope(a, b, 1e-6, turn) for a, b in zip(xd, wd)], (*xd, *wd),
                              [t.double() for t in g])
    for a, b in zip(got[:2], ref[:2]):  # a difference of two terms of the row's size
        check(a, b, unit(dtype) * b.abs() + 2.0 ** -19 * b.abs().amax(-1, keepdim=True).clamp(min=1.0)
              + 2.0 ** -24 * (dtype == torch.float16))
    for a, b, xi, gi in zip(got[2:], ref[2:], x, g):  # sums over tokens and heads: against the terms' sizes
        size = (ref_norm_rope(xi.detach().double(), torch.ones(D, device=cuda).double(), 1e-6, None).abs()
                * ref_norm_rope(gi.double(), None, 0, turn.conj()).abs()).sum((0, 1, 2))
        check(a, b, SLACK * size)


def test_norm_rope_gradient_against_differences(cuda):
    from longcat_video.models.rope_3d import qk_norm_rope

    rope = rope_of((1, 2, 3), 16, cuda)
    x = rand((1, 1, 6, 16), torch.float32, 1, cuda).requires_grad_()
    w = (1 + 0.1 * rand((16,), torch.float32, 2, cuda)).requires_grad_()
    g = rand((1, 1, 6, 16), torch.float32, 3, cuda)
    dx, dw = torch.autograd.grad(qk_norm_rope(x, None, w, rope=rope), (x, w), g)
    f = lambda a, b: (qk_norm_rope(a, None, b, rope=rope).double() * g.double()).sum()  # noqa: E731
    h = 2.0 ** -8  # differences of fp32 results: h^2 of curvature, 2^-24 / h of rounding, for 96 terms
    with torch.no_grad():
        for t, d, at in ((x, dx, (0, 0, 4, 5)), (x, dx, (0, 0, 0, 0)), (w, dw, (7,))):
            step = torch.zeros_like(t)
            step[at] = h
            a = (f(x + step, w) - f(x - step, w)) if t is x else (f(x, w + step) - f(x, w - step))
            assert abs((a / (2 * h)).item() - d[at].item()) < 2e-3


def test_norm_rope_partial_gradients_and_repeats(cuda):
    """Only k's gradient asked for, a broadcast input, and the same bits twice."""
    from longcat_video.models.rope_3d import qk_norm_rope

    q = rand((1, 4, 50, 64), torch.bfloat16, 1, cuda)
    k1 = rand((1, 1, 50, 64), torch.bfloat16, 2, cuda).requires_grad_()
    w = torch.ones(64, device=cuda, requires_grad=True)
    rope = rope_of((1, 5, 10), 64, cuda)
    res = []
    for _ in range(2):
        qo, ko = qk_norm_rope(q, k1.expand(1, 4, 50, 64), None, w, rope=rope)
        res.append(torch.autograd.grad(ko.float().square().sum(), (k1, w)))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    assert torch.isfinite(res[0][0]).all() and not qo.isnan().any()


def test_norm_rope_refusals(cuda):
    from longcat_video.models.rope_3d import qk_norm_rope

    x = rand((1, 2, 6, 64), torch.bfloat16, 1, cuda)
    w = torch.ones(64, device=cuda)
    rope = rope_of((1, 2, 3), 64, cuda)
    for kw in (dict(), dict(rope=rope, start=1), dict(rope=rope, start=-1), dict(rope=rope_of((1, 2, 2), 64, cuda)),
               dict(rope=rope_of((1, 2, 3), 128, cuda)), dict(q_weight=w[:32]), dict(q_weight=w, eps=-1.0),
               dict(q_weight=w, eps=float("nan")), dict(k_weight=w)):
        with pytest.raises(ValueError):
            qk_norm_rope(x, **kw)
    for bad in (x.double(), x[0], x.cpu(), rand((1, 1, 6, 136), torch.bfloat16, 1, cuda),
                rand((1, 1, 6, 12), torch.bfloat16, 1, cuda)):
        with pytest.raises(ValueError):
            qk_norm_rope(bad, q_weight=torch.ones(bad.shape[-1], device=bad.device))
    with pytest.raises(ValueError):
        qk_norm_rope(x, x[:, :, :3], w, w)
    assert qk_norm_rope(x[:, :, :0], q_weight=w).shape == (1, 2, 0, 64)


# ------------------------------------------------------------------------------------------ dense attention
def ref_attention(q, k, v, lo, hi, scale, cap=0.0):
    """64 bits: out, lse, sum p |v|, p.  lo, hi [B or 1, Sq]."""
    B, H, Sq, D = q.shape
    G = H // k.shape[1]
    k, v = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    z = q.double() @ k.transpose(-1, -2) * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    j = torch.arange(k.shape[2], device=q.device)
    see = ((j >= lo[..., None]) & (j < hi[..., None]))[:, None]
    z = torch.where(see, z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(z, -1) if k.shape[2] else torch.full(z.shape[:-1], -math.inf, device=q.device).double()
    p = torch.where(see, torch.exp(z - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None]),
                    torch.zeros_like(z))
    return p @ v, lse, p @ v.abs(), p


def check_attention(out, lse, ref, dtype, p_unit=None):
    o, l, size, _ = ref
    u = unit(dtype)
    # P rounded once, the output once, fp32 around them
    check(out, o, (u if p_unit is None else p_unit) * size + u * o.abs() + SLACK * size + 2.0 ** -24)
    if lse is not None:
        assert torch.equal(lse == -math.inf, l == -math.inf)
        fin = l != -math.inf
        check(lse[fin], l[fin], 2.0 ** -16 * (1 + l[fin].abs()))


def rows_of(mask):
    return mask.ranges[..., 0].long(), mask.ranges[..., 1].long()


def full(Sq, Sk, device):
    z = torch.zeros((1, Sq), dtype=torch.long, device=device)
    return z, z + Sk


SHAPES = [  # B, H, Hk, Sq, Sk, D
    (1, 1, 1, 1, 1, 128),
    (2, 4, 2, 1, 300, 128),
    (1, 2, 1, 129, 127, 64),
    (2, 6, 2, 77, 1001, 128),
    (1, 3, 3, 300, 257, 40),
    (1, 2, 2, 513, 640, 80),
    (3, 2, 1, 256, 128, 8),
    (1, 40, 8, 260, 390, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", SHAPES)
def test_attention_shapes(cuda, dtype, B, H, Hk, Sq, Sk, D):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, k, v = rand((B, H, Sq, D), dtype, 1, cuda), rand((B, Hk, Sk, D), dtype, 2, cuda), rand((B, Hk, Sk, D), dtype, 3, cuda)
    scale = 1 / math.sqrt(D)
    out, lse = masked_attention(q, k, v, return_lse=True)
    check_attention(out, lse, ref_attention(q, k, v, *full(Sq, Sk, cuda), scale), dtype)
    mask = AttentionMask.build(Sq, Sk, causal=True, device=cuda)
    out, lse = masked_attention(q, k, v, mask, softcap=2.0, sm_scale=0.3, return_lse=True)
    check_attention(out, lse, ref_attention(q, k, v, *rows_of(mask), 0.3, 2.0), dtype)


def build_rows(Sq, Sk, causal, prefix, qo=None, ko=None, ql=None, kl=None):
    """The mask's definition, row by row, for one batch entry."""
    docs = list(zip(qo, qo[1:], ko, ko[1:])) if qo else [(0, Sq if ql is None else ql, 0, Sk if kl is None else kl)]
    rows = [(0, 0)] * Sq
    for d, (qs, qe, ks, ke) in enumerate(docs):
        n = ke - ks
        for i in range(qs, qe):
            a = i - qs + n - (qe - qs)
            pre = prefix[d] if isinstance(prefix, list) else prefix
            seen = min(max(pre if 0 < pre and a < pre else a + 1 if causal else n, 0), n)
            rows[i] = (ks, ks + seen) if seen else (0, 0)
    return rows


MASKS = [
    dict(Sq=1, Sk=1, causal=True, prefix=0),
    dict(Sq=300, Sk=300, causal=True, prefix=0),
    dict(Sq=300, Sk=200, causal=True, prefix=0),  # the first rows see nothing
    dict(Sq=200, Sk=333, causal=True, prefix=40),
    dict(Sq=333, Sk=333, causal=False, prefix=100),
    dict(Sq=290, Sk=310, causal=False, prefix=0, qo=[0, 1, 1, 130, 260], ko=[5, 5, 20, 200, 290]),
    dict(Sq=290, Sk=290, causal=True, prefix=[3, 50, 0], qo=[10, 20, 148, 280], ko=[10, 20, 148, 280]),
]


@pytest.mark.parametrize("c", MASKS)
def test_mask_rows(cuda, c):
    from longcat_video.models.masked_attention import AttentionMask

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda) if x is not None else None  # noqa: E731
    prefix = i32(c["prefix"]) if isinstance(c["prefix"], list) else c["prefix"]
    m = AttentionMask.build(c["Sq"], c["Sk"], causal=c["causal"], prefix=prefix, q_offsets=i32(c.get("qo")),
                            k_offsets=i32(c.get("ko")), device=cuda)
    rows = build_rows(**c)
    assert m.ranges[0].tolist() == [list(r) for r in rows]
    for t in range(0, c["Sq"], 128):
        part = rows[t:t + 128]
        some = [r for r in part if r[0] < r[1]]
        x, y, z, w = m.table[0, t // 128].tolist()
        if some:
            assert (x, y) == (min(r[0] for r in some), max(r[1] for r in some))
        else:
            assert x >= y
        assert (z, w) == (max(r[0] for r in part), min(r[1] for r in part))
    again = AttentionMask.from_ranges(m.ranges, c["Sk"])
    assert torch.equal(again.ranges, m.ranges) and torch.equal(again.table, m.table)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c", MASKS)
def test_attention_masks(cuda, dtype, c):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    m = AttentionMask.from_ranges(torch.tensor([build_rows(**c)], dtype=torch.int32, device=cuda), c["Sk"])
    q, k, v = (rand((2, n, s, 64), dtype, i, cuda) for i, (n, s) in enumerate(((4, c["Sq"]), (2, c["Sk"]), (2, c["Sk"]))))
    for cap in (0.0, 5.0):
        out, lse = masked_attention(q * 3, k, v, m, softcap=cap, return_lse=True)
        check_attention(out, lse, ref_attention(q * 3, k, v, *rows_of(m), 0.125, cap), dtype)


def test_attention_padded_batch(cuda):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    kl, ql = [0, 1, 128, 129, 300], [7, 150, 0, 150, 1]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q, k, v = (rand((5, 2, s, 128), torch.bfloat16, i, cuda) for i, s in enumerate((150, 300, 300)))
    for kw in (dict(k_lengths=i32(kl)), dict(k_lengths=i32(kl), q_lengths=i32(ql), causal=True),
               dict(q_lengths=i32(ql), prefix=i32([0, 5, 9, 200, 1]))):
        m = AttentionMask.build(150, 300, **kw)
        pre = kw["prefix"].tolist() if "prefix" in kw else [0] * 5
        for b in range(5):
            want = build_rows(150, 300, kw.get("causal", False), pre[b], ql=ql[b] if "q_lengths" in kw else None,
                              kl=kl[b] if "k_lengths" in kw else None)
            assert m.ranges[b].tolist() == [list(r) for r in want]
        out, lse = masked_attention(q, k, v, m, return_lse=True)
        check_attention(out, lse, ref_attention(q, k, v, *rows_of(m), 128 ** -0.5), torch.bfloat16)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_places_hold_anything(cuda, bad):
    """Keys and values behind the padded length, and scores of the type's lowest value."""
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, k, v = (rand((2, 2, s, 64), torch.bfloat16, i, cuda) for i, s in enumerate((200, 400, 400)))
    lens = torch.tensor([130, 255], dtype=torch.int32, device=cuda)
    m = AttentionMask.build(200, 400, k_lengths=lens)
    want = masked_attention(q, k, v, m)
    for b, n in enumerate(lens.tolist()):
        k[b, :, n:], v[b, :, n:] = bad, bad
    assert torch.equal(masked_attention(q, k, v, m), want)
    # a key whose scores overflow to -inf weighs nothing
    k2 = k[:, :, :130].clone()
    q2 = q.abs()
    k2[:, :, 5] = -torch.finfo(torch.bfloat16).max
    o, lse = masked_attention(q2, k2, v[:, :, :130].nan_to_num(0, 0, 0), return_lse=True)
    assert torch.isfinite(o.float()).all() and torch.isfinite(lse).all()


def test_attention_large_scores_and_late_maximum(cuda):
    """A maximum that rises by more than 2^8 late in the row, in every key tile."""
    from longcat_video.models.masked_attention import masked_attention

    q = rand((1, 2, 130, 64), torch.float16, 1, cuda)
    k = rand((1, 2, 700, 64), torch.float16, 2, cuda)
    k = k * torch.linspace(0.2, 12, 700, device=cuda)[:, None].half()
    v = rand((1, 2, 700, 64), torch.float16, 3, cuda)
    out, lse = masked_attention(q, k, v, sm_scale=1.0, return_lse=True)
    ref = ref_attention(q, k, v, *full(130, 700, cuda), 1.0)
    o, l, size, _ = ref
    # scores near 300: their fp32 error, 2^-23 of the size of the products' sum, is an error of the weights
    zsize = (q.double().abs() @ k.double().abs().transpose(-1, -2)).amax()
    check(out, o, (2 * unit(torch.float16) + SLACK + 2.0 ** -22 * zsize) * size + 2.0 ** -24)
    check(lse, l, 2.0 ** -16 * (1 + l.abs()))


def test_attention_views_streams_and_out(cuda):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    B, N, H, D = 2, 210, 3, 128
    qkv = rand((B, N, 3, H, D), torch.bfloat16, 1, cuda)
    q, k, v = qkv.permute(2, 0, 3, 1, 4)
    m = AttentionMask.build(N, N, prefix=50, device=cuda)
    want = masked_attention(q.contiguous(), k.contiguous(), v.contiguous(), m)
    assert torch.equal(masked_attention(q, k, v, m), want)
    out = torch.empty((B, N, H, D), dtype=torch.bfloat16, device=cuda)
    got = masked_attention(q, k, v, m, out=out.permute(0, 2, 1, 3))
    assert torch.equal(got, want) and torch.equal(out.permute(0, 2, 1, 3), want)
    odd = torch.empty((B, H, N, D + 1), dtype=torch.bfloat16, device=cuda)[..., 1:]  # not 16-byte aligned
    assert torch.equal(masked_attention(odd.copy_(q), k, v, m, out=odd), want)
    assert torch.equal(masked_attention(q, k[:, :, ::2], v[:, :, ::2]),
                       masked_attention(q, k[:, :, ::2].contiguous(), v[:, :, ::2].contiguous()))
    one = masked_attention(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))
    assert torch.equal(one, masked_attention(q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = masked_attention(q, k, v, m)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, want)


def test_attention_from_fresh_threads(cuda):
    """A host thread whose first CUDA work is this call (an autograd worker is one)."""
    import threading

    from longcat_video.models.masked_attention import masked_attention

    q = rand((1, 2, 130, 64), torch.bfloat16, 1, cuda)
    g = rand(q.shape, torch.bfloat16, 2, cuda)
    want = gradients(q, q, q, g, None)
    res, outs = {}, [torch.empty_like(q) for _ in range(4)]

    def work(i):
        try:
            res[i] = masked_attention(q, q, q, out=outs[i])
        except Exception as e:  # noqa: BLE001
            res[i] = e

    for i in range(4):
        t = threading.Thread(target=work, args=(i,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(res[i], want[0]) for i in range(4))


def test_attention_graph_replay(cuda):
    """Captured with its mask: replays follow new lengths and inputs."""
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, k, v = (rand((2, 2, s, 64), torch.bfloat16, i, cuda) for i, s in enumerate((3, 900, 900)))
    lens = torch.tensor([900, 100], dtype=torch.int32, device=cuda)
    masked_attention(q, k, v, AttentionMask.build(3, 900, causal=True, k_lengths=lens))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = masked_attention(q, k, v, AttentionMask.build(3, 900, causal=True, k_lengths=lens))
    for new in ([1, 2], [900, 511], [0, 130]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(rand(q.shape, torch.bfloat16, sum(new), cuda))
        g.replay()
        assert torch.equal(out, masked_attention(q, k, v, AttentionMask.build(3, 900, causal=True, k_lengths=lens)))


def ref_gradients(q, k, v, g, lo, hi, scale, cap):
    """(dq, dk, dv) in 64 bits, and for each the sum of the sizes of its terms."""
    B, H, Sq, D = q.shape
    G = H // k.shape[1]
    o, lse, _, p = ref_attention(q, k, v, lo, hi, scale, cap)
    qd, gd = q.double(), g.double()
    kd, vd = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    t = torch.tanh(qd @ kd.transpose(-1, -2) * scale / cap) if cap else torch.zeros((), device=q.device).double()
    dp = gd @ vd.transpose(-1, -2)
    delta = (gd * o).sum(-1, keepdim=True)
    pt = p * (1 - t * t)
    ds = pt * (dp - delta)
    # what a rounding of p, ds or o can be relative to: ds itself, and delta's error by the rounding of o
    loose = (gd.abs() * o.abs()).sum(-1, keepdim=True)
    share = lambda x: x.view(B, H // G, G, *x.shape[2:]).sum(2)  # noqa: E731
    grads = (ds @ kd * scale, share(ds.transpose(-1, -2) @ qd) * scale, share(p.transpose(-1, -2) @ gd))
    sizes = lambda d: (d @ kd.abs() * scale, share(d.transpose(-1, -2) @ qd.abs()) * scale)  # noqa: E731
    fine = pt * ((gd.abs() @ vd.abs().transpose(-1, -2)) + loose)  # fp32 error is relative to this
    return grads, sizes(ds.abs()), sizes(pt * loose), sizes(fine), share(p.transpose(-1, -2) @ gd.abs())


def check_gradients(got, q, k, v, g, lo, hi, scale, cap=0.0):
    grads, ds, dl, fine, pg = ref_gradients(q, k, v, g, lo, hi, scale, cap)
    u = unit(q.dtype)
    tiny = 2.0 ** -24  # fp16 terms may be subnormal: p and ds are rounded to steps of 2^-24 there, over the row
    for i in range(2):
        n = q.shape[2] if i else k.shape[2]
        x = (q if i else k).double().abs().amax() * scale * n * tiny * (q.dtype == torch.float16)
        check(got[i], grads[i], u * grads[i].abs() + u * ds[i] + u * dl[i] + SLACK * fine[i] + x + tiny)
    x = g.double().abs().amax() * q.shape[2] * (q.shape[1] // k.shape[1]) * tiny * (q.dtype == torch.float16)
    check(got[2], grads[2], u * grads[2].abs() + (u + SLACK) * pg + x + tiny)


def gradients(q, k, v, g, m, **kw):
    from longcat_video.models.masked_attention import masked_attention

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = masked_attention(*leaves, m, **kw)
    return out, torch.autograd.grad(out, leaves, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", SHAPES)
def test_attention_gradients(cuda, dtype, B, H, Hk, Sq, Sk, D):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, g = (rand((B, Sq, H, D), dtype, i, cuda).transpose(1, 2) for i in (1, 4))
    k, v = rand((B, Hk, Sk, D), dtype, 2, cuda), rand((B, Hk, Sk, D), dtype, 3, cuda)
    out, got = gradients(q, k, v, g, None)
    assert torch.equal(out, masked_attention(q, k, v))
    check_gradients(got, q, k, v, g, *full(Sq, Sk, cuda), 1 / math.sqrt(D))
    m = AttentionMask.build(Sq, Sk, causal=True, prefix=5, device=cuda)
    _, got = gradients(q, k, v, g, m, softcap=1.5, sm_scale=0.3)
    check_gradients(got, q, k, v, g, *rows_of(m), 0.3, 1.5)


@pytest.mark.parametrize("c", MASKS)
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_attention_mask_gradients(cuda, c, cap):
    from longcat_video.models.masked_attention import AttentionMask

    m = AttentionMask.from_ranges(torch.tensor([build_rows(**c)], dtype=torch.int32, device=cuda), c["Sk"])
    q, k, v, g = (rand((2, n, s, 128), torch.bfloat16, i, cuda)
                  for i, (n, s) in enumerate(((4, c["Sq"]), (2, c["Sk"]), (2, c["Sk"]), (4, c["Sq"]))))
    _, got = gradients(q, k, v, g, m, softcap=cap)
    check_gradients(got, q, k, v, g, *rows_of(m), 128 ** -0.5, cap)
    _, again = gradients(q, k, v, g, m, softcap=cap)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_gradients_of_a_padded_batch(cuda, bad, cap):
    """Padding of queries, keys and the gradient may hold anything; its own gradients are zeros."""
    from longcat_video.models.masked_attention import AttentionMask

    ql, kl = [200, 131, 0, 5], [130, 255, 300, 0]
    q, k, v, g = (rand((4, n, s, 64), torch.float16, i, cuda)
                  for i, (n, s) in enumerate(((4, 200), (2, 300), (2, 300), (4, 200))))
    m = AttentionMask.build(200, 300, q_lengths=torch.tensor(ql, dtype=torch.int32, device=cuda),
                            k_lengths=torch.tensor(kl, dtype=torch.int32, device=cuda))
    out, want = gradients(q, k, v, g, m, softcap=cap)
    check_gradients(want, q, k, v, g, *rows_of(m), 0.125, cap)
    for b in range(4):
        q[b, :, ql[b]:], g[b, :, ql[b]:], k[b, :, kl[b]:], v[b, :, kl[b]:] = bad, bad, bad, bad
    out2, got = gradients(q, k, v, g, m, softcap=cap)
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(want, got))
    for b in range(4):
        assert (got[0][b, :, ql[b]:] == 0).all() and (got[1][b, :, kl[b]:] == 0).all() and (got[2][b, :, kl[b]:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hk,S", [(2, 2, 1), (4, 1, 7), (2, 1, 130), (1, 1, 500)])
def test_short_gradients_round_once(cuda, dtype, H, Hk, S):
    """Few steps: p and ds keep twice their type's bits, so that dv and, but for delta's share, dq and dk round once."""
    from longcat_video.models.masked_attention import AttentionMask

    q, k, v, g = (rand((2, n, S, 64), dtype, i, cuda) for i, n in enumerate((H, Hk, Hk, H)))
    m = AttentionMask.build(S, S, causal=True, device=cuda)
    _, got = gradients(q, k, v, g, m)
    grads, ds, dl, fine, pg = ref_gradients(q, k, v, g, *rows_of(m), 0.125, 0.0)
    u = unit(dtype)
    tiny = 2.0 ** -24  # steps of fp16's subnormals, of the result and of what a rounding leaves over
    for i in range(2):
        x = (q if i else k).double().abs().amax() * 0.125 * S * H * tiny
        check(got[i], grads[i], u * grads[i].abs() + u * u * ds[i] + u * dl[i] + SLACK * fine[i] + x + tiny)
    # p is raised by 2^15 in fp16, and bf16 has no subnormals here
    check(got[2], grads[2], u * grads[2].abs() + (u * u + SLACK) * pg + g.double().abs().amax() * S * H * tiny / 2 ** 15 + tiny)


def test_small_gradients_in_fp16(cuda):
    """Products of p and do far below fp16's normal numbers: raised by powers of two, they keep their bits."""
    from longcat_video.models.masked_attention import AttentionMask

    q, k, v = (rand((1, n, s, 64), torch.float16, i, cuda) for i, (n, s) in enumerate(((4, 600), (2, 2000), (2, 2000))))
    g = rand((1, 4, 600, 64), torch.float16, 3, cuda) * 2.0 ** -8
    m = AttentionMask.build(600, 2000, prefix=100, causal=True, device=cuda)
    _, got = gradients(q, k, v, g, m)
    grads, ds, dl, fine, pg = ref_gradients(q, k, v, g, *rows_of(m), 0.125, 0.0)
    u, tiny = unit(torch.float16), 2.0 ** -24
    assert g.float().norm(dim=-1).max() < 2.0 ** -4  # so ds is raised by 2^7 at least (2^7 |do| < 2^3)
    for i in range(2):
        x = (q if i else k).double().abs().amax() * 0.125 * (1200 if i else 2000) * tiny / 2 ** 7
        check(got[i], grads[i], u * grads[i].abs() + u * ds[i] + u * dl[i] + SLACK * fine[i] + x + tiny)
    x = g.double().abs().amax() * 1200 * tiny / 2 ** 15
    check(got[2], grads[2], u * grads[2].abs() + (u + SLACK) * pg + x + tiny)


def test_gradients_of_many_heads(cuda):
    q, k, v, g = (rand((1, n, s, 8), torch.bfloat16, i, cuda)
                  for i, (n, s) in enumerate(((70000, 2), (35000, 3), (35000, 3), (70000, 2))))
    _, got = gradients(q, k, v, g, None)
    check_gradients(got, q, k, v, g, *full(2, 3, cuda), 8 ** -0.5)


def test_attention_gradient_against_differences(cuda):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, k, v, g = (rand((1, 1, 9, 16), torch.float16, i, cuda) for i in range(4))
    m = AttentionMask.build(9, 9, causal=True, device=cuda)
    _, got = gradients(q, k, v, g, m, softcap=3.0)
    f = lambda *a: (masked_attention(*a, m, softcap=3.0).double() * g.double()).sum().item()  # noqa: E731
    for i, at in ((0, (0, 0, 5, 3)), (1, (0, 0, 2, 7)), (2, (0, 0, 0, 1))):
        a, b = [[t.clone() for t in (q, k, v)] for _ in range(2)]
        a[i][at] += 0.25
        b[i][at] -= 0.25
        h = (a[i][at] - b[i][at]).item()
        # 9 rows of fp16 outputs below 4: 2^-11 * 4 * |g| each, twice over h; and h^2 of curvature
        assert abs((f(*a) - f(*b)) / h - got[i][at].item()) < 0.05


def test_attention_partial_gradients(cuda):
    """Only some inputs want gradients; a broadcast key head; a gradient of another type and layout."""
    from longcat_video.models.masked_attention import masked_attention

    q, k, v = (rand((2, n, 140, 64), torch.bfloat16, n, cuda) for n in (4, 2, 2))
    g = rand((2, 4, 140, 64), torch.bfloat16, 9, cuda)
    full_g = gradients(q, k, v, g, None)[1]
    for want in ((0,), (1,), (2,), (0, 2)):
        leaves = [t.detach().requires_grad_(i in want) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(masked_attention(*leaves), [leaves[i] for i in want], g)
        assert all(torch.equal(a, full_g[i]) for a, i in zip(got, want))
    k1 = k[:, :1].detach().requires_grad_()
    a = torch.autograd.grad(masked_attention(q, k1.expand(2, 2, 140, 64), v), k1, g)[0]
    _, (_, dk, _) = gradients(q, k[:, :1].expand(2, 2, 140, 64), v, g, None)
    assert torch.equal(a, dk.sum(1, keepdim=True))
    leaf = q.detach().requires_grad_()
    o = masked_attention(leaf, k, v).float().transpose(1, 2)
    assert torch.equal(torch.autograd.grad(o, leaf, g.float().transpose(1, 2))[0], full_g[0])
    one = torch.autograd.grad(masked_attention(leaf, k, v).sum(), leaf)[0]  # an expanded gradient
    assert torch.equal(one, gradients(q, k, v, torch.ones_like(g), None)[1][0])


def test_training_step_in_a_graph(cuda):
    """Norm, rotation, attention and their gradients, captured on a side stream and replayed."""
    from longcat_video.models.masked_attention import AttentionMask, masked_attention
    from longcat_video.models.rope_3d import qk_norm_rope

    rope = rope_of((2, 5, 14), 64, cuda)
    x = [rand((1, n, 140, 64), torch.bfloat16, n, cuda) for n in (4, 2, 2)]
    w = [torch.ones(64, device=cuda), torch.ones(64, device=cuda)]
    g = rand((1, 4, 140, 64), torch.bfloat16, 9, cuda)

    def step():
        leaves = [t.detach().requires_grad_() for t in (*x, *w)]
        q, k = qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], rope=rope)
        out = masked_attention(q, k, leaves[2], AttentionMask.build(140, 140, prefix=70, device=cuda))
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(3):
        for t in (*x, g):
            t.copy_(rand(t.shape, torch.bfloat16, 50 + i + t.shape[1], cuda))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, step()))


def test_attention_output_refusals(cuda):
    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import masked_attention

    q, k, v = (rand((1, 2, 40, 64), torch.bfloat16, i, cuda) for i in range(3))
    cache = KVCache8.from_kv(k, v)
    for f in (lambda o: masked_attention(q, k, v, out=o), lambda o: cache.attend(q, out=o)):
        wide = torch.empty((1, 2, 41, 64), dtype=torch.bfloat16, device=cuda).flatten()
        q, bad = wide[:q.numel()].view_as(q).copy_(q), wide[64:64 + q.numel()].view_as(q)
        for bad in (bad, torch.empty_like(q).requires_grad_()):
            with pytest.raises(ValueError):
                f(bad)
        o = torch.zeros((1, 2, 40, 64), dtype=torch.bfloat16, device=cuda)
        before = o._version
        assert f(o) is o or f(o).data_ptr() == o.data_ptr()
        assert o._version > before and torch.equal(o, f(None))
        own = q.clone()
        assert f(q) is not None and torch.equal(q, o)  # q itself
        q = own
    with pytest.raises(ValueError):
        masked_attention(q, k, v, out=v)
    w = torch.ones_like(q, requires_grad=True)
    o = torch.zeros_like(q)
    y = (w * o).sum()  # o is saved
    masked_attention(q, k, v, out=o)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("causal", [False, True])
def test_lookup_in_a_long_cache(cuda, causal):
    """Many rows over few tokens of a large cache: what its scratch holds behind them does not count."""
    from longcat_video.models.kv_cache import KVCache8

    k, v = (rand((2, 2, 150, 64), torch.bfloat16, i, cuda) for i in range(2))
    q, fk, fv = (rand((2, n, 200, 64), torch.bfloat16, 3 + i, cuda) for i, n in enumerate((4, 2, 2)))
    short, long = KVCache8.from_kv(k, v), KVCache8.from_kv(k, v, capacity=9000)
    for c in (short, long):
        c.truncate(torch.tensor([150, 70], dtype=torch.int32, device=cuda))
    junk = [torch.full((2, 2, 9200, 64), math.nan, dtype=torch.bfloat16, device=cuda) for _ in range(4)]
    del junk  # the allocator hands these bytes out again
    # The longer one is split along its keys.  Either side is off by a rounding of the result, u |o|, and of the weights,
    # u sum p |v - o| <= 2 u max |v|, so they differ by 6 u max |v| at most.
    top = max(t.abs().max().item() for t in (v, fv))
    for fresh in ((), (fk, fv)):
        torch.testing.assert_close(long.attend(q, *fresh, causal=causal), short.attend(q, *fresh, causal=causal), rtol=0,
                                   atol=6 * unit(torch.bfloat16) * top)


def test_lookup_of_many_heads(cuda):
    """More 16-row tiles than a grid is high: the cache is unpacked."""
    from longcat_video.models.kv_cache import KVCache8

    k, v = (rand((1, 20000, 5, 8), torch.bfloat16, i, cuda) for i in range(2))
    q = rand((1, 20000, 64, 8), torch.bfloat16, 2, cuda)
    got = KVCache8.from_kv(k, v).attend(q)
    part = KVCache8.from_kv(k[:, :50], v[:, :50]).attend(q[:, :50])
    # two kernels: each rounds once (2^-8 of a value of at most max |v|) and weighs with 16-bit numbers (2^-8 again)
    torch.testing.assert_close(got[:, :50].float(), part.float(), rtol=0, atol=4 * 2.0**-8 * v.abs().max().item())


def test_gradient_refusals(cuda):
    """Second derivatives; a capture while an eager graph of the same leaf lives on another stream."""
    from longcat_video.models.masked_attention import masked_attention
    from longcat_video.models.rope_3d import qk_norm_rope

    x = rand((1, 2, 20, 64), torch.bfloat16, 1, cuda).requires_grad_()
    w = torch.ones(64, device=cuda, requires_grad=True)
    for f in (lambda: masked_attention(x, x, x), lambda: qk_norm_rope(x, q_weight=w)):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(f().sum(), x, create_graph=True)
        eager = f()
        with pytest.raises(ValueError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                f()
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = torch.autograd.grad(f(), x, torch.ones_like(x))[0]
        graph.replay()
        assert torch.equal(res, torch.autograd.grad(f(), x, torch.ones_like(x))[0])


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (3,), (0, 3), (1, 2), (2, 3)])
def test_norm_rope_some_gradients(cuda, want):
    """Any part of q, k and their weights, with and without rotation: as when all four are asked for."""
    from longcat_video.models.rope_3d import qk_norm_rope

    x = [rand((2, n, 30, 64), torch.bfloat16, n, cuda) for n in (4, 2)]
    x += [rand((64,), torch.bfloat16, 5 + i, cuda) for i in range(2)]
    g = [rand((2, n, 30, 64), torch.bfloat16, 7 + n, cuda) for n in (4, 2)]
    for rope in (None, rope_of((1, 5, 6), 64, cuda)):
        def grads(want):
            leaves = [t.detach().requires_grad_(i in want) for i, t in enumerate(x)]
            out = qk_norm_rope(*leaves, rope=rope)
            at = [i for i in range(2) if out[i].requires_grad]
            return torch.autograd.grad([out[i] for i in at], [leaves[i] for i in want], [g[i] for i in at])

        full = grads((0, 1, 2, 3))
        for a, i in zip(grads(want), want):
            assert a.dtype == torch.bfloat16
            if i < 2:
                assert torch.equal(a, full[i])
            else:  # rows added up in another order (fp32, 240 terms of at most 16), then one rounding: a bf16 step
                torch.testing.assert_close(a, full[i], rtol=2.0**-7, atol=240 * 240 * 16 * 2.0**-24)


def test_attention_refusals(cuda):
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    q, k = rand((1, 4, 10, 64), torch.bfloat16, 1, cuda), rand((1, 2, 20, 64), torch.bfloat16, 2, cuda)
    m = AttentionMask.build(10, 20, causal=True, device=cuda)
    bad = [(q, k, k[:, :, :5]), (q, k.half(), k.half()), (q.float(), k.float(), k.float()), (q[0], k, k),
           (q[:, :3], k, k), (q, rand((2, 2, 20, 64), torch.bfloat16, 1, cuda), k), (q.cpu(), k, k),
           (q[..., :60], k[..., :60], k[..., :60])]
    for a in bad:
        with pytest.raises(ValueError):
            masked_attention(*a)
    for kw in (dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=float("nan")), dict(softcap=-1.0),
               dict(softcap=float("inf")), dict(mask=AttentionMask.build(10, 21, device=cuda)),
               dict(mask=AttentionMask.from_ranges(torch.zeros((3, 10, 2), dtype=torch.int32, device=cuda), 20)),
               dict(out=q.float())):
        with pytest.raises(ValueError):
            masked_attention(q, k, k, **{"mask": m, **kw})
    i32 = dict(dtype=torch.int32, device=cuda)
    o = torch.tensor([0, 10], **i32)
    for kw in (dict(q_offsets=o), dict(q_offsets=o, k_offsets=o, k_lengths=o), dict(prefix=-1),
               dict(q_offsets=o.long(), k_offsets=o.long()), dict(q_offsets=o, k_offsets=torch.zeros(3, **i32)),
               dict(q_lengths=o, k_lengths=torch.zeros(3, **i32)), dict(q_offsets=o[:1], k_offsets=o[:1])):
        with pytest.raises(ValueError):
            AttentionMask.build(10, 20, **{"device": cuda, **kw})
    e = masked_attention(q, k[:, :, :0], k[:, :, :0], return_lse=True)
    assert (e[0] == 0).all() and (e[1] == -math.inf).all()
    assert masked_attention(q[:, :, :0], k, k).shape == (1, 4, 0, 64)


# ---------------------------------------------------------------------------------------------- 8-bit cache
def scale_of(amax):
    """The smallest power of two s with amax / s <= 448, in 64 bits."""
    amax = amax.double()
    s = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)))
    s = torch.where(amax > 448 * s, 2 * s, torch.where(amax <= 224 * s, s / 2, s))
    return torch.where(amax > 0, s.clamp(min=2.0 ** -126), torch.zeros_like(s))


def code_of(x):
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(-6, 8)
    return (torch.round(x * torch.exp2(3 - e)) * torch.exp2(e - 3)).clamp(-448, 448)


class RefCache:
    """Sequence by sequence, block by block, in 64 bits."""

    def __init__(self, B, H, cap, D, device):
        self.codes = [torch.zeros((B, H, cap, D), dtype=torch.float64, device=device) for _ in range(2)]
        self.scale = [torch.zeros((B, H, cap // 64), dtype=torch.float64, device=device) for _ in range(2)]
        self.lengths = [0] * B

    def append(self, k, v, counts=None):
        for b in range(k.shape[0]):
            n0 = self.lengths[b]
            n1 = min(n0 + (k.shape[2] if counts is None else min(max(counts[b], 0), k.shape[2])), self.codes[0].shape[2])
            for codes, scale, x in zip(self.codes, self.scale, (k, v)):
                for t in range(n0 // 64, -(-n1 // 64)):
                    i0, i1 = max(n0, 64 * t), min(n1, 64 * t + 64)
                    if i0 >= i1:
                        continue
                    part = x[b, :, i0 - n0:i1 - n0].double()
                    amax = torch.where(part.isfinite(), part.abs(), 0.0).amax((1, 2))
                    old = scale[b, :, t] if 64 * t < n0 else torch.zeros_like(scale[b, :, t])
                    s = torch.maximum(old, scale_of(amax))
                    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))[:, None, None]
                    codes[b, :, 64 * t:i0] = code_of(codes[b, :, 64 * t:i0] * old[:, None, None] * inv)
                    codes[b, :, i0:i1] = code_of(part * inv)
                    scale[b, :, t] = s
            self.lengths[b] = max(n0, n1)

    def values(self):
        return [c * s.repeat_interleave(64, 2)[..., None] for c, s in zip(self.codes, self.scale)]


def same(cache, ref):
    assert cache.lengths.tolist() == ref.lengths
    for got, want in zip((cache.k_codes, cache.v_codes), ref.codes):
        assert torch.equal(got.double().nan_to_num(777.0), want.nan_to_num(777.0))
    for got, want in zip((cache.k_scale, cache.v_scale), ref.scale):
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,D,steps", [(1, 1, 128, [1, 1, 62, 1, 200]), (3, 2, 64, [130, 1, 5, 64]), (2, 3, 40, [63, 2, 65])])
def test_cache_append(cuda, dtype, B, H, D, steps):
    from longcat_video.models.kv_cache import KVCache8

    cap = 320
    cache, ref = KVCache8.allocate(B, H, cap, D, cuda), RefCache(B, H, cap, D, cuda)
    for i, n in enumerate(steps):
        x = rand((B, n, 2 * H, D), dtype, i, cuda, scale=3.0 ** i * 1e-2).transpose(1, 2)
        k, v = x[:, :H], x[:, H:] * 0 if i == 0 else x[:, H:]
        counts = torch.tensor([max(0, n - 3 * b) for b in range(B)], dtype=torch.int32, device=cuda) if i == 1 else None
        cache.append(k, v, counts)
        ref.append(k, v, counts.tolist() if counts is not None else None)
        same(cache, ref)
    for got, want in zip(cache.dequantize(torch.bfloat16), ref.values()):
        held = torch.arange(cap, device=cuda)[None] < cache.lengths[:, None]
        assert torch.equal(got.double(), torch.where(held[:, None, :, None], want, 0.0))


@pytest.mark.parametrize("H,steps", [(1, [500, 1, 70]), (2, [60, 200, 3]), (5, [64, 1, 65]), (8, [1, 63, 64, 1]), (16, [1, 1, 2]),
                                     (17, [1, 62, 1])])
def test_cache_append_heads(cuda, H, steps):
    """Few blocks and heads go in one launch, with the lengths; both sides of the border, and counts that run over."""
    from longcat_video import _native
    from longcat_video.models.kv_cache import KVCache8

    cap = 576
    cache, ref = KVCache8.allocate(3, H, cap, 16, cuda), RefCache(3, H, cap, 16, cuda)
    for i, n in enumerate(steps):
        k, v = (rand((3, H, n, 16), torch.bfloat16, 2 * i + j, cuda, scale=2.0 ** i) for j in range(2))
        counts = [n, n // 2, 0] if i else [n] * 3
        cache.append(k, v, torch.tensor(counts, dtype=torch.int32, device=cuda))
        ref.append(k, v, counts)
        same(cache, ref)
    assert _native.device_error() == 0
    cache.truncate(cap - 1)
    k = rand((3, H, 2, 16), torch.bfloat16, 9, cuda)
    cache.append(k, k)  # one fits
    assert cache.lengths.tolist() == [cap] * 3 and _native.device_error(clear=True) != 0
    assert _native.device_error() == 0


def test_cache_extremes(cuda):
    """Largest and smallest values, infinities and NaN, zeros; a full cache; rows behind the last stay."""
    from longcat_video import _native
    from longcat_video.models.kv_cache import KVCache8

    for dtype in (torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        x = rand((1, 4, 64, 32), dtype, 1, cuda)
        x[0, 0] = 0
        x[0, 1, 3, 4], x[0, 1, 9, 9] = info.max, -info.max
        x[0, 2, 0, 0], x[0, 2, 1, 0], x[0, 2, 2, 0] = math.inf, -math.inf, math.nan
        x[0, 3] = x[0, 3].sign() * info.tiny * torch.rand((64, 32), device=cuda).to(dtype)
        cache, ref = KVCache8.allocate(1, 4, 128, 32, cuda), RefCache(1, 4, 128, 32, cuda)
        cache.k_codes.view(torch.uint8)[:, :, 64:] = 17  # behind the tokens
        ref.codes[0][:, :, 64:] = cache.k_codes[:, :, 64:].double()
        cache.append(x, x)
        ref.append(x, x)
        same(cache, ref)
        kd, _ = cache.dequantize(dtype)
        assert kd[:, :, 64:].eq(0).all() and torch.isfinite(kd[:, :2]).all()
    assert _native.device_error(clear=True) == 0
    cache.append(x, x)
    cache.append(x[:, :, :1], x[:, :, :1])  # no room: dropped and reported
    assert cache.lengths.tolist() == [128]
    assert _native.device_error(clear=True) == _native.BSA_ERR_INDEX
    assert _native.device_error() == 0


def test_cache_truncate(cuda):
    from longcat_video.models.kv_cache import KVCache8

    x = rand((2, 1, 200, 64), torch.bfloat16, 1, cuda)
    cache, fresh = KVCache8.from_kv(x, x, 256), KVCache8.from_kv(x[:, :, :64], x[:, :, :64], 256)
    cache.truncate(64)
    y = x[:, :, :100] * 0.01  # the blocks behind hold no token: they take new scales
    cache.append(y, y)
    fresh.append(y, y)
    assert torch.equal(cache.k_codes[:, :, :164].view(torch.uint8), fresh.k_codes[:, :, :164].view(torch.uint8))
    assert torch.equal(cache.k_scale[..., :3], fresh.k_scale[..., :3])
    cache.truncate(torch.tensor([3, 0], dtype=torch.int32, device=cuda))
    assert cache.lengths.tolist() == [3, 0]


def cache_of(B, Hk, cap, D, lens, dtype, device, seed=1):
    from longcat_video.models.kv_cache import KVCache8

    cache = KVCache8.allocate(B, Hk, cap, D, device)
    x = rand((2, B, Hk, max(max(lens), 1), D), dtype, seed, device)
    cache.append(x[0], x[1], torch.tensor(lens, dtype=torch.int32, device=device))
    # what lies behind the tokens may be anything
    for codes in (cache.k_codes, cache.v_codes):
        for b, n in enumerate(lens):
            codes.view(torch.uint8)[b, :, n:] = 0x7F  # NaN
    return cache


def ref_cache_attention(cache, q, causal, scale, k=None, v=None):
    """Sequence by sequence: (out, lse, size)."""
    outs, sizes = [], []
    for b, n in enumerate(cache.lengths.tolist()):
        kb, vb = (c[b:b + 1, :, :n].double() * s[b:b + 1].double().repeat_interleave(64, 2)[:, :, :n, None]
                  for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))
        if k is not None:
            kb, vb = torch.cat([kb, k[b:b + 1].double()], 2), torch.cat([vb, v[b:b + 1].double()], 2)
        Sq, Sk = q.shape[2], kb.shape[2]
        hi = torch.full((1, Sq), Sk, device=q.device)
        if causal:
            hi = (torch.arange(Sq, device=q.device)[None] + Sk - Sq + 1).clamp(0, Sk)
        o, _, size, _ = ref_attention(q[b:b + 1], kb, vb, torch.zeros_like(hi), hi, scale)
        outs.append(o)
        sizes.append(size)
    return torch.cat(outs), torch.cat(sizes)


CACHE_CASES = [  # Hk, G, Sq, D, lengths
    (1, 1, 1, 128, [1]),
    (2, 4, 1, 128, [0, 1, 63, 64, 65, 700]),
    (1, 8, 3, 64, [2, 129, 1000]),
    (2, 1, 17, 80, [17, 400]),
    (1, 3, 5, 40, [5000, 3, 64]),
    (1, 2, 32, 16, [40, 333]),
    (2, 2, 100, 128, [99, 512]),
    (1, 16, 1, 128, [30000]),
    (1, 3, 50, 128, [49, 300]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Hk,G,Sq,D,lens", CACHE_CASES)
def test_cache_attention(cuda, dtype, causal, Hk, G, Sq, D, lens):
    B = len(lens)
    cache = cache_of(B, Hk, -(-max(max(lens), 1) // 64) * 64 + 64, D, lens, dtype, cuda)
    q = rand((B, Sq, Hk * G, D), dtype, 9, cuda).transpose(1, 2)
    out = cache.attend(q, causal=causal)
    o, size = ref_cache_attention(cache, q, causal, 1 / math.sqrt(D))
    few = G * Sq <= 128  # P in fp16 there, in the input's type in the tile kernel
    check(out, o, ((2.0 ** -11 if few else unit(dtype)) + SLACK) * size + unit(dtype) * o.abs() + 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Hk,G,Sq,D,lens", [(2, 1, 150, 128, [100, 0]), (1, 4, 1, 64, [64]), (2, 2, 300, 40, [37])])
def test_cache_attention_with_fresh_keys(cuda, dtype, causal, Hk, G, Sq, D, lens):
    B = len(lens)
    cache = cache_of(B, Hk, 192, D, lens, dtype, cuda)
    q, k, v = (rand((B, n, Sq, D), dtype, 9 + i, cuda) for i, n in enumerate((Hk * G, Hk, Hk)))
    out = cache.attend(q, k, v, causal=causal, sm_scale=0.2)
    o, size = ref_cache_attention(cache, q, causal, 0.2, k, v)
    check(out, o, (unit(dtype) + SLACK) * size + unit(dtype) * o.abs() + 2.0 ** -24)


def test_cache_decoding_in_a_graph(cuda):
    """One captured step, replayed: append, attend; against the same steps eagerly."""
    from longcat_video.models.kv_cache import KVCache8

    x = rand((2, 3, 2, 70, 64), torch.bfloat16, 1, cuda)
    a, b = (KVCache8.from_kv(x[0], x[1], 256) for _ in range(2))
    q, k, v = (rand((3, n, 1, 64), torch.bfloat16, i, cuda) for i, n in enumerate((4, 2, 2)))
    a.append(k, v)
    a.attend(q, causal=True)
    a.truncate(70)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.append(k, v)
        out = a.attend(q, causal=True)
    for i in range(5):
        for t, s in ((q, 10), (k, 20), (v, 30)):
            t.copy_(rand(t.shape, torch.bfloat16, s + i, cuda))
        b.append(k, v)
        want = b.attend(q, causal=True)
        g.replay()
        assert torch.equal(out, want) and a.lengths.tolist() == b.lengths.tolist() == [71 + i] * 3


def test_cache_refusals(cuda):
    from longcat_video.models.kv_cache import KVCache8

    c = KVCache8.allocate(2, 2, 100, 64, cuda)
    assert c.capacity == 128
    x = rand((2, 2, 5, 64), torch.bfloat16, 1, cuda)
    big = rand((2, 2, 129, 64), torch.bfloat16, 1, cuda)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=cuda)  # noqa: E731
    for a in ((x[:1], x[:1]), (x, x[:, :, :3]), (x.float(), x.float()), (x, x.half()), (x.cpu(), x.cpu()), (big, big),
              (x, x, i32(3)), (x, x, i32(2).long())):
        with pytest.raises(ValueError):
            c.append(*a)
    for a, kw in (((x[:, :, :, :32],), {}), ((x[:1],), {}), ((rand((2, 3, 5, 64), torch.bfloat16, 1, cuda),), {}),
                  ((x.float(),), {}), ((x, x), {}), ((x, x.half(), x.half()), {}), ((x,), dict(sm_scale=0.0)),
                  ((x,), dict(out=x[:1])), ((x.detach().requires_grad_(),), {})):
        with pytest.raises(ValueError):
            c.attend(*a, **kw)
    for n in (-1, 129, i32(3)):
        with pytest.raises(ValueError):
            c.truncate(n)
    with pytest.raises(ValueError):
        c.dequantize(torch.float32)
    good = (c.k_codes, c.k_scale, c.v_codes, c.v_scale, c.lengths)
    for i, t in ((0, c.k_codes[:, :, :64]), (0, c.k_codes.view(torch.uint8)), (1, c.k_scale[..., :1]), (3, c.v_scale.half()),
                 (4, c.lengths.long()), (4, c.lengths[:1])):
        with pytest.raises(ValueError):
            KVCache8(*[t if i == j else g for j, g in enumerate(good)])
    c.append(x[:, :, :0], x[:, :, :0])
    assert (c.attend(x) == 0).all() and c.attend(x[:, :, :0]).shape == (2, 2, 0, 64)


# ------------------------------------------------------------------------------- the attention hook's dense side
def hook(cuda, dtype=torch.bfloat16, dim=128, heads=2):
    from longcat_video.models.attention import Attention

    torch.manual_seed(3)
    m = Attention(dim, heads).to(cuda, dtype)
    with torch.no_grad():
        for n in (m.q_norm, m.k_norm):
            n.weight.add_(0.2 * torch.randn_like(n.weight))
    return m


def near(a, b, rel):
    assert a.shape == b.shape and torch.isfinite(a).all()
    assert ((a.double() - b.double()).norm() / b.double().norm()).item() <= rel


# The torch path rounds after each step, the kernels once a stage: a handful of roundings each way, averaged over
# the block's sums.  2^-8 of bf16 a rounding, two dozen of them in independent directions at most.
HOOK_REL = 5 * 2.0 ** -8


@pytest.mark.parametrize("cond", [None, 0, 2])
@pytest.mark.parametrize("B", [1, 2])
def test_hook_forward(cuda, B, cond):
    m = hook(cuda)
    shape = (5, 6, 7)
    x = rand((B, 210, 128), torch.bfloat16, 1, cuda)
    with torch.no_grad():
        want, kv = m(x, shape, cond, return_kv=True)
        m.dense_kernels = True
        got = m(x, shape, cond)
        got2, kv2 = m(x, shape, cond, return_kv=True)
    near(got, want, HOOK_REL)
    near(got2, want, HOOK_REL)
    near(kv2[0], kv[0], HOOK_REL)
    assert torch.equal(kv2[1], kv[1])


def test_hook_gradients(cuda):
    m = hook(cuda)
    x = rand((1, 210, 128), torch.bfloat16, 1, cuda).requires_grad_()
    g = rand((1, 210, 128), torch.bfloat16, 2, cuda)
    leaves = [x, m.q_norm.weight, m.k_norm.weight, m.qkv.weight]
    want = torch.autograd.grad(m(x, (5, 6, 7), 2), leaves, g)
    m.dense_kernels = True
    got = torch.autograd.grad(m(x, (5, 6, 7), 2), leaves, g)
    for a, b in zip(got, want):
        near(a, b, 2 * HOOK_REL)


@pytest.mark.parametrize("cond", [None, 2])
@pytest.mark.parametrize("B", [1, 2])
def test_hook_continuation(cuda, B, cond):
    """Over the (k, v) of earlier tokens, as tensors and as an 8-bit cache."""
    m = hook(cuda)
    x0, x = rand((1, 84, 128), torch.bfloat16, 1, cuda), rand((B, 126, 128), torch.bfloat16, 2, cuda)
    with torch.no_grad():
        _, kv = m(x0, (2, 6, 7), None, return_kv=True)
        want = m.forward_with_kv_cache(x, (3, 6, 7), cond, kv)
        cache = m.quantize_kv_cache(kv, (2, 6, 7), cond)
        eight = m.forward_with_kv_cache(x, (3, 6, 7), cond, cache)
        m.dense_kernels = True
        got = m.forward_with_kv_cache(x, (3, 6, 7), cond, kv)
    assert cache.lengths.tolist() == [84]
    near(got, want, HOOK_REL)
    near(eight, want, HOOK_REL + 2 * 2.0 ** -4)  # keys and values in e4m3: half a step is 2^-4
    with pytest.raises(ValueError):
        m.quantize_kv_cache(kv, (2, 6, 7), 1)


@pytest.mark.parametrize("cond", [None, 2])
def test_hook_continuation_gradients(cuda, cond):
    """Over a cache in 8 bits: the gradients of the same step over what it holds, as tensors."""
    m = hook(cuda)
    m.dense_kernels = True
    x0, x = rand((1, 84, 128), torch.bfloat16, 1, cuda), rand((2, 126, 128), torch.bfloat16, 2, cuda).requires_grad_()
    g = rand((2, 126, 128), torch.bfloat16, 3, cuda)
    with torch.no_grad():
        _, kv = m(x0, (2, 6, 7), None, return_kv=True)
        cache = m.quantize_kv_cache(kv, (2, 6, 7), cond)
        eight = m.forward_with_kv_cache(x, (3, 6, 7), cond, cache)
    leaves = [x, m.q_norm.weight, m.k_norm.weight, m.qkv.weight, m.proj.weight]
    out = m.forward_with_kv_cache(x, (3, 6, 7), cond, cache)
    near(out, eight, HOOK_REL)
    got = torch.autograd.grad(out, leaves, g)
    want = torch.autograd.grad(m.forward_with_kv_cache(x, (3, 6, 7), cond, kv), leaves, g)
    for a, b in zip(got, want):
        near(a, b, 2 * HOOK_REL + 4 * 2.0 ** -4)  # held keys and values in e4m3: half a step is 2^-4, in k and in v


def test_hook_bsa_keeps_its_path(cuda):
    """dense_kernels leaves block-sparse calls alone, and serves the hook's fallback for odd shapes."""
    m = hook(cuda)
    m.enable_bsa, m.bsa_sparsity = True, 0.5
    x = rand((1, 512, 128), torch.bfloat16, 1, cuda)
    odd = rand((1, 210, 128), torch.bfloat16, 2, cuda)
    with torch.no_grad():
        want, want_odd = m(x, (8, 8, 8)), m(odd, (5, 6, 7))
        m.dense_kernels = True
        assert torch.equal(m(x, (8, 8, 8)), want)
        near(m(odd, (5, 6, 7)), want_odd, HOOK_REL)


def test_hook_bsa_conditioning(cuda):
    """With BSA on, the noise tokens' dense part of the conditioning branch runs on the engine's kernel."""
    m = hook(cuda)
    m.enable_bsa, m.bsa_sparsity = True, 0.5
    x = rand((1, 512, 128), torch.bfloat16, 1, cuda)
    with torch.no_grad():
        want = m(x, (8, 8, 8), 4)
        m.dense_kernels = True
        near(m(x, (8, 8, 8), 4), want, HOOK_REL)


# ------------------------------------------------------------------------------- large sizes
def test_cache_beyond_32_bits(cuda):
    """Codes of the last head start behind 2^31 bytes: all keys weigh the same, values are ones in the last 100 tokens."""
    from longcat_video.models.kv_cache import KVCache8

    Hk, cap = 9, 1 << 21
    c = KVCache8.allocate(1, Hk, cap, 128, cuda)
    c.truncate(cap - 100)
    ones = torch.ones((1, Hk, 100, 128), dtype=torch.bfloat16, device=cuda)
    ones[:, :8] = 0
    c.append(ones * 0, ones)
    assert c.lengths.tolist() == [cap]
    out = c.attend(rand((1, Hk, 1, 128), torch.bfloat16, 1, cuda)).float()
    assert (out[:, :8] == 0).all()
    want = 100 / cap  # one rounding, and sums of 2^21 equal weights in 32 bits, block by block: 2^-24 of it for each join
    assert ((out[:, 8] - want).abs() <= want * (2.0 ** -8 + 2.0 ** -12)).all()


def test_norm_rope_beyond_32_bits(cuda):
    from longcat_video.models.rope_3d import qk_norm_rope

    grid, H, D = (33, 64, 64), 126, 128  # 2.2e9 values
    S = grid[0] * grid[1] * grid[2]
    rope = rope_of(grid, D, cuda)
    x = torch.empty((1, H, S, D), dtype=torch.bfloat16, device=cuda).normal_()
    w = torch.ones(D, device=cuda)
    y = qk_norm_rope(x, q_weight=w, rope=rope)
    for rows in (slice(0, 3), slice(S - 3, S)):
        turn = turns(rope, rows.start, 3)
        ref = ref_norm_rope(x[:, -2:, rows].double(), w.double(), 1e-6, turn)
        check(y[:, -2:, rows], ref, unit(torch.bfloat16) * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True))


def test_attention_over_many_keys(cuda):
    """A query tile over 300,000 keys in splits, and a long ragged mask of a few rows."""
    from longcat_video.models.masked_attention import AttentionMask, masked_attention

    Sk = 300001
    q, k, v = (rand((1, 2, s, 64), torch.bfloat16, i, cuda) for i, s in enumerate((5, Sk, Sk)))
    m = AttentionMask.from_ranges(torch.tensor([[[0, Sk], [Sk - 1, Sk], [7, 7], [100, 250000], [299990, Sk]]],
                                               dtype=torch.int32, device=cuda), Sk)
    out, lse = masked_attention(q, k, v, m, return_lse=True)
    check_attention(out, lse, ref_attention(q, k, v, *rows_of(m), 0.125), torch.bfloat16)
