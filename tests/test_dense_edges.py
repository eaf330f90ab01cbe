"""Edges of the dense side of the attention hook that its main tests leave out.

Tolerances as in test_dense_side.py: a rounding is off by half a step at most."""

import math

import pytest
import torch

from test_dense_side import (SLACK, check, check_gradients, full, gradients, hook, rand, ref_attention, ref_gradients, rope_of,
                             unit)

pytestmark = pytest.mark.gpu


def junk(shape, dtype, device):
    """Freed memory of NaN, which the allocator hands out again."""
    held = [torch.full(shape, math.nan, dtype=dtype, device=device) for _ in range(4)]
    del held


# ------------------------------------------------------------------------------------------ norm + rope
@pytest.mark.parametrize("heads", [(3, 0), (0, 2), (0, 0)])
def test_norm_rope_side_without_heads(cuda, heads):
    """One side empty: the other is computed all the same, and the empty one's weight has a gradient of zeros."""
    from longcat_video.models.rope_3d import qk_norm_rope

    rope = rope_of((1, 5, 6), 64, cuda)
    x = [rand((2, n, 30, 64), torch.bfloat16, n, cuda) for n in heads]
    w = [1 + 0.2 * rand((64,), torch.float32, 7 + i, cuda) for i in range(2)]
    g = [rand((2, n, 30, 64), torch.bfloat16, 9 + n, cuda) for n in heads]

    def alone(i):
        a, b = x[i].detach().requires_grad_(), w[i].detach().requires_grad_()
        y = qk_norm_rope(a, None, b, rope=rope)
        return (y.detach(), *torch.autograd.grad(y, (a, b), g[i]))

    want = [alone(i) for i in range(2)]
    junk((2, 3, 30, 64), torch.bfloat16, cuda)
    got = qk_norm_rope(*x, *w, rope=rope)
    for i in range(2):
        assert got[i].shape == x[i].shape and torch.equal(got[i], want[i][0])
    leaves = [t.detach().requires_grad_() for t in (*x, *w)]
    out = qk_norm_rope(*leaves, rope=rope)
    junk((2, 3, 30, 64), torch.bfloat16, cuda)
    got = torch.autograd.grad(out, leaves, g)
    for i in range(2):
        assert torch.equal(got[i], want[i][1]) and torch.equal(got[2 + i], want[i][2])
        assert heads[i] or not got[2 + i].any()


def test_hook_norms_with_their_own_eps(cuda):
    """q and k are normalised with their own constants, in one call or two."""
    from longcat_video.models.rope_3d import qk_norm_rope

    m = hook(cuda)
    m.k_norm.eps = 0.5
    q, k = (rand((1, 2, 210, 64), torch.bfloat16, i, cuda) for i in range(2))
    rope = m.rope_3d.tables((5, 6, 7), q.device)
    with torch.no_grad():
        got = m._norm_rope(q, k, (5, 6, 7))
        for y, x, n in zip(got, (q, k), (m.q_norm, m.k_norm)):
            assert torch.equal(y, qk_norm_rope(x, None, n.weight, eps=n.eps, rope=rope))


def test_forward_mode_is_refused(cuda):
    """A tangent would be lost: every call that has one among its inputs says so."""
    import torch.autograd.forward_ad as fwd

    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import masked_attention
    from longcat_video.models.rope_3d import qk_norm_rope

    x = rand((1, 2, 20, 64), torch.bfloat16, 1, cuda)
    w = torch.ones(64, device=cuda)
    cache = KVCache8.from_kv(x, x)
    with fwd.dual_level():
        d, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
        for f in (lambda: masked_attention(d, x, x), lambda: masked_attention(x, d, x), lambda: masked_attention(x, x, d),
                  lambda: masked_attention(x, x, x, out=d), lambda: qk_norm_rope(d, q_weight=w),
                  lambda: qk_norm_rope(x, d, w, w), lambda: qk_norm_rope(x, q_weight=dw), lambda: cache.attend(d),
                  lambda: cache.attend(x, d, x), lambda: cache.attend(x, x, d)):
            with pytest.raises(ValueError, match="forward-mode"):
                f()
        masked_attention(x, x, x)  # without a tangent


def fp16_case(H, Hk, Sq, Sk, gs, vs, device, seed=0):
    q, k = rand((1, H, Sq, 128), torch.float16, seed, device, 0.5), rand((1, Hk, Sk, 128), torch.float16, seed + 1, device, 0.5)
    v = rand((1, Hk, Sk, 128), torch.float16, seed + 2, device, vs)
    # gradients along the values, so that their products are as large as their norms allow
    g = v[:, :1, torch.arange(Sq, device=device) % Sk].expand(1, H, Sq, 128).float() * (gs / vs)
    return q, k, v, g.half()


@pytest.mark.parametrize("H,Hk,Sq,Sk,gs,vs", [(2, 1, 6, 5, 6000.0, 1.0), (2, 2, 7, 3, 0.12, 8000.0), (4, 1, 300, 6, 60.0, 100.0),
                                              (1, 1, 130, 300, 12000.0, 3.0), (2, 1, 1, 2, 15000.0, 1.0)])
def test_large_gradients_in_fp16(cuda, H, Hk, Sq, Sk, gs, vs):
    """Products of p, do and v beyond fp16's largest number, of a gradient that is not: finite, with their bits."""
    from longcat_video.models.masked_attention import AttentionMask

    q, k, v, g = fp16_case(H, Hk, Sq, Sk, gs, vs, cuda)
    scale = 2.0 ** -8
    for m in (None, AttentionMask.build(Sq, Sk, causal=True, device=cuda)):
        rows = full(Sq, Sk, cuda) if m is None else (m.ranges[..., 0].long(), m.ranges[..., 1].long())
        _, got = gradients(q, k, v, g, m, sm_scale=scale)
        want = ref_gradients(q, k, v, g, *rows, scale, 0.0)[0]
        assert all(w.abs().max() < 65504 for w in want)  # the result itself fits
        check_gradients(got, q, k, v, g, *rows, scale)


def test_large_values_do_not_cost_other_rows_their_bits(cuda):
    """A row's dq depends on its own gradient's size, a key's dk on its own value's: the others keep their precision.

    dq of rows with small gradients beside rows with large ones; values behind the padded length that are large but finite."""
    from longcat_video.models.masked_attention import AttentionMask

    q, k, v, g = (rand((1, 2, n, 64), torch.float16, i, cuda) for i, n in enumerate((200, 400, 400, 200)))
    g = g * torch.where(torch.arange(200, device=cuda) % 2 == 0, 8000.0, 2.0 ** -6)[:, None].half()
    m = AttentionMask.build(200, 400, k_lengths=torch.tensor([300], dtype=torch.int32, device=cuda))
    rows = (m.ranges[..., 0].long(), m.ranges[..., 1].long())
    _, want = gradients(q, k, v, g, m)
    check_gradients(want, q, k, v, g, *rows, 0.125)
    grads, ds, dl, fine, _ = ref_gradients(q, k, v, g, *rows, 0.125, 0.0)
    u, odd = unit(torch.float16), slice(1, None, 2)
    # the small rows' ds is raised by 2^10 at least (2^-6 * 8 * 2^4 * 2^10 < 2^12): steps of 2^-34 over the row's 300 keys
    x = k.double().abs().amax() * 0.125 * 300 * 2.0 ** -34
    part = lambda t: t[:, :, odd]  # noqa: E731
    check(part(want[0]), part(grads[0]), u * part(grads[0]).abs() + u * part(ds[0]) + u * part(dl[0]) + SLACK * part(fine[0])
          + x + 2.0 ** -24)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 300:], v2[:, :, 300:] = 60000.0, 60000.0
    _, got = gradients(q, k2, v2, g, m)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_a_block_of_zeros(cuda, dtype):
    """Infinities are the block's largest code whatever else it holds; NaN stays; a lookup stays finite."""
    from longcat_video.models.kv_cache import KVCache8

    x = torch.zeros((1, 3, 70, 16), dtype=dtype, device=cuda)
    x[0, 0, 3, 4], x[0, 0, 9, 9] = math.inf, -math.inf
    x[0, 1, 65, 1] = math.inf
    x[0, 2, 5, 5] = math.nan
    cache = KVCache8.from_kv(x, x)
    codes = cache.k_codes.float()
    assert codes[0, 0, 3, 4] == 448 and codes[0, 0, 9, 9] == -448 and codes[0, 1, 65, 1] == 448
    assert codes[0, 2, 5, 5].isnan() and codes.nan_to_num(0).count_nonzero() == 3
    assert torch.equal(cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8))
    out = cache.attend(rand((1, 3, 1, 16), dtype, 1, cuda))
    assert torch.isfinite(out[:, :2]).all()
    kd, _ = cache.dequantize(dtype)
    assert torch.isfinite(kd[:, :2]).all()
    one = torch.ones((1, 3, 1, 16), dtype=dtype, device=cuda)  # a finite value sets the scale as ever
    cache.append(one, one)
    assert cache.k_scale[0, :, 1].tolist() == [2.0 ** -8] * 3
    assert (cache.dequantize(dtype)[0][:, :, 70] == 1).all()


def sink(dtype, rows, n, device):
    """A key 18 nats above n - 1 others, whose values alone count: (q, k, v, the result in 64 bits)."""
    q = torch.zeros((1, 1, rows, 16), dtype=dtype, device=device)
    q[..., 0] = 1
    k = torch.zeros((1, 1, n, 16), dtype=dtype, device=device)
    k[0, 0, 777, 0] = 18
    v = torch.ones((1, 1, n, 16), dtype=dtype, device=device)
    v[0, 0, 777] = 0
    return q, k, v, ref_attention(q[:, :, :1], k, v, *full(1, n, device), 1.0)[:3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 130])
def test_long_tail_under_a_sink(cuda, dtype, rows):
    """20,000 keys 18 nats below one: each weighs 2^-26, together they are the result.

    Beside the roundings that check_attention counts, a weight may be off by half of a subnormal step of fp16, 2^-25, of what
    it is raised by, 2^7 at least: 2^-32 a key of the largest weight, of which the row's sum is one at least.  80 heads
    leave no split along the keys, which would part the sink from most of the others."""
    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import masked_attention

    n = 20_000
    q, k, v, (o, lse, size) = sink(dtype, rows, n, cuda)
    bound = (2.0 ** -11 + unit(dtype) + SLACK) * size + unit(dtype) * o.abs() + n * 2.0 ** -32
    wide = lambda t: t.expand(1, 80, *t.shape[2:])  # noqa: E731
    got, l = masked_attention(wide(q), k, v, sm_scale=1.0, return_lse=True)
    check(got, o.expand(got.shape), bound)
    check(l, lse.expand(l.shape), 2.0 ** -16 * (1 + lse.abs()))
    if rows > 128:  # the cache is unpacked
        check(KVCache8.from_kv(wide(k), wide(v)).attend(wide(q), sm_scale=1.0), o.expand(got.shape), bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lookup_of_a_long_tail_under_a_sink(cuda, dtype):
    """As above from the codes, which hold these keys and values exactly; 900 key heads leave no split."""
    from longcat_video.models.kv_cache import KVCache8

    q, k, v, (o, _, size) = sink(dtype, 1, 20_000, cuda)
    wide = lambda t: t.expand(1, 900, *t.shape[2:])  # noqa: E731
    got = KVCache8.from_kv(wide(k), wide(v)).attend(wide(q), sm_scale=1.0)
    check(got, o.expand(got.shape), (2.0 ** -11 + SLACK) * size + unit(dtype) * o.abs() + 20_000 * 2.0 ** -32)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("times", [2.0, 6.0, 9.0, 12.0])
@pytest.mark.parametrize("Sq,Sk", [(3, 5), (140, 700)])
def test_slope_of_the_cap_far_out(cuda, times, sign, Sq, Sk):
    """Scores at several times the cap: 1 - tanh^2 falls like 4 e^(-2 |s| / cap) and keeps its digits."""
    from longcat_video.models.masked_attention import AttentionMask

    q, k, v, g = (rand((1, 2, n, 64), torch.bfloat16, i, cuda, 0.02 if i < 2 else 1.0) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    cap = 4.0
    q[..., 0], k[..., 0] = times, sign
    scale = cap  # scores near times * cap
    for m in (None, AttentionMask.build(Sq, Sk, causal=True, device=cuda)):
        rows = full(Sq, Sk, cuda) if m is None else (m.ranges[..., 0].long(), m.ranges[..., 1].long())
        _, got = gradients(q, k, v, g, m, softcap=cap, sm_scale=scale)
        grads, ds, dl, fine, _ = ref_gradients(q, k, v, g, *rows, scale, cap)
        u = unit(torch.bfloat16)
        # 2 |s| / cap in fp32: an error of 2^-20 of it (sums, scale and the exponential) is one of the slope
        e = SLACK + 2.0 ** -18 * 2 * (times + 1)
        for i in range(2):
            check(got[i], grads[i], u * grads[i].abs() + (u + e) * ds[i] + u * dl[i] + SLACK * fine[i] + 1e-37)


def test_outputs_over_packed_inputs(cuda):
    """Slots of one packed projection: over q in place, over k or v refused, beside them in place."""
    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import masked_attention

    for H, N in ((3, 210), (4, 64)):
        packed = rand((2, N, 4, H, 64), torch.bfloat16, 1, cuda)
        q, k, v, free = packed.permute(2, 0, 3, 1, 4)
        want = masked_attention(q, k, v)
        cache = KVCache8.from_kv(k, v)
        held = cache.attend(q, k, v)
        for bad in (k, v):
            with pytest.raises(ValueError, match="overlaps"):
                masked_attention(q, k, v, out=bad)
            with pytest.raises(ValueError, match="overlaps"):
                cache.attend(q, k, v, out=bad)
        before = packed.clone()
        masked_attention(q, k, v, out=free)
        assert torch.equal(free, want) and torch.equal(packed[:, :, :3], before[:, :, :3])
        cache.attend(q, k, v, out=free)
        assert torch.equal(free, held) and torch.equal(packed[:, :, :3], before[:, :, :3])
        masked_attention(q, k, v, out=q)
        assert torch.equal(q, want) and torch.equal(packed[:, :, 1:3], before[:, :, 1:3])


def test_outputs_that_shift_or_turn_an_input(cuda):
    from longcat_video.models.masked_attention import masked_attention

    row = rand((1, 2 * 41, 2, 64), torch.bfloat16, 1, cuda)
    q = row[:, 0:80:2].transpose(1, 2)  # every second token of both heads
    k = rand((1, 2, 50, 64), torch.bfloat16, 2, cuda)
    want = masked_attention(q, k, k)
    for bad in (row[:, 2:82:2].transpose(1, 2), row[:, 1:41].transpose(1, 2)):  # shifted, and of another step
        with pytest.raises(ValueError, match="overlaps"):
            masked_attention(q, k, k, out=bad)
    odd = row[:, 1:81:2].transpose(1, 2)  # the tokens between
    assert torch.equal(masked_attention(q, k, k, out=odd), want)
    square = rand((1, 6, 6, 64), torch.bfloat16, 3, cuda)
    with pytest.raises(ValueError, match="overlaps"):
        masked_attention(square, square.clone(), square.clone(), out=square.transpose(1, 2))
    flat = torch.zeros(4096, dtype=torch.bfloat16, device=cuda)
    for bad in (flat.as_strided((1, 2, 40, 64), (8192, 2048, 32, 1)), flat[:64].expand(1, 2, 40, 64)):  # rows over one another
        with pytest.raises(ValueError, match="overlaps"):
            masked_attention(q.contiguous(), k, k, out=bad)


def test_overlaps_of_views_against_their_places(cuda):
    """Random views into one buffer: refused where, and only where, a place of the output is one of an input or its own."""
    import random

    from longcat_video.models.masked_attention import masked_attention

    r = random.Random(5)
    buf = torch.zeros(6000, dtype=torch.bfloat16, device=cuda)
    index = torch.arange(6000)

    def view(S):
        while True:
            H = r.choice([1, 2, 2, 3])
            step = [8 * r.choice([0, 1, 1, 2, 3, 4, 5, 12, 20, 40, 41]) if r.random() < 0.9 else r.randint(1, 70) for _ in range(3)]
            at, shape = r.choice([8 * r.randint(0, 200), r.randint(0, 1000)]), (2, H, S, 8)
            if at + sum((n - 1) * s for n, s in zip(shape, step)) + 8 <= 6000:
                return lambda t: t.as_strided(shape, (*step, 1), at)

    seen = {True: 0, False: 0}
    for _ in range(400):
        make = [view(5), view(7)]
        out = make[0](buf)
        q = torch.ones_like(out)
        k, H = make[1](buf), out.shape[1]
        if H % k.shape[1]:
            continue
        own, other = make[0](index).flatten().tolist(), set(make[1](index).flatten().tolist())
        meets = len(set(own)) < len(own) or not other.isdisjoint(own)
        seen[meets] += 1
        if meets:
            with pytest.raises(ValueError, match="overlaps"):
                masked_attention(q, k, torch.ones_like(k), out=out)
        else:
            masked_attention(q, k, torch.ones_like(k), out=out)
            assert (out == 1).all() and buf.count_nonzero() == out.numel()
            buf.zero_()
    assert min(seen.values()) > 40


def test_cache_without_heads_is_refused(cuda):
    from longcat_video.models.kv_cache import KVCache8

    with pytest.raises(ValueError, match="heads"):
        KVCache8.allocate(1, 0, 64, 64, cuda)
    with pytest.raises(ValueError, match="heads"):
        KVCache8.from_kv(*(torch.empty((1, 0, 5, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2)))


def test_a_cap_below_every_float_is_refused(cuda):
    """It would be rounded to 0, which means no cap."""
    from longcat_video.models.masked_attention import masked_attention

    x = rand((1, 1, 4, 16), torch.bfloat16, 1, cuda)
    with pytest.raises(ValueError, match="softcap"):
        masked_attention(x, x, x, softcap=1e-60)
