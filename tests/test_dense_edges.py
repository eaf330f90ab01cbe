"""Edges of the dense side of the attention hook that its main tests leave out.

Tolerances as in test_dense_side.py: a rounding is off by half a step at most."""

import math

import pytest
import torch

from test_dense_side import hook, rand, rope_of

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
