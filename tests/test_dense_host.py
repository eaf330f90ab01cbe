"""The dense side without a GPU: the barrier protocols of its attention kernels, and what is refused before any launch.

The kernels' roles are restated as sequences of waits and arrivals on the same barriers with the same phase
arithmetic, and run under random timing (see test_attn_protocol.py): no schedule may deadlock, and no parity wait
may meet a barrier that is a phase further than a wait can tell apart."""

import ctypes
import os
import random

import pytest
import torch

from test_attn_protocol import Barrier, wait

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WARPS = 8


class Machine:
    """Barriers, asynchronous completions (loads in any order, products of one thread in theirs), a random scheduler."""

    def __init__(self, seed):
        self.rng, self.bars, self.loads, self.products, self.pairs = random.Random(seed), {}, [], [], {}

    def bar(self, name, n=1, count=1):
        for i in range(n):
            self.bars[name, i] = Barrier(f"{name}{i}", count)

    def wait(self, name, i, phase):
        while not wait(self.bars[name, i], phase):
            yield

    def arrive(self, name, i=0):
        self.bars[name, i].arrive()

    def load(self, name, i=0):
        self.loads.append((name, i))

    def commit(self, name, i=0):
        self.products.append((name, i))

    def pair(self, key):
        """A barrier of two roles (named barrier of two warps)."""
        n = self.pairs[key] = self.pairs.get(key, 0) + 1
        while self.pairs[key] < (n + 1) // 2 * 2:
            yield

    def run(self, roles):
        live = list(roles)
        idle = 0
        while live:
            x = self.rng.random()
            if x < 0.15 and self.loads:
                self.arrive(*self.loads.pop(self.rng.randrange(len(self.loads))))
                idle = 0
            elif x < 0.3 and self.products:
                self.arrive(*self.products.pop(0))
                idle = 0
            else:
                r = self.rng.choice(live)
                before = (sum(b.pending + b.completed for b in self.bars.values()), len(self.loads), len(self.products),
                          sum(self.pairs.values()))
                try:
                    next(r)
                except StopIteration:
                    live.remove(r)
                    idle = 0
                after = (sum(b.pending + b.completed for b in self.bars.values()), len(self.loads), len(self.products),
                         sum(self.pairs.values()))
                idle = 0 if before != after else idle + 1
                assert idle < 4000 or self.loads or self.products, "deadlock"


def ring_order(steps):
    """The forward kernel's loads: K(0) K(1) K(2), then V(j) K(j+3)."""
    ik = iv = 0
    order = []
    for _ in range(2 * steps):
        is_v = ik == steps or ik > iv + 2
        order.append(("v", iv) if is_v else ("k", ik))
        iv, ik = iv + is_v, ik + (not is_v)
    return order


def forward(steps, stages, seed, raises=0.3):
    m = Machine(seed)
    for name, n, count in (("q_full", 1, 1), ("q_ready", 1, 4), ("full", stages, 1), ("empty", stages, 1), ("s_full", 2, 1),
                           ("s_read", 2, WARPS), ("p_full", 2, WARPS), ("o_full", 2, 1)):
        m.bar(name, n, count)
    votes = [[random.Random(1000 * seed + 10 * p + j).random() < raises for j in range(steps)] for p in range(4)]

    def loader():
        m.load("q_full")
        for i in range(2 * steps):
            if i >= stages:
                yield from m.wait("empty", i % stages, i // stages - 1)
            m.load("full", i % stages)
            yield

    def issuer():
        at = 0

        def ring(kind, j):
            nonlocal at
            assert ring_order(steps)[at] == (kind, j)
            yield from m.wait("full", at % stages, at // stages)
            at += 1
            return (at - 1) % stages

        def qk(j):
            if j >= 2:
                yield from m.wait("s_read", j & 1, (j - 2) >> 1)
            slot = yield from ring("k", j)
            m.commit("s_full", j & 1)
            m.commit("empty", slot)

        yield from m.wait("q_ready", 0, 0)
        for j in range(min(3, steps)):
            yield from qk(j)
        for j in range(steps):
            slot = yield from ring("v", j)
            yield from m.wait("p_full", j & 1, j >> 1)
            m.commit("o_full", j & 1)
            m.commit("empty", slot)
            yield
            if j + 3 < steps:
                yield from qk(j + 3)

    def softmax(w):
        p = w & 3
        if w < 4:
            yield from m.wait("q_full", 0, 0)
            m.arrive("q_ready")
        yield from m.wait("s_full", 0, 0)
        m.arrive("s_read", 0)
        for j in range(steps):
            yield from m.pair((p, "vote"))
            if votes[p][j]:
                yield from m.pair((p, "max"))
                if j > 0:
                    yield from m.wait("o_full", (j - 1) & 1, (j - 1) >> 1)
            if j > 0:
                yield from m.wait("o_full", (j - 1) & 1, (j - 1) >> 1)
            if j + 1 < steps:
                yield from m.wait("s_full", (j + 1) & 1, (j + 1) >> 1)
            yield
            m.arrive("p_full", j & 1)
            if j + 1 < steps:
                m.arrive("s_read", (j + 1) & 1)
            yield
        yield from m.pair((p, "end"))
        yield from m.wait("o_full", (steps - 1) & 1, (steps - 1) >> 1)

    m.run([loader(), issuer(), *(softmax(w) for w in range(WARPS))])


def backward_kv(steps, kq, kg, seed):
    m = Machine(seed)
    for name, n, count in (("kv_full", 1, 1), ("q_full", kq, 1), ("q_empty", kq, 1), ("g_full", kg, 1), ("g_empty", kg, 1),
                           ("s_full", 1, 1), ("dp_full", 1, 1), ("p_full", 1, WARPS), ("ds_full", 1, WARPS), ("done", 1, 1)):
        m.bar(name, n, count)

    def loader():
        m.load("kv_full")
        for n in range(steps):
            if n >= kq:
                yield from m.wait("q_empty", n % kq, n // kq - 1)
            m.load("q_full", n % kq)
            if n >= kg:
                yield from m.wait("g_empty", n % kg, n // kg - 1)
            m.load("g_full", n % kg)
            yield

    def issuer():
        def dv(n):
            yield from m.wait("p_full", 0, n)
            m.commit("g_empty", n % kg)

        def dk(n):
            yield from m.wait("ds_full", 0, n)
            m.commit("q_empty", n % kq)

        yield from m.wait("kv_full", 0, 0)
        for n in range(steps):
            if n > 0:
                yield from dv(n - 1)
            yield from m.wait("q_full", n % kq, n // kq)
            m.commit("s_full")
            if n > 0:
                yield from dk(n - 1)
            yield from m.wait("g_full", n % kg, n // kg)
            m.commit("dp_full")
            yield
        yield from dv(steps - 1)
        yield from dk(steps - 1)
        m.commit("done")

    def compute():
        for n in range(steps):
            yield from m.wait("q_full", n % kq, n // kq)  # the tile's statistics
            yield from m.wait("s_full", 0, n)
            m.arrive("p_full")
            yield
            yield from m.wait("dp_full", 0, n)
            m.arrive("ds_full")
            yield
        yield from m.wait("done", 0, 0)

    m.run([loader(), issuer(), *(compute() for _ in range(WARPS))])


def backward_q(steps, kk, kv, seed):
    m = Machine(seed)
    for name, n, count in (("qg_full", 1, 1), ("k_full", kk, 1), ("k_empty", kk, 1), ("v_full", kv, 1), ("v_empty", kv, 1),
                           ("s_full", 1, 1), ("s_read", 1, WARPS), ("dp_full", 2, 1), ("ds_full", 2, WARPS), ("done", 1, 1)):
        m.bar(name, n, count)

    def loader():
        m.load("qg_full")
        for n in range(steps):
            if n >= kk:
                yield from m.wait("k_empty", n % kk, n // kk - 1)
            m.load("k_full", n % kk)
            if n >= kv:
                yield from m.wait("v_empty", n % kv, n // kv - 1)
            m.load("v_full", n % kv)
            yield

    def issuer():
        def scores(n):
            yield from m.wait("k_full", n % kk, n // kk)
            m.commit("s_full")
            yield from m.wait("v_full", n % kv, n // kv)
            m.commit("dp_full", n & 1)
            m.commit("v_empty", n % kv)

        yield from m.wait("qg_full", 0, 0)
        yield from scores(0)
        for n in range(steps):
            if n + 1 < steps:
                yield from m.wait("s_read", 0, n)
                yield from scores(n + 1)
            yield from m.wait("ds_full", n & 1, n >> 1)
            m.commit("k_empty", n % kk)
            yield
        m.commit("done")

    def compute():
        for n in range(steps):
            yield from m.wait("s_full", 0, n)
            m.arrive("s_read")
            yield
            yield from m.wait("dp_full", n & 1, n >> 1)
            m.arrive("ds_full", n & 1)
            yield
        yield from m.wait("done", 0, 0)

    m.run([loader(), issuer(), *(compute() for _ in range(WARPS))])


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 9, 16])
def test_protocols(steps):
    for seed in range(12):
        for stages in (5, 8):
            forward(steps, stages, seed)
        for kq, kg in ((2, 2), (4, 4)):
            backward_kv(steps, kq, kg, seed)
        for kk, kv in ((3, 2), (5, 4)):
            backward_q(steps, kk, kv, seed)


def test_protocol_model_sees_mistakes():
    """One barrier instead of two for P V would be misread by a softmax that is a step behind."""
    m = Machine(0)
    m.bar("o_full")
    for _ in range(2):
        m.arrive("o_full")
    with pytest.raises(AssertionError):
        next(m.wait("o_full", 0, 0))


def test_division_by_multiplication():
    """n // d for n < 2^31 as the norm + rope kernel divides: (n * ceil(2^(31 + k) / d)) >> (31 + k), 2^k >= d."""
    r = random.Random(1)
    for d in [2, 3, 5, 7, 26, 45, 52, 80, 1560, 3600, 86400, 2 ** 20, 2 ** 31 - 1, *(r.randrange(2, 2 ** 31) for _ in range(200))]:
        k = (d - 1).bit_length()
        m = -(-(1 << (31 + k)) // d)
        assert m < 2 ** 32
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 ** 31 - 1, *(r.randrange(2 ** 31) for _ in range(50))]:
            if n < 2 ** 31:
                assert ((n * m) >> 32) >> (k - 1) == n // d


# ------------------------------------------------------------------------------------- refusals, before any launch
@pytest.fixture(scope="module")
def lib():
    import build  # longcat-video-mlx_b200/build.py

    return ctypes.CDLL(build.build())


FAKE = 1 << 20  # 16-byte aligned, never dereferenced: the checks below run on the host


def strides(*v):
    return (ctypes.c_int64 * 3)(*v)


def call(lib, name, types, args):
    f = getattr(lib, name)
    f.argtypes = [{"p": ctypes.c_void_p, "s": ctypes.POINTER(ctypes.c_int64), "i": ctypes.c_int, "f": ctypes.c_float}[t]
                  for t in types]
    f.restype = ctypes.c_int
    rc = f(*args)
    buf = ctypes.create_string_buffer(512)
    lib.bsa_last_error(buf, 512)
    return rc, buf.value.decode()


ST = (64 * 128, 64 * 128, 128)


@pytest.mark.parametrize("change,code", [
    ({0: None}, 7), ({1: FAKE + 8}, 3), ({3: 0}, 2), ({4: 0}, 1), ({6: 3}, 1), ({9: 136}, 1), ({9: 12}, 1), ({10: None}, 7),
    ({11: strides(64 * 128, 64 * 128, 129)}, 3), ({13: FAKE}, 7), ({13: FAKE, 14: FAKE, 15: 3}, 1), ({13: FAKE + 4, 14: FAKE}, 3),
    ({16: 0.0}, 7), ({16: float("nan")}, 7), ({17: -1.0}, 7), ({17: float("inf")}, 7), ({18: None}, 7), ({19: None}, 7),
    ({20: FAKE + 2}, 3)])
def test_masked_attention_refusals(lib, change, code):
    args = [FAKE, FAKE, FAKE, 2, 2, 4, 2, 64, 64, 128, strides(4 * 64 * 128, *ST[1:]), strides(2 * 64 * 128, *ST[1:]),
            strides(2 * 64 * 128, *ST[1:]), None, None, 1, 0.1, 0.0, FAKE, strides(4 * 64 * 128, *ST[1:]), None, None, None, None]
    for i, v in change.items():
        args[i] = v
    rc, msg = call(lib, "bsa_masked_attention", "pppiiiiiiisssppiffpspppp", args)
    assert rc == code and msg


@pytest.mark.parametrize("change,code", [
    ({0: None}, 7), ({1: FAKE + 4}, 3), ({2: 0}, 1), ({3: 0}, 1), ({4: -1}, 1), ({7: -1}, 7), ({9: FAKE}, 7),
    ({9: FAKE, 10: FAKE, 11: 0}, 1), ({9: FAKE, 10: FAKE, 11: 2, 13: FAKE}, 7)])
def test_ranges_refusals(lib, change, code):
    args = [FAKE, FAKE, 1, 10, 10, None, 0, 0, None, None, None, 0, None, None, 0, None]
    for i, v in change.items():
        args[i] = v
    rc, msg = call(lib, "bsa_attention_ranges", "ppiiipiipppippip", args)
    assert rc == code and msg


@pytest.mark.parametrize("change,code", [
    ({0: None}, 7), ({4: None}, 7), ({5: 0}, 1), ({7: 100}, 1), ({7: 0}, 1), ({8: 12}, 1), ({0: FAKE + 8}, 3), ({9: None}, 7),
    ({10: FAKE + 2}, 3), ({11: 0}, 2), ({12: 0}, 1), ({12: 129}, 1), ({13: None}, 7), ({6: 70000}, 1)])
def test_cache_append_refusals(lib, change, code):
    args = [FAKE, FAKE, FAKE, FAKE, FAKE, 1, 2, 128, 128, FAKE, FAKE, 2, 5, strides(*ST), strides(*ST), None, None]
    for i, v in change.items():
        args[i] = v
    rc, msg = call(lib, "bsa_kv8_append", "pppppiiiippiisspp", args)
    assert rc == code and msg


@pytest.mark.parametrize("change,code", [
    ({0: None}, 7), ({1: 0}, 2), ({3: 5}, 1), ({4: 0}, 1), ({5: None}, 7), ({6: None}, 7), ({12: 100}, 1), ({15: 0.0}, 7),
    ({16: None}, 7), ({17: None}, 7), ({4: 1 << 24}, 1)])
def test_cache_attention_refusals(lib, change, code):
    args = [FAKE, 2, 1, 4, 1, strides(*ST), FAKE, FAKE, FAKE, FAKE, FAKE, 2, 128, 128, 0, 0.1, FAKE, strides(*ST), FAKE, None]
    for i, v in change.items():
        args[i] = v
    rc, msg = call(lib, "bsa_kv8_attention", "piiiispppppiiiifpspp", args)
    assert rc == code and msg


@pytest.mark.parametrize("change,code", [
    ({0: None}, 7), ({1: None}, 7), ({2: 0}, 1), ({4: None}, 7), ({4: FAKE + 8}, 3), ({10: 5}, 2), ({11: 9}, 2), ({13: 0}, 1),
    ({14: 130}, 1), ({15: -1.0}, 7), ({16: FAKE}, 1), ({16: FAKE, 17: 44, 18: 42, 19: 42, 20: 1, 21: 4, 22: 15}, 1),
    ({16: FAKE, 17: 44, 18: 42, 19: 42, 20: 1, 21: 4, 22: 16, 23: 1}, 1)])
def test_norm_rope_refusals(lib, change, code):
    args = [FAKE, strides(*ST), 2, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 64, 128, 1e-6, None, 0, 0, 0, 0, 0, 0, 0, None]
    for i, v in change.items():
        args[i] = v
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == code and msg


@pytest.mark.parametrize("name,types,args", [
    ("bsa_masked_attention", "pppiiiiiiisssppiffpspppp",
     [FAKE, FAKE, FAKE, 2, 1, 1, 1, 64, 8192, 128, strides(*ST), strides(*ST), strides(*ST), None, None, 1, 0.1, 0.0, FAKE,
      strides(*ST), None, None, FAKE + 8, None]),
    ("bsa_kv8_attention", "piiiispppppiiiifpspp",
     [FAKE, 2, 1, 4, 1, strides(*ST), FAKE, FAKE, FAKE, FAKE, FAKE, 2, 8192, 128, 0, 0.1, FAKE, strides(*ST), FAKE + 4, None])])
def test_scratch_alignment(lib, name, types, args):
    """Few rows over many keys are split and need scratch, which is read 16 bytes at a time."""
    rc, msg = call(lib, name, types, args)
    assert rc == 3 and "scratch" in msg
    args[-2] = None
    rc, msg = call(lib, name, types, args)
    assert rc == 7 and "scratch" in msg


def test_most_tokens(lib):
    for Sq, Sk in ((2 ** 30 + 1, 1), (1, 2 ** 30 + 1)):
        args = [FAKE, FAKE, FAKE, 2, 1, 1, 1, Sq, Sk, 8, strides(8, 8, 8), strides(8, 8, 8), strides(8, 8, 8), None, None, 1,
                0.1, 0.0, FAKE, strides(8, 8, 8), None, None, None, None]
        assert call(lib, "bsa_masked_attention", "pppiiiiiiisssppiffpspppp", args)[0] == 1
        args = [FAKE, FAKE, 1, Sq, Sk, None, 0, 0, None, None, None, 0, None, None, 0, None]
        assert call(lib, "bsa_attention_ranges", "ppiiipiipppippip", args)[0] == 1
    args = [FAKE, FAKE, 2 ** 20, 2 ** 20, 1, None, 0, 0, None, None, None, 0, None, None, 0, None]
    rc, msg = call(lib, "bsa_attention_ranges", "ppiiipiipppippip", args)
    assert rc == 1 and "too many rows" in msg


def test_host_tensors_are_refused():
    from longcat_video.models.kv_cache import KVCache8
    from longcat_video.models.masked_attention import AttentionMask, masked_attention
    from longcat_video.models.rope_3d import qk_norm_rope

    x = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
    for f in (lambda: masked_attention(x, x, x), lambda: qk_norm_rope(x, q_weight=torch.ones(64)),
              lambda: AttentionMask.build(4, 4, device="cpu"), lambda: AttentionMask.build(4, 4, k_lengths=torch.ones(2).int()),
              lambda: KVCache8.allocate(1, 1, 64, 64, "cpu"), lambda: qk_norm_rope(x)):
        with pytest.raises(ValueError):
            f()


def test_dit_switch():
    from longcat_video.models.longcat_video_dit import LongCatVideoTransformer3DModel

    d = LongCatVideoTransformer3DModel.from_config(dict(hidden_size=64, depth=2, num_heads=2, enable_dense_kernels=True))
    assert all(a.dense_kernels and not a.enable_bsa for a in d.attention_modules())
    d.disable_dense_kernels()
    assert not any(a.dense_kernels for a in d.attention_modules())
