"""The dense side without a GPU, further: refusals before any launch, and how the attention kernels wind down after a wait
that ran out of time.

The barrier model is test_dense_host.py's, with the tiles that the loading warp mends before it hands them on (it waits for
their loads on a barrier of its own, `fix`) and with an abort at any moment, after which every wait that is not over fails.
Whatever happens, the loading role ends with none of its loads in flight, and without waiting for one that was not issued."""

import random

import pytest

from test_attn_protocol import wait
from test_dense_host import FAKE, ST, WARPS, Machine, call, lib, ring_order, strides  # noqa: F401


@pytest.mark.parametrize("dims,grid", [((128, 0, 0), (2 ** 26, 1, 1)), ((0, 128, 0), (1, 2 ** 26, 1)), ((44, 42, 42), (1, 1, 2 ** 27)),
                                       ((0, 0, 128), (2 ** 10, 1, 2 ** 25))])
def test_rope_tables_beyond_32_bits(lib, dims, grid):  # noqa: F811
    """The kernels index an axis's table of cosines with 32 bits."""
    rope = [FAKE, *dims, *grid, 0]
    args = [FAKE, strides(*ST), 2, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 64, 128, 1e-6, *rope, None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "table" in msg
    args = [FAKE, strides(*ST), FAKE, strides(*ST), 2, FAKE, FAKE, None, None, None, None, None, 0, None, None, None, 2, 0, 1, 64, 128,
            1e-6, *rope, None, None]
    rc, msg = call(lib, "bsa_norm_rope_backward", "pspsippppspsipppiiiiifpiiiiiiipp", args)
    assert rc == 1 and "table" in msg


def test_rope_places_beyond_32_bits(lib):  # noqa: F811
    """A grid may hold more than 2^31 places; the tokens' own stay within 32 bits."""
    rope = [FAKE, 44, 42, 42, 2 ** 11, 2 ** 10, 2 ** 11, 2 ** 31 - 32]
    args = [FAKE, strides(*ST), 2, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 64, 128, 1e-6, *rope, None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "32 bits" in msg


def test_tokens_at_the_32_bit_border(lib):  # noqa: F811
    """The last tile's rows behind the last token are counted in 32 bits too."""
    args = [FAKE, strides(8, 8, 8), 1, FAKE, FAKE, None, None, 0, None, None, 2, 0, 1, 2 ** 31 - 3, 8, 1e-6, None, 0, 0, 0, 0, 0, 0, 0,
            None]
    rc, msg = call(lib, "bsa_norm_rope", "psipppsippiiiiifpiiiiiiip", args)
    assert rc == 1 and "too many tokens" in msg


# ------------------------------------------------------------------------------------------------ wind-down
class Aborting(Machine):
    """A machine whose waits fail once `abort` is set, at a random moment of a run."""

    def __init__(self, seed, runs_out):
        super().__init__(seed)
        self.abort, self.left = False, random.Random(seed).randrange(400) if runs_out else None

    def tick(self):
        if self.left is not None:
            self.left -= 1
            self.abort = self.abort or self.left < 0

    def wait(self, name, i, phase):
        while not wait(self.bars[name, i], phase):
            self.tick()
            if self.abort:
                return False
            yield
        return True

    def drain(self, name, i, phase):
        """As long as it takes (a limit ends it in the kernel: here the scheduler finds a deadlock)."""
        while not wait(self.bars[name, i], phase):
            yield

    def drain_ring(self, name, stages, issued):
        for i in range(max(0, issued - stages), issued):
            yield from self.drain(name, i % stages, i // stages)


class Loader:
    """The loading warp's books: tiles whose barrier will complete, by ring, and the load that `fix` still waits for."""

    def __init__(self, m, fix_tiles, careful=True):
        self.m, self.fix_tiles, self.careful = m, fix_tiles, careful
        self.issued, self.fixes, self.fixing = {}, 0, False

    def put(self, ring, stages, fix):
        """A load into the ring's next slot; False: a wait ran out."""
        m, n = self.m, self.issued.get(ring, 0)
        if not fix:
            m.load(ring, n % stages)
            self.issued[ring] = n + 1
            return True
        m.load("fix")
        self.fixing = True
        if not (yield from m.wait("fix", 0, self.fixes)):
            return False
        self.fixing = False
        self.fixes += 1
        yield
        m.arrive(ring, n % stages)
        self.issued[ring] = n + 1
        return True

    def end(self, singles, rings, finished):
        m = self.m
        if self.careful or not finished:
            for name in singles:
                yield from m.drain(name, 0, 0)
            for ring, stages in rings:
                yield from m.drain_ring(ring, stages, self.issued.get(ring, 0))
            if self.careful and self.fixing:
                yield from m.drain("fix", 0, self.fixes)
        assert not m.loads, "a load in flight as the loading warp ends"


def bars(m, *specs):
    for name, n, count in specs:
        m.bar(name, n, count)


def forward(steps, stages, seed, runs_out, careful=True):
    m, r = Aborting(seed, runs_out), random.Random(seed + 7)
    bars(m, ("q_full", 1, 1), ("q_ready", 1, 4), ("full", stages, 1), ("empty", stages, 1), ("s_full", 2, 1), ("s_read", 2, WARPS),
         ("p_full", 2, WARPS), ("o_full", 2, 1), ("fix", 1, 1))
    fix = {("v", j) for j in range(steps) if r.random() < 0.4}

    def loader():
        load = Loader(m, fix, careful)
        m.load("q_full")
        ok = True
        for i, tile in enumerate(ring_order(steps)):
            ok = (i < stages or (yield from m.wait("empty", i % stages, i // stages - 1))) and (
                yield from load.put("full", stages, tile in fix))
            if not ok:
                break
            yield
        yield from load.end(["q_full"], [("full", stages)], ok)

    def issuer():
        at = 0

        def ring():
            nonlocal at
            at += 1
            return (yield from m.wait("full", (at - 1) % stages, (at - 1) // stages))

        def qk(j):
            if j >= 2 and not (yield from m.wait("s_read", j & 1, (j - 2) >> 1)):
                return False
            if not (yield from ring()):
                return False
            m.commit("s_full", j & 1)
            m.commit("empty", (at - 1) % stages)
            return True

        ok = yield from m.wait("q_ready", 0, 0)
        for j in range(min(3, steps)):
            ok = ok and (yield from qk(j))
        for j in range(steps):
            ok = ok and (yield from ring()) and (yield from m.wait("p_full", j & 1, j >> 1))
            if not ok:
                return
            m.commit("o_full", j & 1)
            m.commit("empty", (at - 1) % stages)
            yield
            ok = j + 3 >= steps or (yield from qk(j + 3))

    def softmax(w):
        if w < 4:
            if not (yield from m.wait("q_full", 0, 0)):
                return
            m.arrive("q_ready")
        if not (yield from m.wait("s_full", 0, 0)):
            return
        m.arrive("s_read", 0)
        for j in range(steps):
            if j > 0 and not (yield from m.wait("o_full", (j - 1) & 1, (j - 1) >> 1)):
                return
            if j + 1 < steps and not (yield from m.wait("s_full", (j + 1) & 1, (j + 1) >> 1)):
                return
            yield
            m.arrive("p_full", j & 1)
            if j + 1 < steps:
                m.arrive("s_read", (j + 1) & 1)
            yield
        yield from m.wait("o_full", (steps - 1) & 1, (steps - 1) >> 1)

    m.run([loader(), issuer(), *(softmax(w) for w in range(WARPS))])
    return m


def backward_kv(steps, kq, kg, seed, runs_out, careful=True):
    m, r = Aborting(seed, runs_out), random.Random(seed + 7)
    bars(m, ("kv_full", 1, 1), ("q_full", kq, 1), ("q_empty", kq, 1), ("g_full", kg, 1), ("g_empty", kg, 1), ("s_full", 1, 1),
         ("dp_full", 1, 1), ("p_full", 1, WARPS), ("ds_full", 1, WARPS), ("done", 1, 1), ("fix", 1, 1))
    fix = {n for n in range(steps) if r.random() < 0.4}  # the tiles' queries, and then their gradients

    def loader():
        load = Loader(m, fix, careful)
        m.load("kv_full")
        ok = True
        for n in range(steps):
            ok = ((n < kq or (yield from m.wait("q_empty", n % kq, n // kq - 1)))
                  and (yield from load.put("q_full", kq, n in fix))
                  and (n < kg or (yield from m.wait("g_empty", n % kg, n // kg - 1)))
                  and (yield from load.put("g_full", kg, n in fix)))
            if not ok:
                break
            yield
        if not careful and not ok:  # as if the tile in hand had gone the plain way
            load.issued["q_full"] = n + 1
        yield from load.end(["kv_full"], [("q_full", kq), ("g_full", kg)], ok)

    def issuer():
        def dv(n):
            ok = yield from m.wait("p_full", 0, n)
            if ok:
                m.commit("g_empty", n % kg)
            return ok

        def dk(n):
            ok = yield from m.wait("ds_full", 0, n)
            if ok:
                m.commit("q_empty", n % kq)
            return ok

        ok = yield from m.wait("kv_full", 0, 0)
        for n in range(steps):
            ok = ok and (n == 0 or (yield from dv(n - 1))) and (yield from m.wait("q_full", n % kq, n // kq))
            if not ok:
                return
            m.commit("s_full")
            ok = (n == 0 or (yield from dk(n - 1))) and (yield from m.wait("g_full", n % kg, n // kg))
            if not ok:
                return
            m.commit("dp_full")
            yield
        if (yield from dv(steps - 1)) and (yield from dk(steps - 1)):
            m.commit("done")

    def compute():
        if not (yield from m.wait("kv_full", 0, 0)):
            return
        for n in range(steps):
            if not ((yield from m.wait("q_full", n % kq, n // kq)) and (yield from m.wait("s_full", 0, n))):
                return
            m.arrive("p_full")
            yield
            if not (yield from m.wait("dp_full", 0, n)):
                return
            m.arrive("ds_full")
            yield
        yield from m.wait("done", 0, 0)

    m.run([loader(), issuer(), *(compute() for _ in range(WARPS))])
    return m


def backward_q(steps, kk, kv, seed, runs_out, careful=True):
    m, r = Aborting(seed, runs_out), random.Random(seed + 7)
    bars(m, ("qg_full", 1, 1), ("k_full", kk, 1), ("k_empty", kk, 1), ("v_full", kv, 1), ("v_empty", kv, 1), ("s_full", 1, 1),
         ("s_read", 1, WARPS), ("dp_full", 2, 1), ("ds_full", 2, WARPS), ("done", 1, 1), ("fix", 1, 1))
    fix = {n for n in range(steps) if r.random() < 0.4}  # the tiles' keys

    def loader():
        load = Loader(m, fix, careful)
        m.load("qg_full")
        ok = True
        for n in range(steps):
            ok = ((n < kk or (yield from m.wait("k_empty", n % kk, n // kk - 1)))
                  and (yield from load.put("k_full", kk, n in fix))
                  and (n < kv or (yield from m.wait("v_empty", n % kv, n // kv - 1)))
                  and (yield from load.put("v_full", kv, False)))
            if not ok:
                break
            yield
        if not careful and not ok:
            load.issued["k_full"] = n + 1
        yield from load.end(["qg_full"], [("k_full", kk), ("v_full", kv)], ok)

    def issuer():
        def scores(n):
            if not (yield from m.wait("k_full", n % kk, n // kk)):
                return False
            m.commit("s_full")
            if not (yield from m.wait("v_full", n % kv, n // kv)):
                return False
            m.commit("dp_full", n & 1)
            m.commit("v_empty", n % kv)
            return True

        ok = (yield from m.wait("qg_full", 0, 0)) and (yield from scores(0))
        for n in range(steps):
            if n + 1 < steps:
                ok = ok and (yield from m.wait("s_read", 0, n)) and (yield from scores(n + 1))
            if not (ok and (yield from m.wait("ds_full", n & 1, n >> 1))):
                return
            m.commit("k_empty", n % kk)
            yield
        m.commit("done")

    def compute():
        for n in range(steps):
            if not (yield from m.wait("s_full", 0, n)):
                return
            m.arrive("s_read")
            yield
            if not (yield from m.wait("dp_full", n & 1, n >> 1)):
                return
            m.arrive("ds_full", n & 1)
            yield
        yield from m.wait("done", 0, 0)

    m.run([loader(), issuer(), *(compute() for _ in range(WARPS))])
    return m


KERNELS = [(forward, (5,)), (forward, (8,)), (backward_kv, (2, 2)), (backward_kv, (4, 4)), (backward_q, (3, 2)), (backward_q, (5, 4))]


@pytest.mark.parametrize("kernel,stages", KERNELS)
@pytest.mark.parametrize("steps", [1, 2, 5, 9])
def test_no_load_in_flight_at_the_end(kernel, stages, steps):
    aborted = 0
    for seed in range(60):
        kernel(steps, *stages, seed, False)
        aborted += kernel(steps, *stages, seed, True).abort
    assert aborted > 10


@pytest.mark.parametrize("kernel,stages", KERNELS)
def test_the_model_sees_a_load_left_behind(kernel, stages):
    """Draining the rings alone, and only after a failed wait: a load for `fix`, or the last ones, may outlive the CTA."""
    found = 0
    for seed in range(60):
        try:
            kernel(5, *stages, seed, True, careful=False)
        except AssertionError:
            found += 1
    assert found


def test_kernels_behind_another_read_coherently():
    """A kernel that may begin before the one in front of it has ended reads what that one wrote: its loads are ordered by
    after_previous().  Loads of read-only memory are not, and may be moved in front of it."""
    import os

    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "longcat-video-mlx_b200", "csrc")
    behind = [f for f in os.listdir(src) if f.endswith(".cu") and "after_previous()" in open(os.path.join(src, f)).read()]
    assert {"bsa_normrope.cu", "bsa_kv8.cu", "bsa_dense.cu"} <= set(behind)
    for f in (*behind, "bsa_rows.cuh", "bsa_dense.cuh"):
        text = open(os.path.join(src, f)).read()
        assert "__ldg" not in text and ".nc." not in text and "__restrict__" not in text, f


@pytest.mark.parametrize("scale,cap", [(3e38, 0.0), (1.0, 1e-39), (1e30, 1e-12), (1.0, 3e38)])
def test_scales_whose_products_overflow(lib, scale, cap):  # noqa: F811
    """sm_scale log2(e), its quotient by the cap and cap log2(e) are fp32: an infinite one would make NaN of a score of 0."""
    st = strides(*ST)
    args = [FAKE, FAKE, FAKE, 2, 1, 1, 1, 64, 64, 128, st, st, st, None, None, 1, scale, cap, FAKE, st, None, None, None, None]
    rc, msg = call(lib, "bsa_masked_attention", "pppiiiiiiisssppiffpspppp", args)
    assert rc == 7 and "range" in msg
    args = [*args[:3], FAKE, FAKE, FAKE, FAKE, *args[3:13], st, st, None, None, 1, scale, cap, FAKE, FAKE, FAKE, FAKE, None]
    rc, msg = call(lib, "bsa_masked_attention_backward", "pppppppiiiiiiisssssppiffppppp", args)
    assert rc == 7 and "range" in msg
    if not cap:
        args = [FAKE, 2, 1, 4, 1, st, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 128, 128, 0, scale, FAKE, st, FAKE, None]
        rc, msg = call(lib, "bsa_kv8_attention", "piiiispppppiiiifpspp", args)
        assert rc == 7 and "range" in msg
