"""The calls around drafted tokens and adapters that the contexts' workspaces
decide: captured first calls, allocations that fail, results that depend on
how a call is cut."""
import gc

import numpy as np
import pytest

from hachiue_amd import Sampler, SamplerError, hip
from hachiue_amd import sampler as hs
from tests.conftest import _context
from tests.serving_util import Drafts, Graph, dev, expected, random_case, verify
from tests.test_gpu_lora import Adapters, check, run
from tests.test_oracle_lmhead import random_blocks

pytestmark = pytest.mark.gpu

@pytest.fixture(autouse=True)
def nothing_left():
    """No array that only a traceback still holds is left to be collected, and
    so freed, in a later capture."""
    yield
    gc.collect()


TYPES = {"q6_k": 14, "q4_k": 12, "q4_0": 2, "f32": 0}


class Projection:
    """Weights, adapters and rows of one gemv_lora_device call."""

    def __init__(self, fmt, hadamard, M, K=1024, N=3001, seed=50):
        rng = np.random.default_rng(seed + M)
        if fmt == "f32":
            raw = (rng.standard_normal((N, K)) / 32).astype(np.float32).view(np.uint8)
        else:
            raw = random_blocks(TYPES[fmt], N, K, rng)
        self.M, self.K, self.N = M, K, N
        self.dw = dev(np.ascontiguousarray(raw).reshape(-1))
        self.w = hs.weights(TYPES[fmt], N, K, self.dw.addr, None, hadamard, None)
        self.ad = Adapters(rng, "f16", 3, 12, K, N)
        self.x, self.slots = rng.standard_normal((M, K)).astype(np.float32), rng.integers(-1, 3, M).astype(np.int32)
        self.dx, self.ds = dev(self.x), dev(self.slots)
        self.cfg, self.u = hs.make_configs(dict(temperature=0.8, topK=30), M), dev(np.full(M, 0.5))
        self.tok = dev(np.full(M, -7, np.int32))
        self.y, self.plain = hip.DeviceArray((M, N), np.float32), hip.DeviceArray((M, N), np.float32)

    def gemv(self, ctx, st):
        ctx.gemv_device_ex(self.dx.addr, self.M, self.K, self.w, self.plain.addr, self.N, stream=st)

    def both(self, ctx, st):
        ctx.gemv_lora_device(self.dx.addr, self.M, self.K, self.w, self.ad.desc, self.ds.addr, self.y.addr,
                             self.N, stream=st)

    def sampled(self, ctx, st):
        ctx.lm_head_lora_sample_device(self.dx.addr, self.M, self.K, self.w, self.ad.desc, self.ds.addr,
                                       self.y.addr, self.N, None, None, self.cfg, self.u.addr, self.tok.addr,
                                       stream=st)

    def check(self, ctx, st):
        """The eager calls of a context, one after the other, are right."""
        for _ in range(3):
            self.y.upload(np.zeros((self.M, self.N), np.float32))
            self.plain.upload(np.zeros((self.M, self.N), np.float32))
            hip.synchronize()
            self.gemv(ctx, st)
            self.both(ctx, st)
            st.synchronize()
            check(self.ad, self.x, self.slots, self.plain.download(), self.y.download())
        return self.y.download()


def refused(call, *args):
    with pytest.raises(SamplerError) as e:
        call(*args)
    assert e.value.status == 4 and "capture" in str(e.value), str(e.value)


def captured(st, call, mode=0):
    """The call's graph.  (An array of an earlier test that is collected, and so
    freed, while a stream is captured would end the capture.)"""
    gc.collect()
    gc.disable()
    try:
        return Graph(st, call, mode)
    finally:
        gc.enable()


@pytest.mark.parametrize("mode", [0, 2])          # global, relaxed
@pytest.mark.parametrize("fmt,hadamard,M", [("q6_k", False, 1), ("q4_k", False, 2), ("q4_0", True, 5),
                                            ("q6_k", True, 1)])
def test_a_captured_first_projection_that_needs_workspace(fmt, hadamard, M, mode):
    """Nothing is allocated or cleared in a capture: the call is refused, its
    graph stays empty, the eager calls behind it count from zero, and once they
    have been made the capture holds the call."""
    p, st = Projection(fmt, hadamard, M), hip.Stream()
    with Sampler(0) as ctx:
        print(f"[gpu] first call captured {fmt} {hadamard} M={M} mode={mode}", flush=True)
        for call in (p.gemv, p.both):
            g = captured(st, lambda call=call: refused(call, ctx, st), mode)
            g.launch()
            st.synchronize()
            g.destroy()
        want = p.check(ctx, st)
        g = captured(st, lambda: p.both(ctx, st), mode)
        for _ in range(3):
            p.y.upload(np.zeros((M, p.N), np.float32))
            hip.synchronize()
            g.launch()
            st.synchronize()
            assert np.array_equal(p.y.download().view(np.uint32), want.view(np.uint32))
            assert np.array_equal(p.check(ctx, st).view(np.uint32), want.view(np.uint32))
        g.destroy()
    st.destroy()


def test_captured_sampling_with_adapters_is_refused():
    """Before anything is enqueued, for a fresh context and a used one."""
    p, st = Projection("f32", False, 5), hip.Stream()
    with Sampler(0) as ctx:
        for _ in range(2):
            g = captured(st, lambda: refused(p.sampled, ctx, st))
            p.y.upload(np.full((p.M, p.N), 7.0, np.float32))
            hip.synchronize()
            g.launch()
            st.synchronize()
            assert (p.y.download() == 7.0).all()
            g.destroy()
            p.sampled(ctx, st)
            st.synchronize()
            assert (p.tok.download() >= 0).all()
    st.destroy()


# ---- allocations that fail

def _reset():
    """A context created with injection off resets the process-wide counter."""
    _context({"HS_INJECT_HIP_FAILURE": "-1"}).close()


def test_room_for_the_call_alone():
    """A workspace that cannot have twice its size takes what the call needs;
    one that cannot have that either says so, and the call behind it works."""
    rng = np.random.default_rng(60)
    ad = Adapters(rng, "bf16", 2, 200, 16, 8)
    x = rng.standard_normal((5000, 16)).astype(np.float32)
    # the checked calls of a first call that grows: the growth, then the two
    # sizes that it asks for
    for n, grows in ((1, True), (0, False)):
        with _context({"HS_INJECT_HIP_FAILURE": str(n)}) as ctx:
            print(f"[gpu] the larger allocation fails ({n})", flush=True)
            if grows:
                y, b = run(ctx, ad, x, [1] * 5000)
                check(ad, x[-40:], [1] * 40, b[-40:], y[-40:])
            else:
                with pytest.raises(SamplerError) as e:
                    run(ctx, ad, x, [1] * 5000)
                assert e.value.status == 2
            x2 = rng.standard_normal((9000, 16)).astype(np.float32)
            y, b = run(ctx, ad, x2, [1] * 9000)
            check(ad, x2[-40:], [1] * 40, b[-40:], y[-40:])
    _reset()


def test_an_allocation_that_the_card_refuses():
    """A workspace larger than the card has: the call reports it, once, and the
    next call's launches do not report it again."""
    rng = np.random.default_rng(61)
    ad = Adapters(rng, "bf16", 1, 4, 8, 6)
    x = rng.standard_normal((3, 8)).astype(np.float32)
    big = hs.draft_batch(65535, 63, 65535 * 63, None, ad.arr[0].addr, ad.arr[0].addr, ad.arr[0].addr,
                         ad.arr[0].addr)
    rows = hs.distribution(hs.DIST_LOGITS, ad.arr[0].addr, 1 << 28)
    with Sampler(0) as ctx:
        print("[gpu] a workspace of 8 TB", flush=True)
        with pytest.raises(SamplerError) as e:     # (131072 parts of 16 bytes a row)
            ctx.verify_drafts_device(rows, None, 1 << 28, big)
        assert e.value.status == 2
        y, b = run(ctx, ad, x, [0, 0, -1])
        check(ad, x, [0, 0, -1], b, y)


def test_whatever_fails_leaves_the_counters_that_were_there():
    """Every checked call of a batch that makes the counters grow fails in turn
    (the clearing of the new ones among them): a captured call of a size that
    the context has from its creation goes on, and so does the large one."""
    rng = np.random.default_rng(62)
    V, lens, many = 3001, [3, 1, 0, 2], [8] * 600
    t, d, ids, u = random_case(rng, lens, V)
    total = sum(many)
    big_t = (rng.standard_normal((40, 300)) * 2).astype(np.float32)
    small, st = Drafts(lens, ids, u), hip.Stream()
    dt, dd = dev(t), dev(d)
    td, qd = hs.distribution(0, dt.addr, V), hs.distribution(0, dd.addr, V)
    row = np.arange(total + 600) % 40
    failures = 0
    for n in range(16):
        big = Drafts(many, rng.integers(0, 300, total), rng.random(total + 600))
        print(f"[gpu] verify, injected failure {n}", flush=True)
        with _context({"HS_INJECT_HIP_FAILURE": str(n)}) as ctx:
            try:
                live = verify(ctx, big, 300, big_t[row], None)
                injected = False
            except SamplerError as e:
                injected = True
                assert e.status == 2, str(e)
            hip.synchronize()
            small.tokens.upload(np.full(small.tokens.shape, -77, np.int32))
            hip.synchronize()
            g = captured(st, lambda: ctx.verify_drafts_device(td, qd, V, small.desc, stream=st))
            for _ in range(2):
                g.launch()
                st.synchronize()
                small.check(expected(small, t, d), f"captured after {n}")
            live = verify(ctx, big, 300, big_t[row], None)
            hip.synchronize()
            big.check(expected(big, big_t[row], None), f"large after {n}")
            g.launch()
            st.synchronize()
            small.check(expected(small, t, d), f"replayed behind {n}")
            g.destroy()
            del live
        if not injected and n > 4:
            break
        failures += injected
    _reset()
    assert failures >= 2, failures      # the counters' growth, their clearing
    st.destroy()


def test_the_next_stream_comes_behind_a_call_that_failed():
    """A timed call whose events cannot be made has cleared the counters, or
    rotated its rows, already: the next call on another stream waits for that."""
    rng = np.random.default_rng(63)
    total = 8 * 600
    rows = (rng.standard_normal((40, 300)) * 2).astype(np.float32)[np.arange(total + 600) % 40]
    a, b = hip.Stream(), hip.Stream()
    p = Projection("q4_0", True, 5)
    with Sampler(0) as ctx:
        want = p.check(ctx, a)
    verified = rotated = 0
    for n in range(12):
        big = Drafts([8] * 600, rng.integers(0, 300, total), rng.random(total + 600))
        print(f"[gpu] two streams, injected failure {n}", flush=True)
        with _context({"HS_INJECT_HIP_FAILURE": str(n)}) as ctx:
            ctx.set_timing(True)
            try:
                live = [verify(ctx, big, 300, rows, None, stream=a)]
            except SamplerError:
                verified += 1
            _reset()
            live = [verify(ctx, big, 300, rows, None, stream=b)]
            hip.synchronize()
            big.check(expected(big, rows, None), f"behind failure {n}")
        with _context({"HS_INJECT_HIP_FAILURE": str(n)}) as ctx:
            ctx.set_timing(True)
            try:
                p.both(ctx, a)
            except SamplerError:
                rotated += 1
            _reset()
            p.both(ctx, b)
            b.synchronize()
            assert np.array_equal(p.y.download().view(np.uint32), want.view(np.uint32)), n
        del live
    assert verified >= 4 and rotated >= 4, (verified, rotated)
    for st in (a, b):
        st.destroy()


# ---- how a call is cut

@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_row_in_calls_of_other_sizes(sampler, kind):
    """Four, three, two and one shares of K (1, 1100, 1400 and 4200 rows at rank
    64) and the second product through LDS (from 384 workgroups on) or not: each
    within the bound of binary32 sums, and the same bits for the same size."""
    rng = np.random.default_rng(80)
    K, N = 4096, 600
    ad = Adapters(rng, kind, 3, 64, K, N)
    x = rng.standard_normal((4200, K)).astype(np.float32)
    slots = rng.integers(-1, 3, 4200).astype(np.int32)
    slots[0] = 2
    for M in (1, 17, 1100, 1400, 4200):
        y, _ = run(sampler, ad, x[:M], slots[:M], None)
        rows = np.unique(np.concatenate([[0], rng.integers(0, M, 12), [M - 1]]))
        check(ad, x[rows], slots[rows], None, y[rows])
        # other neighbours, the same row
        order = np.concatenate([[0], 1 + rng.permutation(M - 1)])
        y2, _ = run(sampler, ad, x[order], slots[order], None)
        assert np.array_equal(y[order].view(np.uint32), y2.view(np.uint32)), M
