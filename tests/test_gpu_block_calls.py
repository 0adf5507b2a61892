"""Calls of norms between blocks and 8-bit products as programs make them: captured
and replayed, on several streams and from threads, timed, growing workspaces, with
failing HIP calls, and rows far apart or far into memory."""
import gc
import threading

import numpy as np
import pytest

from hachiue_amd import Sampler, SamplerError, hip
from hachiue_amd import sampler as hs
from oracle import block_oracle as bo
from tests.block_util import ACT_IDS, Rows, Weight, quantised, random_q
from tests.conftest import _context
from tests.serving_util import Graph
from tests.test_gpu_int8 import gated_bound, same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_left():
    """No array that only a traceback still holds is freed in a later capture."""
    yield
    gc.collect()


def captured(st, call, mode=0):
    gc.collect()
    gc.disable()
    try:
        return Graph(st, call, mode)
    finally:
        gc.enable()


class Block:
    """A feed-forward block: norm, gated pair in 8 bits, projection, norm."""

    def __init__(self, M, C=128, N=272, seed=0, x="i8"):
        rng = np.random.default_rng(seed + M)
        self.M, self.C, self.N = M, C, N
        self.x, self.xv = Rows.of(rng.standard_normal((M, C)), "bf16")
        self.r, self.rv = Rows.of(rng.standard_normal((M, C)), "f32")
        self.gate, self.up, self.down = Weight(rng, N, C), Weight(rng, N, C), Weight(rng, C, N)
        self.mid, self.q = Rows("f32", M, C), Rows(x, M, C)
        self.h, self.y, self.out = Rows("i8", M, N), Rows("f32", M, C), Rows("f32", M, C)
        n = hs.norm(hs.NORM_RMS, 1e-6)
        self.first = hs.block_norm(M, C, self.x.desc, self.r.desc, sum=self.mid.desc, before=n, out=self.q.desc)
        self.last = hs.block_norm(M, C, self.y.desc, self.mid.desc, 0.5, after=n, out=self.out.desc)

    def enqueue(self, ctx, st):
        ctx.block_norm_device(self.first, st)
        ctx.gated_int_device(self.M, self.q.desc, self.gate.desc, self.up.desc, hs.ACT_SILU, self.h.desc, st)
        ctx.matmul_int_device(self.M, self.h.desc, self.down.desc, None, self.y.desc, st)
        ctx.block_norm_device(self.last, st)

    def wipe(self):
        for r in (self.mid, self.q, self.h, self.y, self.out):
            r.arr.upload(r.before)
        hip.synchronize()

    def check(self):
        """The products to the bit from the rows as they came out."""
        assert np.array_equal(self.mid.get(), (self.xv + self.rv).astype(np.float32))
        q, s = self.q.get() if self.q.kind == "i8" else bo.quantise(self.q.get())
        h, hsc = self.h.get()
        want, bound = gated_bound(q, s, self.gate, self.up, "silu")
        assert np.all(np.abs(h * hsc[:, None].astype(np.float64) - want) <= 0.5005 * hsc[:, None] + bound)
        same(self.y.get(), bo.product(h, hsc, self.down.w, self.down.s), "f32")
        return [r.arr.download().tobytes() for r in (self.mid, self.q, self.h, self.y, self.out)]


@pytest.mark.parametrize("x", ["i8", "f32"])
@pytest.mark.parametrize("M", [1, 2, 20, 70, 300])
@pytest.mark.parametrize("mode", [0, 2])
def test_a_captured_block(M, x, mode):
    """A fresh context's first calls captured; replays between eager calls of
    another size give the same bytes."""
    b, other, st = Block(M, x=x), Block(M + 3, seed=1, x=x), hip.Stream()
    with Sampler(0) as ctx:
        print(f"[gpu] captured block M={M} x={x} mode={mode}", flush=True)
        g = captured(st, lambda: b.enqueue(ctx, st), mode)
        want = None
        for _ in range(3):
            b.wipe()
            g.launch()
            st.synchronize()
            got = b.check()
            assert want is None or got == want
            want = got
            other.enqueue(ctx, st)
            st.synchronize()
            other.check()
        b.wipe()
        b.enqueue(ctx, st)
        st.synchronize()
        assert b.check() == want
        g.destroy()
    st.destroy()


def test_a_captured_call_that_needs_a_larger_workspace():
    """Refused with nothing enqueued, until a call of its size has run; the old
    workspace stays for the graphs that hold it."""
    st = hip.Stream()
    rng = np.random.default_rng(3)
    M, K, N = 400, 8192, 40
    w = Weight(rng, N, K)
    X, v = Rows.of(rng.standard_normal((M, K)), "f16")
    Y, H = Rows("f32", M, N), Rows("i8", 12000, 64)
    small, small_v = Rows.of(rng.standard_normal((2, K)), "f16")
    small_y = Rows("f32", 2, N)
    w64 = Weight(rng, 64, 16)
    q64, s64 = random_q(rng, 12000, 16)
    xq = quantised(q64, s64)
    with Sampler(0) as ctx:
        print("[gpu] captured calls above the workspace", flush=True)

        def large():
            ctx.matmul_int_device(M, X.desc, w.desc, None, Y.desc, st)

        def results():
            ctx.matmul_int_device(12000, xq.desc, w64.desc, None, H.desc, st)

        g0 = captured(st, lambda: ctx.matmul_int_device(2, small.desc, w.desc, None, small_y.desc, st))
        for call in (large, results):
            def inside(call=call):
                with pytest.raises(SamplerError) as e:
                    call()
                assert e.value.status == 4 and "capture" in str(e.value)
            g = captured(st, inside)
            g.launch()
            st.synchronize()
            g.destroy()
        assert np.all(Y.arr.download() == Y.before)
        large()
        results()
        st.synchronize()
        same(Y.get(), bo.product(*bo.quantise(v.astype(np.float32)), w.w, w.s), "f32")
        g = captured(st, lambda: (large(), results()))
        for _ in range(2):
            Y.arr.upload(Y.before)
            hip.synchronize()
            g.launch()
            g0.launch()
            st.synchronize()
            same(Y.get(), bo.product(*bo.quantise(v.astype(np.float32)), w.w, w.s), "f32")
            same(small_y.get(), bo.product(*bo.quantise(small_v.astype(np.float32)), w.w, w.s), "f32")
        q, s = H.get()
        wq, ws = bo.quantise(bo.product(q64, s64, w64.w, w64.s))
        assert np.array_equal(q, wq) and np.array_equal(s, ws)
        g.destroy()
        g0.destroy()
    st.destroy()


def test_sampling_behind_a_norm_is_not_captured():
    rng = np.random.default_rng(1)
    st, w = hip.Stream(), Weight(rng, 300, 64)
    X, out, Z = Rows.of(rng.standard_normal((2, 64)), "f32")[0], Rows("f32", 2, 64), Rows("f32", 2, 300)
    tok, u = hip.DeviceArray.from_numpy(np.full(2, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(2))
    block = hs.block_norm(2, 64, X.desc, out=out.desc)
    with Sampler(0) as ctx:
        def inside():
            with pytest.raises(SamplerError) as e:
                ctx.lm_head_norm_sample_device(block, w.desc, Z.desc.data, 300, None, None, dict(temperature=0.0),
                                               u.addr, tok.addr, stream=st)
            assert e.value.status == 4
        g = captured(st, inside)
        g.launch()
        st.synchronize()
        g.destroy()
    assert np.all(tok.download() == -7) and np.all(out.arr.download() == out.before)
    st.destroy()


def test_streams_in_turn(sampler):
    """Each call on another stream than the one before, with no wait by the caller:
    the context orders them."""
    streams = [hip.Stream() for _ in range(3)] + [None]
    b = Block(90, x="f32")
    want = None
    for turn in range(6):
        b.wipe()
        for i, call in enumerate((lambda st: sampler.block_norm_device(b.first, st),
                                  lambda st: sampler.gated_int_device(b.M, b.q.desc, b.gate.desc, b.up.desc,
                                                                      hs.ACT_SILU, b.h.desc, st),
                                  lambda st: sampler.matmul_int_device(b.M, b.h.desc, b.down.desc, None, b.y.desc, st),
                                  lambda st: sampler.block_norm_device(b.last, st))):
            call(streams[(turn + i) % 4])
        hip.synchronize()
        got = b.check()
        assert want is None or got == want
        want = got
    for st in streams[:3]:
        st.destroy()


def test_threads_on_one_context_and_contexts_beside_each_other(sampler):
    blocks = [Block(m, seed=m, x="f32") for m in (1, 17, 80, 200)]
    want = []
    for b in blocks:
        b.enqueue(sampler, None)
        hip.synchronize()
        want.append(b.check())
        b.wipe()
    errors = []

    def work(ctx, mine):
        try:
            st = hip.Stream()
            for _ in range(5):
                for b in mine:
                    b.enqueue(ctx, st)
            st.synchronize()
            st.destroy()
        except Exception as e:          # noqa: BLE001 (reported below)
            errors.append(e)

    with Sampler(0) as second:
        threads = [threading.Thread(target=work, args=(sampler, blocks[:1])),
                   threading.Thread(target=work, args=(sampler, blocks[1:2])),
                   threading.Thread(target=work, args=(second, blocks[2:]))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    hip.synchronize()
    assert not errors
    assert [b.check() for b in blocks] == want


def test_timed_calls():
    b = Block(70, x="f32")
    with Sampler(0) as ctx:
        ctx.set_timing(True)
        b.enqueue(ctx, None)
        ms, calls = ctx.kernel_times()
        assert calls == 4
        assert all(ms[k] > 0 for k in ("block_norm_kernel", "int8_kernel", "requant_kernel"))
        ctx.set_timing(False)
    b.check()


def test_failing_hip_calls():
    """Each checked call of a block's calls fails once: the error is reported and
    the context's next calls are right."""
    b = Block(40, x="f32")
    seen = 0
    for n in range(40):
        ctx = _context({"HS_INJECT_HIP_FAILURE": str(n)})
        failed = 0
        try:
            b.wipe()
            for _ in range(2):
                try:
                    b.enqueue(ctx, None)
                    break
                except SamplerError as e:
                    assert e.status == 2
                    failed += 1
            hip.synchronize()
            b.check()
        finally:
            ctx.close()
        seen += failed
        if not failed:
            break
    _context({"HS_INJECT_HIP_FAILURE": "-1"}).close()     # (of the process: nothing is left to fail)
    assert seen >= 6


@pytest.mark.parametrize("M", [1, 5, 40, 129, 600])
def test_weights_and_rows_behind_4_gib(sampler, M):
    """Channels whose bytes, rows and results lie more than 2^32 apart."""
    N, K = 70000, 65536                   # 4.6 GB of weights
    if M > 5:
        N, K = 300, 1024
    ld = 1 << 23 if M <= 129 else 1 << 21
    far = hip.DeviceArray((max(M - 1, 0) * ld + K,), np.int8) if M > 1 else None
    rng = np.random.default_rng(M)
    q, s = random_q(rng, M, K)
    scales = hip.DeviceArray.from_numpy(s)
    if M > 1:
        for m in range(M):
            hip.check(hip.runtime().hipMemcpy(far.addr + m * ld, q[m].ctypes.data, K, 1))
        X = hs.rows(24, far.addr, ld, scales.addr)
    else:
        near = quantised(q, s)
        X = near.desc
    if M <= 5:
        w = hip.DeviceArray((N * K,), np.int8)
        hip.check(hip.runtime().hipMemset(w.addr, 1, N * K))
        last = rng.integers(-127, 128, (16, K)).astype(np.int8)
        hip.check(hip.runtime().hipMemcpy(w.addr + (N - 16) * K, last.ctypes.data, last.size, 1))
        host = np.concatenate([np.ones((1, K), np.int8), last])
        pick = [N - 17] + list(range(N - 16, N))
    else:
        host = rng.integers(-127, 128, (N, K)).astype(np.int8)
        w, pick = hip.DeviceArray.from_numpy(host.reshape(-1)), list(range(N))
    ws = rng.uniform(0.0005, 0.002, N).astype(np.float32)      # (no result above binary16's range)
    dws = hip.DeviceArray.from_numpy(ws)
    ldy = 1 << 29 if 1 < M <= 5 else N
    y = hip.DeviceArray(((M - 1) * ldy + N,), np.float16)
    print(f"[gpu] far rows M={M} N={N} K={K} ldx={ld} ldy={ldy}", flush=True)
    sampler.matmul_int_device(M, X, hs.weights(24, N, K, w.addr, dws.addr), None, hs.rows(1, y.addr, ldy))
    hip.synchronize()
    got = np.empty((M, N), np.float16)
    for m in range(M):
        hip.check(hip.runtime().hipMemcpy(got[m].ctypes.data, y.addr + 2 * m * ldy, 2 * N, 2))
    same(got[:, pick], bo.product(q, s, host, ws[pick]), "f16")


def test_more_rows_than_a_grids_dimension(sampler):
    M, C = 70001, 520
    rng = np.random.default_rng(1)
    x = rng.standard_normal((M, C)).astype(np.float32)
    X, O = Rows("f32", M, C, x), Rows("i8", M, C)
    sampler.block_norm_device(hs.block_norm(M, C, X.desc, out=O.desc))
    hip.synchronize()
    q, s = O.get()
    wq, wsc = bo.quantise(x)
    assert np.array_equal(q, wq) and np.array_equal(s, wsc)


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_one_weight_for_both_halves(sampler, act):
    rng = np.random.default_rng(2)
    M, N, K = 90, 200, 144
    w, (q, s) = Weight(rng, N, K), random_q(rng, M, K)
    Y = Rows("f32", M, N)
    x = quantised(q, s)
    sampler.gated_int_device(M, x.desc, w.desc, w.desc, ACT_IDS[act], Y.desc)
    hip.synchronize()
    want, bound = gated_bound(q, s, w, w, act)
    assert np.all(np.abs(Y.get() - want) <= bound)
