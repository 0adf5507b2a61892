"""GPU parity of the low-rank adapters with binary64, within what binary32
sums of the same terms can be off (serving_oracle.lora); then a whole
speculative step of adapters, projection and verification."""
import numpy as np
import pytest

from hachiue_amd import Sampler, SamplerError, hip
from hachiue_amd import sampler as hs
from hachiue_amd.decode import DecodeState
from oracle import pyoracle as o
from oracle import serving_oracle as so
from tests.serving_util import Drafts, Graph, dev, expected

pytestmark = pytest.mark.gpu

TYPES = {"f32": 0, "f16": 1, "bf16": 30}


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def stored(x, kind):
    """(the device's elements, their values)"""
    if kind == "f32":
        return np.ascontiguousarray(x, np.float32), np.asarray(x, np.float32)
    if kind == "f16":
        h = np.ascontiguousarray(x, np.float16)
        return h, h.astype(np.float32)
    u = bf16(x)
    return u, (u.astype(np.uint32) << 16).view(np.float32)


class Adapters:
    def __init__(self, rng, kind, count, rank, K, N, ranks=None, scales=True, garbage=True):
        a = rng.standard_normal((count, rank, K)) / np.sqrt(K)
        b = rng.standard_normal((count, N, rank))
        self.ranks = np.full(count, rank, np.int32) if ranks is None else np.asarray(ranks, np.int32)
        if garbage:      # behind an adapter's own ranks its stack holds anything
            for s in range(count):
                r = min(max(int(self.ranks[s]), 0), rank)
                a[s, r:], b[s, :, r:] = np.nan, np.inf
        ra, self.a = stored(a, kind)
        rb, self.b = stored(b, kind)
        self.scales = rng.uniform(0.5, 2, count).astype(np.float32) if scales else np.ones(count, np.float32)
        self.arr = [dev(ra), dev(rb), dev(self.scales), dev(self.ranks)]
        self.desc = hs.adapters(TYPES[kind], count, rank, K, N, self.arr[0].addr, self.arr[1].addr,
                                self.arr[2].addr if scales else None,
                                self.arr[3].addr if ranks is not None else None)
        self.count, self.K, self.N = count, K, N


def padded(x, ld, skew=0):
    p = np.full((x.shape[0], ld), np.nan, np.float32)
    p[:, :x.shape[1]] = x
    return dev(np.concatenate([np.zeros(skew, np.float32), p.reshape(-1)]))


def run(sampler, ad, x, slots, base="apart", pad=0, skew=0, stream=None):
    """y [M, N] with what surrounds its rows unchanged."""
    M, N = x.shape[0], ad.N
    ldx, ldb, ldy = ad.K + pad, N + 2 * pad, N + pad
    dx, ds = padded(x, ldx, skew), dev(np.asarray(slots, np.int32))
    y0 = np.full((M, N), 123.0, np.float32)
    rng = np.random.default_rng(M + N)
    b = rng.standard_normal((M, N)).astype(np.float32) if base else None
    db = padded(b, ldb, skew) if base == "apart" else None
    dy = padded(b if base == "in place" else y0, ldy, skew)
    print(f"[gpu] lora M={M} K={ad.K} N={N} rank={ad.desc.rank} type={ad.desc.type} count={ad.count} "
          f"base={base} pad={pad} skew={skew}", flush=True)
    at = dy.addr + 4 * skew
    d_base = {"apart": db.addr + 4 * skew if db else 0, "in place": at, None: None}[base]
    sampler.lora_device(dx.addr + 4 * skew, M, ldx, ad.desc, ds.addr, d_base,
                        ldy if base == "in place" else ldb, at, ldy, stream=stream)
    hip.synchronize()
    y = dy.download()[skew:].reshape(M, ldy)
    assert np.isnan(y[:, N:]).all()
    return y[:, :N], b


def check(ad, x, slots, base, y):
    want, bound = so.lora(x, ad.a, ad.b, ad.scales, ad.ranks, slots, base)
    err = np.abs(y - want)
    assert np.all(err <= bound), (float((err / bound).max()), np.argwhere(~(err <= bound))[:4])
    none = [m for m, s in enumerate(slots) if not 0 <= s < ad.count]
    if none:    # rows without an adapter: base to the bit
        b = np.zeros_like(y) if base is None else base
        assert np.array_equal(y[none].view(np.uint32), b[none].view(np.uint32))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K,N,rank,count", [
    (1, 1, 1, 1, 1), (1, 64, 257, 16, 3), (2, 33, 15, 5, 2), (15, 100, 64, 8, 4), (16, 128, 65, 17, 20),
    (17, 255, 1000, 32, 2), (33, 31, 63, 33, 5), (70, 7, 129, 64, 3), (5, 2049, 77, 100, 2),
    (20, 40, 16, 128, 30), (3, 520, 300, 200, 2), (40, 9, 5, 256, 4)])
def test_shapes(sampler, kind, M, K, N, rank, count):
    rng = np.random.default_rng(M * 31 + K + N + rank)
    ad = Adapters(rng, kind, count, rank, K, N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    slots = rng.integers(0, count, M)
    for base, pad, skew in (("apart", 0, 0), ("in place", 3, 1), (None, 4, 2)):
        y, b = run(sampler, ad, x, slots, base, pad, skew)
        check(ad, x, slots, b, y)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rank", [4, 6, 16, 40, 129])
def test_ranks_slots_and_scales(sampler, kind, rank):
    """Ranks of their own (0 and beyond the stack's among them), rows without
    an adapter, no scales."""
    rng = np.random.default_rng(rank)
    ranks = [rank, 0, 1, max(1, rank - 1), rank + 7, -2, (rank + 1) // 2]
    ad = Adapters(rng, kind, 7, rank, 96, 200, ranks=ranks)
    ad.ranks = np.clip(ad.ranks, 0, rank).astype(np.int32)
    x = rng.standard_normal((50, 96)).astype(np.float32)
    slots = np.concatenate([rng.integers(-2, 9, 44), [-1, 7, 2 ** 31 - 1, -2 ** 31, 0, 6]])
    for base in ("apart", "in place", None):
        y, b = run(sampler, ad, x, slots, base)
        check(ad, x, slots, b, y)
    plain = Adapters(rng, kind, 2, rank, 96, 200, scales=False)
    y, b = run(sampler, plain, x[:5], [0, 1, 1, -1, 0])
    check(plain, x[:5], [0, 1, 1, -1, 0], b, y)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rank,K,N", [(64, 300, 4100), (83, 17, 4353), (130, 256, 4096), (256, 64, 4097)])
def test_many_results_of_long_ranks(sampler, kind, rank, K, N):
    """The second product through LDS: chunks that an adapter's ranks fill, end
    in or do not reach, columns that end in a workgroup's tile, prompts beside
    rows without an adapter, and what is not finite."""
    rng = np.random.default_rng(rank + N)
    ranks = [rank, 0, rank // 2, 33, 1, rank - 1]
    ad = Adapters(rng, kind, 6, rank, K, N, ranks=ranks)
    M = 390
    x = rng.standard_normal((M, K)).astype(np.float32)
    slots = np.concatenate([np.repeat([0, 5, -1, 2], [100, 37, 9, 64]), rng.integers(-1, 7, 180)]).astype(np.int32)
    x[7, K // 2] = np.inf
    for base, pad, skew in (("apart", 1, 1), ("in place", 0, 0), (None, 3, 2)):
        y, b = run(sampler, ad, x, slots, base, pad, skew)
        fine = np.arange(M) != 7
        check(ad, x[fine], slots[fine], b[fine] if b is not None else None, y[fine])
        assert not np.isfinite(y[7]).any()
    # an adapter whose last row of B is not finite
    bad = ad.b.copy()
    bad[3, N - 1, 0] = np.nan
    ad.arr[1].upload(stored(bad, kind)[0])
    y, b = run(sampler, ad, x, slots)
    rows = fine & (slots != 3)
    check(ad, x[rows], slots[rows], b[rows], y[rows])
    assert np.isnan(y[fine & (slots == 3)][:, N - 1]).all()


def test_a_failed_allocation():
    """The workspace cannot grow: the call says so, the next one works."""
    import os
    rng = np.random.default_rng(12)
    ad = Adapters(rng, "bf16", 2, 200, 16, 8)
    x = rng.standard_normal((5000, 16)).astype(np.float32)
    old = os.environ.get("HS_INJECT_HIP_FAILURE")
    os.environ["HS_INJECT_HIP_FAILURE"] = "0"
    try:
        ctx = Sampler(0)
    finally:
        if old is None:
            del os.environ["HS_INJECT_HIP_FAILURE"]
        else:
            os.environ["HS_INJECT_HIP_FAILURE"] = old
    with ctx:
        with pytest.raises(SamplerError) as e:
            run(ctx, ad, x, [1] * 5000)
        assert e.value.status == 2
        y, b = run(ctx, ad, x, [1] * 5000)
        check(ad, x[-40:], [1] * 40, b[-40:], y[-40:])


def test_no_adapters_at_all(sampler):
    rng = np.random.default_rng(1)
    ad = Adapters(rng, "bf16", 1, 4, 8, 100)
    x = rng.standard_normal((20, 8)).astype(np.float32)
    y, b = run(sampler, ad, x, [-1] * 20)
    assert np.array_equal(y, b)
    ad.desc.count, ad.desc.a, ad.desc.b = 0, None, None
    for base in ("apart", "in place", None):
        y, b = run(sampler, ad, x, [0] * 20, base)
        assert np.array_equal(y, b if b is not None else np.zeros_like(y))


@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_not_finite_stays_in_its_rows(sampler, kind):
    """An infinity or NaN in one row's x, or one adapter's A or B, reaches no
    row of another adapter."""
    rng = np.random.default_rng(3)
    ad = Adapters(rng, kind, 4, 20, 70, 90)
    slots = np.array([0, 1, 2, 3, 0, 1, 2, 3, 0, -1, 2, 3, 0, 1, 2, -1, 3, 2], np.int32)
    x = rng.standard_normal((18, 70)).astype(np.float32)
    x[4, 3], x[9, 0], x[12, 69] = np.nan, np.inf, np.inf
    a = ad.a.copy()
    b = ad.b.copy()
    a[1, 2, 5], b[3, 7, 19] = np.inf, np.nan
    for arr, v in ((ad.arr[0], a), (ad.arr[1], b)):
        arr.upload(stored(v, kind)[0])
    y, base = run(sampler, ad, x, slots)
    fine = [m for m in range(18) if slots[m] in (0, 2) and np.isfinite(x[m]).all()]
    want, bound = so.lora(x[fine], ad.a, ad.b, ad.scales, ad.ranks, slots[fine], base[fine])
    assert np.all(np.abs(y[fine] - want) <= bound)
    assert np.array_equal(y[[9, 15]], base[[9, 15]])
    for m in (1, 5, 13, 4, 12):
        assert not np.isfinite(y[m]).any(), m
    for m in (3, 7, 11, 16):
        assert np.isnan(y[m, 7]) and np.isfinite(np.delete(y[m], 7)).all(), m


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rank,N", [(12, 77), (40, 300), (64, 98400)])
def test_scales_and_infinities(sampler, kind, rank, N):
    """Far from 1 the error stays relative (2^-100 keeps every term's last bit a
    normal number but for terms that are themselves that much smaller); an
    infinity times positive elements is one, a NaN one whatever its bits."""
    rng = np.random.default_rng(rank)
    ad = Adapters(rng, kind, 2, rank, 300, N)
    x = rng.standard_normal((5, 300)).astype(np.float32)
    slots = [1, 0, 0, 1, 1]
    for e in (-100, 100):
        y, _ = run(sampler, ad, np.ldexp(x, e).astype(np.float32), slots, None)
        check(ad, np.ldexp(x, e).astype(np.float32), slots, None, y)
    arr = [dev(stored(np.full(shape, 0.5), kind)[0]) for shape in ((2, rank, 300), (2, N, rank))]
    ad.arr, ad.desc = arr, hs.adapters(TYPES[kind], 2, rank, 300, N, arr[0].addr, arr[1].addr)
    x[0, 3] = np.array([0x7F800001], np.uint32).view(np.float32)[0]
    x[1, 299], x[2, 255], x[3, 8] = np.inf, -np.inf, np.nan
    y, _ = run(sampler, ad, x, slots, None)
    assert np.isnan(y[0]).all() and (y[1] == np.inf).all() and (y[2] == -np.inf).all()
    assert np.isnan(y[3]).all() and np.isfinite(y[4]).all()


def test_a_row_is_the_same_in_any_company(sampler):
    """Bit for bit, whatever rows and adapters share its tile."""
    rng = np.random.default_rng(4)
    ad = Adapters(rng, "bf16", 6, 24, 300, 500)
    x = rng.standard_normal((40, 300)).astype(np.float32)
    slots = rng.integers(-1, 6, 40)
    y, b = run(sampler, ad, x, slots, None)
    for rows in (np.arange(40)[::-1], np.array([7, 7, 3]), np.arange(5, 22)):
        y2, _ = run(sampler, ad, x[rows], slots[rows], None)
        assert np.array_equal(y[rows].view(np.uint32), y2.view(np.uint32))


def test_many_rows(sampler):
    """Prompts of several requests one after another, and the most rows that a
    call takes."""
    rng = np.random.default_rng(5)
    ad = Adapters(rng, "bf16", 5, 16, 64, 48)
    x = rng.standard_normal((1037, 64)).astype(np.float32)
    slots = np.repeat([3, -1, 0, 4, 1], [400, 17, 300, 19, 301])
    y, b = run(sampler, ad, x, slots)
    check(ad, x, slots, b, y)
    one = Adapters(rng, "f16", 2, 3, 2, 1)
    x = rng.standard_normal((65535, 2)).astype(np.float32)
    slots = (np.arange(65535) // 7 % 3 - 1).astype(np.int32)
    y, b = run(sampler, one, x, slots, "in place")
    s, t = slots >= 0, np.maximum(slots, 0)
    d = (np.einsum("mk,mjk->mj", x.astype(np.float64), one.a[t].astype(np.float64))
         * one.b[t, 0].astype(np.float64)).sum(-1) * one.scales[t]
    assert np.abs(y[:, 0] - b[:, 0] - np.where(s, d, 0)).max() < 1e-4
    with pytest.raises(SamplerError):
        sampler.lora_device(1 << 20, 65536, 2, one.desc, 4096, None, 0, 1 << 30, 1)


def test_offsets_past_32_bits(sampler):
    """The last adapter of stacks above 4 GiB, rows of y above 2^32 bytes
    apart."""
    rng = np.random.default_rng(6)
    K, N, rank, count = 4096, 70000, 256, 130
    small = Adapters(rng, "bf16", 1, rank, K, N)
    A = hip.DeviceArray(count * rank * K, np.uint16)
    B = hip.DeviceArray(count * N * rank, np.uint16)
    for big, one, size in ((A, small.arr[0], rank * K), (B, small.arr[1], N * rank)):
        hip.check(hip.runtime().hipMemcpy(big.addr + 2 * (count - 1) * size, one.addr, 2 * size, hip.D2D),
                  "hipMemcpy")
    x = rng.standard_normal((2, K)).astype(np.float32)
    ldy = (1 << 30) + 8
    dx, ds = dev(x), dev(np.array([count - 1, count - 1], np.int32))
    dy = hip.DeviceArray(ldy + N, np.float32)
    print("[gpu] lora far stacks", flush=True)
    ad = hs.adapters(30, count, rank, K, N, A.addr, B.addr)
    sampler.lora_device(dx.addr, 2, K, ad, ds.addr, None, 0, dy.addr, ldy)
    hip.synchronize()
    y = np.empty((2, N), np.float32)
    for m in range(2):
        hip.check(hip.runtime().hipMemcpy(y[m].ctypes.data, dy.addr + 4 * m * ldy, 4 * N, hip.D2H), "hipMemcpy")
    small.scales[:] = 1
    check(small, x, [0, 0], None, y)


@pytest.mark.parametrize("fmt,hadamard", [("f32", False), ("q6_k", False), ("q4_0", True)])
@pytest.mark.parametrize("M", [1, 5, 20])
def test_beside_the_projection(sampler, fmt, hadamard, M):
    """gemv_lora_device is the projection followed by the adapters; the
    lm_head's tokens are the sampler's on that."""
    wt = {"f32": 0, "q6_k": 14, "q4_0": 2}[fmt]
    rng = np.random.default_rng(M)
    K, N = 1024, 5003
    if fmt == "f32":
        raw = (rng.standard_normal((N, K)) / 32).astype(np.float32).view(np.uint8)
    else:
        from tests.test_oracle_lmhead import random_blocks
        raw = random_blocks(wt, N, K, rng)
    dw = dev(np.ascontiguousarray(raw).reshape(-1))
    w = hs.weights(wt, N, K, dw.addr, None, hadamard, None)
    ad = Adapters(rng, "f16", 3, 12, K, N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    slots = rng.integers(-1, 3, M).astype(np.int32)
    dx, ds = dev(x), dev(slots)
    plain, y = hip.DeviceArray((M, N), np.float32), hip.DeviceArray((M, N), np.float32)
    print(f"[gpu] gemv + lora {fmt} M={M}", flush=True)
    sampler.gemv_device_ex(dx.addr, M, K, w, plain.addr, N)
    sampler.gemv_lora_device(dx.addr, M, K, w, ad.desc, ds.addr, y.addr, N)
    hip.synchronize()
    check(ad, x, slots, plain.download(), y.download())
    cfg, u = hs.make_configs(dict(temperature=0.8, topK=30), M), dev(rng.random(M))
    t1, t2 = hip.DeviceArray(M, np.int32), hip.DeviceArray(M, np.int32)
    sampler.lm_head_lora_sample_device(dx.addr, M, K, w, ad.desc, ds.addr, plain.addr, N, None, None, cfg,
                                       u.addr, t1.addr)
    sampler.sample_device(y.addr, M, N, N, None, None, cfg, u.addr, t2.addr)
    hip.synchronize()
    assert np.array_equal(plain.download(), y.download()) and np.array_equal(t1.download(), t2.download())


def test_streams_timing_and_graphs():
    """Two streams on one context, timed calls, a captured projection with
    adapters replayed with eager calls between."""
    rng = np.random.default_rng(8)
    K, N, M = 512, 3001, 9
    ad = Adapters(rng, "bf16", 4, 16, K, N)
    w = dev((rng.standard_normal((N, K)) / 20).astype(np.float32))
    wt = hs.weights(0, N, K, w.addr)
    xs = [rng.standard_normal((M, K)).astype(np.float32) for _ in range(3)]
    slots = np.array([0, 1, 2, 3, -1, 0, 1, 1, 3], np.int32)
    ds, dx = dev(slots), dev(xs[0])
    y, y2 = hip.DeviceArray((M, N), np.float32), hip.DeviceArray((M, N), np.float32)
    st, other = hip.Stream(), hip.Stream()
    with Sampler(0) as ctx:
        print("[gpu] captured gemv + lora", flush=True)
        g = Graph(st, lambda: ctx.gemv_lora_device(dx.addr, M, K, wt, ad.desc, ds.addr, y.addr, N, stream=st))
        for x in xs:
            dx.upload(x)
            for _ in range(2):
                y.upload(np.zeros((M, N), np.float32))
                hip.synchronize()
                g.launch()
                st.synchronize()
                ctx.gemv_lora_device(dx.addr, M, K, wt, ad.desc, ds.addr, y2.addr, N, stream=other)
                other.synchronize()
                assert np.array_equal(y.download().view(np.uint32), y2.download().view(np.uint32))
            base = hip.DeviceArray((M, N), np.float32)
            ctx.gemv_device_ex(dx.addr, M, K, wt, base.addr, N, stream=st)
            st.synchronize()
            check(ad, x, slots, base.download(), y2.download())
            big = Adapters(rng, "bf16", 1, 100, 16, 8)          # the workspace grows
            bx = rng.standard_normal((9000, 16)).astype(np.float32)
            yb, bb = run(ctx, big, bx, [0] * 9000)
            check(big, bx[:50], [0] * 50, bb[:50], yb[:50])
        g.destroy()
        ctx.kernel_times()
        ctx.set_timing(True)
        for s in (st, other, st):
            ctx.lora_device(dx.addr, M, K, ad.desc, ds.addr, None, 0, y.addr, N, stream=s)
        hip.synchronize()
        ms, calls = ctx.kernel_times()
        assert calls == 3 and ms["lora_shrink_kernel"] > 0 and ms["lora_expand_kernel"] > 0
    for s in (st, other):
        s.destroy()


@pytest.mark.parametrize("fmt,hadamard,M", [("q6_k", False, 1), ("q4_0", True, 5)])
def test_captured_projection_before_a_larger_one(fmt, hadamard, M):
    """A graph keeps the addresses of the projection's own workspaces (the
    hand-over of split tiles, the rotated rows): calls that need larger ones
    leave them where they are."""
    from tests.test_oracle_lmhead import random_blocks
    wt = {"q6_k": 14, "q4_0": 2}[fmt]
    rng = np.random.default_rng(40 + M)
    K, N, more = 1024, 3001, 40
    dw = dev(np.ascontiguousarray(random_blocks(wt, N, K, rng)).reshape(-1))
    w = hs.weights(wt, N, K, dw.addr, None, hadamard, None)
    ad = Adapters(rng, "f16", 3, 12, K, N)
    x = rng.standard_normal((more, K)).astype(np.float32)
    dx, ds = dev(x), dev(rng.integers(-1, 3, more).astype(np.int32))
    y, yl = hip.DeviceArray((M, N), np.float32), hip.DeviceArray((more, N), np.float32)
    st = hip.Stream()
    with Sampler(0) as ctx:
        call = lambda: ctx.gemv_lora_device(dx.addr, M, K, w, ad.desc, ds.addr, y.addr, N, stream=st)
        print(f"[gpu] captured gemv + lora {fmt} M={M}, then M={more}", flush=True)
        call()
        st.synchronize()
        want = y.download()
        g = Graph(st, call)
        for _ in range(3):
            ctx.gemv_lora_device(dx.addr, more, K, w, ad.desc, ds.addr, yl.addr, N, stream=st)
            filler = [hip.DeviceArray((more, K), np.float32) for _ in range(4)]   # (in freed memory, if any)
            for f in filler:
                f.upload(np.full((more, K), np.nan, np.float32))
            y.upload(np.zeros((M, N), np.float32))
            hip.synchronize()
            g.launch()
            st.synchronize()
            assert np.array_equal(y.download().view(np.uint32), want.view(np.uint32))
        g.destroy()
    st.destroy()


@pytest.mark.parametrize("captured", [False, True])
def test_a_speculative_step_with_adapters(captured):
    """Hidden states of all drafted positions, through a shared lm_head with
    each request's adapter, verified against a draft's logits, into the
    histories: step after step, as a server runs them."""
    rng = np.random.default_rng(9)
    K, V, lens = 512, 4001, [3, 2, 3, 1]
    rows, total, seqs = sum(lens) + 4, sum(lens), 4
    raw = (rng.standard_normal((V, K)) / 12).astype(np.float32)
    dw = dev(raw)
    w = hs.weights(0, V, K, dw.addr)
    ad = Adapters(rng, "bf16", 3, 8, K, V)
    slots = np.repeat(np.array([2, -1, 0, 1], np.int32), np.array(lens) + 1)
    at = [i for i in range(rows) if i not in set(np.cumsum(np.array(lens) + 1) - 1)]
    stops = [17, 1234]
    st = hip.Stream()
    with Sampler(0) as ctx:
        state = DecodeState(ctx, [[1, 2], [], [5] * 140, [7]], stop_ids=stops, ring_cap=128)
        hist, done = [[1, 2], [], [5] * 140, [7]], [False] * 4
        dx, ds = hip.DeviceArray((rows, K), np.float32), dev(slots)
        logits, draft = hip.DeviceArray((rows, V), np.float32), hip.DeviceArray((total, V), np.float32)
        temps = np.array([0.8, 0.0, 1.0, 0.6])
        d_t, d_q = dev(temps), dev(np.maximum(temps, 0.5))
        b = Drafts(lens, np.zeros(total, np.int32), np.zeros(total + seqs))
        td = hs.distribution(hs.DIST_LOGITS, logits.addr, V, d_t.addr)
        qd = hs.distribution(hs.DIST_LOGITS, draft.addr, V, d_q.addr)

        def step():
            ctx.gemv_lora_device(dx.addr, rows, K, w, ad.desc, ds.addr, logits.addr, V, stream=st)
            state.verify_drafts(td, qd, V, b.desc, stream=st)

        hip.synchronize()
        print(f"[gpu] speculative steps, captured={captured}", flush=True)
        g = Graph(st, step) if captured else None
        for i in range(6):
            x = rng.standard_normal((rows, K)).astype(np.float32)
            y, bound = so.lora(x, ad.a, ad.b, ad.scales, ad.ranks, slots, None)
            near = (x[at] @ raw.T + y[at] + 0.3 * rng.standard_normal((total, V))).astype(np.float32)
            seq = np.repeat(np.arange(4), lens)
            ids = [so.draw(so.softmax(near[j], max(temps[seq[j]], 0.5)), rng.random()) for j in range(total)]
            if i == 3:
                ids[0] = 17
            b.drafts, b.u = np.array(ids, np.int32), rng.random(total + seqs)
            if i == 3:
                b.u[0] = 0.0
            b.d_drafts.upload(np.concatenate([b.drafts, [0]]).astype(np.int32))
            b.d_u.upload(np.concatenate([b.u, [0.0]]))
            dx.upload(x)
            draft.upload(near)
            hip.synchronize()
            g.launch() if captured else step()
            st.synchronize()
            got = logits.download()
            exact, mag = o.gemv_exact(o.W_F32 if hasattr(o, "W_F32") else 0, x, raw.view(np.uint8), V)
            assert np.all(np.abs(got - (exact + y)) <= 2.0 ** -16 * mag + bound + 2.0 ** -22 * np.abs(exact + y))
            want = expected(b, got, near, temps=temps, dtemps=np.maximum(temps, 0.5))
            toks, counts, _ = b.outputs()
            for s in range(4):
                tok, done[s] = so.append(want[s][0], hist[s], done[s], stops)
                assert counts[s] == len(tok) and toks[s].tolist() == tok + [-1] * (lens[s] + 1 - len(tok))
            assert state.lengths().tolist() == [len(h) for h in hist]
            assert ((state.done.download() != 0) == done).all()
        assert done[0]
        if g:
            g.destroy()
        state.free()
    st.destroy()
