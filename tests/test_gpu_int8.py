"""GPU parity of the 8-bit products with the exact integer sums, to the bit;
gated pairs within the activations' bounds; the paths that take I8 weights."""
import numpy as np
import pytest

from hachiue_amd import hip
from hachiue_amd import sampler as hs
from oracle import block_oracle as bo
from tests.block_util import ACT_IDS, Rows, Weight, quantised, random_q

pytestmark = pytest.mark.gpu
FLOATS = ["f32", "f16", "bf16"]
# tokens of each kernel, tiles' edges; one row of weights; K of one piece, tails
# of a step and of a stage
SIZES = [(1, 1, 16), (1, 100, 64), (2, 17, 48), (5, 300, 1040), (16, 129, 4096), (17, 64, 112), (31, 65, 528),
         (33, 1001, 272), (64, 250, 2064), (65, 127, 144), (77, 1001, 1040), (128, 130, 128), (129, 256, 256),
         (200, 513, 384), (500, 300, 400), (513, 257, 1296), (700, 1000, 112), (1030, 384, 640),
         # one token over tiles enough that a workgroup has several, and longer than
         # its kernel takes; K split among four waves; tiles of every form
         (1, 40001, 272), (1, 17000, 2064), (1, 300, 4096), (1, 300, 4112), (9, 8200, 80), (16, 12290, 48),
         (25, 8190, 1040), (16, 20000, 160), (50, 20001, 64), (64, 33000, 144), (64, 40000, 528),
         (300, 10000, 656), (70, 33000, 272), (260, 9000, 1200), (1001, 8190, 2576), (1901, 8190, 4112)]


def same(got, want, kind):
    """Bits of results, NaNs alike."""
    raw, val = bo.store(want, kind)
    g = bo.values(got, kind)
    ok = (np.ascontiguousarray(got).view(raw.dtype) == raw) | (np.isnan(g) & np.isnan(val)) | ((g == 0) & (val == 0))
    assert ok.all(), (np.argwhere(~ok)[:4], g[~ok][:4], val[~ok][:4])


def project(sampler, x, w, M, N, out="f32", bias=None, pad=0):
    Y = Rows(out, M, N, None, pad)
    b = None if bias is None else hip.DeviceArray.from_numpy(bias)
    print(f"[gpu] int8 product M={M} N={N} K={x.C} x={x.kind} out={out} bias={bias is not None}", flush=True)
    sampler.matmul_int_device(M, x.desc, w.desc, b.addr if b else None, Y.desc)
    hip.synchronize()
    return Y.get()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(sampler, M, N, K):
    rng = np.random.default_rng(M + N + K)
    w, (q, s) = Weight(rng, N, K), random_q(rng, M, K)
    same(project(sampler, quantised(q, s), w, M, N), bo.product(q, s, w.w, w.s), "f32")
    bias = rng.standard_normal(N).astype(np.float32)
    same(project(sampler, quantised(q, s, 32), w, M, N, "bf16", bias, 3), bo.product(q, s, w.w, w.s, bias), "bf16")


@pytest.mark.parametrize("M", [1, 20, 100, 600])
@pytest.mark.parametrize("out", FLOATS)
@pytest.mark.parametrize("x", FLOATS)
def test_float_rows_are_quantised_first(sampler, x, out, M):
    rng = np.random.default_rng(M)
    N, K = 130, 208
    w = Weight(rng, N, K)
    X, v = Rows.of(rng.standard_normal((M, K)) * 3, x, 5, 1)
    q, s = bo.quantise(v.astype(np.float32))
    same(project(sampler, X, w, M, N, out), bo.product(q, s, w.w, w.s), out)


# Rows that the product's workgroups quantise themselves (16 rows, 8192 elements, 4096
# channels at most) and their neighbours beyond each limit; tails of 16 elements.
FEW = [(1, 70, 4112), (1, 4096, 8192), (1, 70, 8208), (2, 4096, 4096), (2, 33, 4112), (3, 4097, 1040), (4, 300, 2048),
       (5, 777, 1040), (7, 800, 1104), (8, 16, 1024), (13, 50, 624), (15, 4096, 528), (16, 33, 16), (16, 100, 512),
       (16, 100, 528), (17, 40, 48)]


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("M,N,K", FEW)
def test_few_float_rows(sampler, M, N, K, x):
    """Rows anywhere, of zeros, with an infinity and a NaN among them."""
    rng = np.random.default_rng(M * K + N)
    w, up = Weight(rng, N, K), Weight(rng, N, K)
    v = rng.standard_normal((M, K)) * rng.uniform(0.1, 30, (M, 1))
    if M > 3:
        v[1], v[2, K - 1], v[M - 1, 0] = 0.0, np.inf, np.nan
    X, v = Rows.of(v, x, 3, 1)
    q, s = bo.quantise(v.astype(np.float32))
    bias = rng.standard_normal(N).astype(np.float32)
    same(project(sampler, X, w, M, N), bo.product(q, s, w.w, w.s), "f32")
    same(project(sampler, X, w, M, N, "f16", bias, 3), bo.product(q, s, w.w, w.s, bias), "f16")
    own, (q8, s8) = project(sampler, X, w, M, N, "i8"), bo.quantise(bo.product(q, s, w.w, w.s))
    assert np.array_equal(own[0], q8) and np.array_equal(own[1], s8, equal_nan=True)
    # a pair: the bits that the rows give when they come quantised
    pair = [gated(sampler, rows, w, up, "gelu", M, N) for rows in (X, quantised(q, s))]
    same(pair[0], pair[1], "f32")


@pytest.mark.parametrize("M,K", [(1, 65536), (40, 65536), (130, 32768), (600, 16384)])
def test_the_largest_sums(sampler, M, K):
    """Every product 2^14 or its negative: sums up to 2^30."""
    rng = np.random.default_rng(K)
    w = Weight(rng, 40, K, np.full((40, K), -128, np.int8))
    w.w[1::2, ::2] = 127
    w.arr[0].upload(w.w.reshape(-1))
    q = np.full((M, K), -128, np.int8)
    s = np.full(M, 2.0 ** -20, np.float32)
    same(project(sampler, quantised(q, s), w, M, 40), bo.product(q, s, w.w, w.s), "f32")


@pytest.mark.parametrize("M", [3, 50, 90, 600])
def test_scales_that_are_not_finite_stay_in_their_row_and_channel(sampler, M):
    rng = np.random.default_rng(M)
    N, K = 70, 96
    w, (q, s) = Weight(rng, N, K), random_q(rng, M, K)
    s[M - 1], s[1] = np.nan, 0.0
    w.s[5], w.s[69] = np.inf, np.nan
    w.arr[1].upload(w.s)
    same(project(sampler, quantised(q, s), w, M, N), bo.product(q, s, w.w, w.s), "f32")


@pytest.mark.parametrize("M", [1, 64, 200, 520])
def test_results_do_not_depend_on_the_rows_beside(sampler, M):
    rng = np.random.default_rng(M)
    N, K = 300, 640
    w, (q, s) = Weight(rng, N, K), random_q(rng, M, K)
    whole = project(sampler, quantised(q, s), w, M, N)
    for rows in ([0], list(range(M))[-17:]):
        part = project(sampler, quantised(q[rows], s[rows]), w, len(rows), N)
        assert np.array_equal(part.view(np.uint32), whole[rows].view(np.uint32))


@pytest.mark.parametrize("M", [1, 17, 65, 300])
def test_results_in_8_bits(sampler, M):
    rng = np.random.default_rng(M)
    N, K = 333, 80
    w, (q, s) = Weight(rng, N, K), random_q(rng, M, K)
    if M > 1:
        s[1] = np.nan
    got, scale = project(sampler, quantised(q, s), w, M, N, "i8", pad=3)
    wq, ws = bo.quantise(bo.product(q, s, w.w, w.s))
    assert np.array_equal(got, wq) and np.array_equal(scale, ws, equal_nan=True)


def gated(sampler, x, gate, up, act, M, N, out="f32", pad=0):
    Y = Rows(out, M, N, None, pad)
    print(f"[gpu] gated M={M} N={N} K={x.C} x={x.kind} act={act} out={out}", flush=True)
    sampler.gated_int_device(M, x.desc, gate.desc, up.desc, ACT_IDS[act], Y.desc)
    hip.synchronize()
    return Y.get()


def gated_bound(q, s, gate, up, act):
    g, u = (bo.product(q, s, v.w, v.s).astype(np.float64) for v in (gate, up))
    a, rel = bo.act(act, g)
    want = a * u
    return want, np.abs(want) * (rel + 2 * bo.U) + 2.0 ** -126 * (1 + np.abs(u))


@pytest.mark.parametrize("M,N,K", SIZES)
def test_gated(sampler, M, N, K):
    rng = np.random.default_rng(M * N + K)
    gate, up, (q, s) = Weight(rng, N, K), Weight(rng, N, K), random_q(rng, M, K)
    want, bound = gated_bound(q, s, gate, up, "silu")
    for out, pad in (("f32", 0), ("f16", 5)):
        got = bo.values(gated(sampler, quantised(q, s, pad * 16), gate, up, "silu", M, N, out, pad), out)
        err, b = np.abs(got - want), bo.rounded(bound, want, out)
        assert np.all(err <= b), (float((err / b).max()), np.argwhere(~(err <= b))[:4])


@pytest.mark.parametrize("M", [3, 70, 600])
@pytest.mark.parametrize("act", bo.ACTS)
def test_activations(sampler, act, M):
    rng = np.random.default_rng(M)
    N, K = 96, 64
    gate, up, (q, s) = Weight(rng, N, K), Weight(rng, N, K), random_q(rng, M, K)
    s[:] = np.exp2(rng.uniform(-6, 4, M))          # results near 0 and far from it
    want, bound = gated_bound(q, s, gate, up, act)
    got = gated(sampler, quantised(q, s), gate, up, act, M, N)
    err = np.abs(got - want)
    assert np.all(err <= bound), (float((err / bound).max()), np.argwhere(~(err <= bound))[:4])


@pytest.mark.parametrize("M", [1, 40, 100, 600])
def test_a_chain_of_a_feed_forward_block(sampler, M):
    """Norm, gated pair in 8 bits, projection back, norm: each step against the
    steps before it as they came out."""
    rng = np.random.default_rng(M)
    C, N = 272, 528
    x, r = (Rows.of(rng.standard_normal((M, C)), "bf16") for _ in range(2))
    nw = rng.normal(1, 0.2, C).astype(np.float32)
    d_nw = hip.DeviceArray.from_numpy(nw)
    gate, up, down = Weight(rng, N, C), Weight(rng, N, C), Weight(rng, C, N)
    mid, q, h, y, out = (Rows(k, M, c) for k, c in (("f32", C), ("i8", C), ("i8", N), ("f32", C), ("bf16", C)))
    n = hs.norm(hs.NORM_RMS, 1e-6, d_nw.addr)
    sampler.block_norm_device(hs.block_norm(M, C, x[0].desc, r[0].desc, sum=mid.desc, before=n, out=q.desc))
    sampler.gated_int_device(M, q.desc, gate.desc, up.desc, hs.ACT_SILU, h.desc)
    sampler.matmul_int_device(M, h.desc, down.desc, None, y.desc)
    sampler.block_norm_device(hs.block_norm(M, C, y.desc, mid.desc, 0.5, after=n, out=out.desc))
    hip.synchronize()
    assert np.array_equal(mid.get(), (x[1] + r[1]).astype(np.float32))
    qv, qs = q.get()
    want, bound = bo.norm(bo.RMS, 1e-6, nw.astype(np.float64), None, mid.get().astype(np.float64), np.zeros((M, C)))
    assert np.all(np.abs(qv * qs[:, None].astype(np.float64) - want) <= 0.5005 * qs[:, None] + bound)
    hv, hsc = h.get()
    want, bound = gated_bound(qv, qs, gate, up, "silu")
    assert np.all(np.abs(hv * hsc[:, None].astype(np.float64) - want) <= 0.5005 * hsc[:, None] + bound)
    same(y.get(), bo.product(hv, hsc, down.w, down.s), "f32")
    s, ds, o, do = bo.block_norm(y.get().astype(np.float64), (bo.RMS, 1e-6, nw.astype(np.float64), None), None,
                                 "none", 0.5, mid.get().astype(np.float64), (bo.NONE, 0, None, None))
    assert np.all(np.abs(bo.values(out.get(), "bf16") - o) <= bo.rounded(do, o, "bf16"))


@pytest.mark.parametrize("M", [1, 5, 70])
def test_the_lm_head_takes_8_bit_weights(sampler, M):
    """gemv_device_ex, then the whole call: the logits of the product, greedy tokens of them."""
    rng = np.random.default_rng(M)
    N, K = 4099, 4112                                    # (K above the other types' limit)
    w = Weight(rng, N, K)
    X, v = Rows.of(rng.standard_normal((M, K)), "f32", 7)
    want = bo.product(*bo.quantise(v.astype(np.float32)), w.w, w.s)
    Y, Z = Rows("f32", M, N, None, 1), Rows("f32", M, N)
    sampler.gemv_device_ex(X.desc.data, M, X.ld, w.desc, Y.desc.data, Y.ld)
    tok, u = hip.DeviceArray.from_numpy(np.full(M, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(M))
    sampler.lm_head_sample_device_ex(X.desc.data, M, X.ld, w.desc, Z.desc.data, N, None, None,
                                     dict(temperature=0.0), u.addr, tok.addr)
    hip.synchronize()
    same(Y.get(), want, "f32")
    same(Z.get(), want, "f32")
    assert np.array_equal(tok.download(), want.argmax(1))


@pytest.mark.parametrize("kind", ["f32", "i8"])
@pytest.mark.parametrize("M", [1, 6, 80])
def test_the_lm_head_behind_its_norm(sampler, kind, M):
    rng = np.random.default_rng(M)
    N, K = 1025, 512
    w = Weight(rng, N, K)
    x, r = (Rows.of(rng.standard_normal((M, K)), k) for k in ("bf16", "f32"))
    out, total = Rows(kind, M, K), Rows("f32", M, K)
    Z = Rows("f32", M, N)
    tok, u = hip.DeviceArray.from_numpy(np.full(M, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(M))
    block = hs.block_norm(M, K, x[0].desc, r[0].desc, sum=total.desc, before=hs.norm(hs.NORM_RMS), out=out.desc)
    sampler.lm_head_norm_sample_device(block, w.desc, Z.desc.data, N, None, None, dict(temperature=0.0),
                                       u.addr, tok.addr)
    hip.synchronize()
    assert np.array_equal(total.get(), (x[1] + r[1]).astype(np.float32))
    q, s = out.get() if kind == "i8" else bo.quantise(out.get())
    same(Z.get(), bo.product(q, s, w.w, w.s), "f32")
    assert np.array_equal(tok.download(), Z.get().argmax(1))


def test_the_norm_before_other_weights(sampler):
    rng = np.random.default_rng(9)
    M, N, K = 3, 700, 256
    wf = (rng.standard_normal((N, K)) / 16).astype(np.float32)
    dw = hip.DeviceArray.from_numpy(wf.reshape(-1))
    X, v = Rows.of(rng.standard_normal((M, K)), "f16")
    out, Z = Rows("f32", M, K), Rows("f32", M, N)
    tok, u = hip.DeviceArray.from_numpy(np.full(M, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(M))
    block = hs.block_norm(M, K, X.desc, before=hs.norm(hs.NORM_LAYER, 1e-5), out=out.desc)
    sampler.lm_head_norm_sample_device(block, hs.weights(0, N, K, dw.addr), Z.desc.data, N, None, None,
                                       dict(temperature=0.0), u.addr, tok.addr)
    hip.synchronize()
    h = out.get().astype(np.float64)
    want, mag = h @ wf.T.astype(np.float64), np.abs(h) @ np.abs(wf.T).astype(np.float64)
    assert np.all(np.abs(Z.get() - want) <= 2.0 ** -16 * mag)
    assert np.array_equal(tok.download(), Z.get().argmax(1))


def test_adapters_beside_8_bit_weights(sampler):
    from tests.test_gpu_lora import Adapters
    from oracle import serving_oracle as so
    rng = np.random.default_rng(4)
    M, N, K = 9, 515, 256
    w, ad = Weight(rng, N, K), Adapters(rng, "bf16", 3, 16, K, N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    slots = rng.integers(-1, 3, M).astype(np.int32)
    dx, ds, Y = hip.DeviceArray.from_numpy(x), hip.DeviceArray.from_numpy(slots), Rows("f32", M, N)
    sampler.gemv_lora_device(dx.addr, M, K, w.desc, ad.desc, ds.addr, Y.desc.data, N)
    hip.synchronize()
    base = bo.product(*bo.quantise(x), w.w, w.s)
    want, bound = so.lora(x, ad.a, ad.b, ad.scales, ad.ranks, slots, base)
    assert np.all(np.abs(Y.get() - want) <= bound)


def test_nothing_to_do(sampler):
    rng = np.random.default_rng(1)
    w, empty = Weight(rng, 8, 16), hs.weights(24, 0, 16, 0)
    X, Y = Rows("i8", 1, 16), Rows("f32", 1, 8)
    sampler.matmul_int_device(0, X.desc, w.desc, None, Y.desc)
    sampler.matmul_int_device(1, X.desc, empty, None, Y.desc)
    sampler.gated_int_device(0, X.desc, w.desc, w.desc, 1, Y.desc)
    hip.synchronize()
    Y.get()
