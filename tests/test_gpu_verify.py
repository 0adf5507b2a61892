"""GPU parity of draft verification against whole rows with its binary64
definition: every token, count and acceptance probability.  A draw falls
within 1e-12 of a running sum's step about once in 1e7 draws, so tokens are
equal."""
import numpy as np
import pytest

from hachiue_amd import Sampler, SamplerError, hip
from hachiue_amd import sampler as hs
from hachiue_amd.decode import DecodeState
from oracle import serving_oracle as so
from tests.serving_util import Drafts, Graph, dev, expected, random_case, verify

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan
LOW = np.finfo(np.float32).min


def run(sampler, lens, vocab, seed, draft=True, kind="logits", dkind="logits", temps=None,
        dtemps=None, pad=0, skew=0, **kw):
    rng = np.random.default_rng(seed)
    t, d, ids, u = random_case(rng, lens, vocab, draft, kind, dkind, temps)
    b = Drafts(lens, ids, u, **kw)
    print(f"[gpu] verify seqs={len(lens)} drafts={list(lens)[:6]} vocab={vocab} {kind}/"
          f"{dkind if draft else None} pad={pad} skew={skew}", flush=True)
    live = verify(sampler, b, vocab, t, d, kind, dkind, temps, dtemps, pad, skew)
    hip.synchronize()
    b.check(expected(b, t, d, kind, dkind, temps, dtemps))
    return live


@pytest.mark.parametrize("vocab", [1, 2, 63, 256, 1001, 8191, 8192, 8193, 16385, 40007])
@pytest.mark.parametrize("draft", ["logits", "probs", None])
def test_vocabularies(sampler, vocab, draft):
    run(sampler, [3, 1, 4, 0, 2], vocab, vocab, draft is not None, "logits", draft or "logits")


@pytest.mark.parametrize("kind", ["logits", "probs"])
@pytest.mark.parametrize("dkind", ["logits", "probs", None])
@pytest.mark.parametrize("pad,skew", [(0, 0), (1, 0), (3, 1), (0, 3), (4, 2)])
def test_kinds_and_strides(sampler, kind, dkind, pad, skew):
    run(sampler, [2, 5, 0, 3, 1, 1, 4], 9001, pad * 5 + skew, dkind is not None, kind,
        dkind or "logits", pad=pad, skew=skew)


@pytest.mark.parametrize("seqs,drafts", [(1, 1), (1, 7), (2, 63), (64, 3), (33, 0), (300, 2)])
@pytest.mark.parametrize("draft", [True, False])
def test_batches(sampler, seqs, drafts, draft):
    run(sampler, [drafts] * seqs, 1003, seqs + drafts, draft, offsets=False, max_drafts=drafts)


def test_full_vocabulary(sampler):
    temps = np.array([0.7, 0.0, 1.3, 0.4])
    run(sampler, [4, 3, 4, 2], 151936, 1, temps=temps, dtemps=np.maximum(temps, 0.5))


@pytest.mark.parametrize("draft", ["logits", "probs", None])
def test_more_rows_than_start_at_once(sampler, draft):
    """Rows behind a rejection that was found in time are left out, rows in the
    middle of it given up: over several calls, whatever was left out."""
    temps = np.where(np.arange(64) % 9 == 4, 0.0, 0.9)
    for seed in range(3):
        run(sampler, [8] * 60 + [0, 3, 1, 5], 40007, seed, draft is not None, dkind=draft or "logits",
            temps=temps, dtemps=np.maximum(temps, 0.5))


def test_one_long_row(sampler):
    """More chunks than a wave has lanes."""
    run(sampler, [1, 0], 700001, 2)
    run(sampler, [1, 0], 700001, 3, kind="probs", dkind="probs")


def test_slack_behind_the_last_sequence(sampler):
    run(sampler, [2, 0, 3], 500, 4, max_drafts=6, slack=9)


def test_the_same_call_twice(sampler):
    """The counters are zero again after every outcome: rejected early, all
    accepted, greedy."""
    for seed in range(12):
        lens = [5, 2, 0, 7, 1]
        temps = np.array([0.9, 0.0, 1.1, 0.6, 0.0]) if seed % 2 else None
        run(sampler, lens, 20011, seed // 3, draft=seed % 4 != 3, temps=temps)


@pytest.mark.parametrize("T", [0.0, -1.0, NAN, 1e-300, 1e-3, 1.0, 50.0, 1e300, INF])
def test_temperatures(sampler, T):
    for dT in (T, 0.7):
        rng = np.random.default_rng(7)
        t, d, ids, u = random_case(rng, [3, 2, 0], 9000)
        ids[::2] = t[[0, 2, 5]].argmax(-1)          # some that a greedy target accepts
        b = Drafts([3, 2, 0], ids, u)
        temps, dtemps = np.full(3, T), np.full(3, dT)
        live = verify(sampler, b, 9000, t, d, temps=temps, dtemps=dtemps)
        hip.synchronize()
        b.check(expected(b, t, d, temps=temps, dtemps=dtemps), f"T {T}")
        del live


def masked_rows(V):
    rng = np.random.default_rng(3)
    base = (rng.standard_normal(V) * 2).astype(np.float32)

    def put(at, v):
        x = base.copy()
        x[at] = v
        return x
    return {
        "nothing": np.full(V, -INF), "all NaN": np.full(V, NAN), "lowest": np.full(V, LOW),
        "lowest but one": np.where(np.arange(V) == V - 2, 0, LOW),
        "one left": np.where(np.arange(V) == V // 2, 1.5, -INF),
        "last left": np.where(np.arange(V) == V - 1, -3e38, -INF),
        "NaN inside": put(slice(10, V, 7), NAN), "half masked": put(slice(0, V // 2), -INF),
        "infinite": put([5, V - 3], INF), "infinite and NaN": put([[1, 2], [3, V - 1]], [[INF, NAN]] * 2),
        "equal": np.zeros(V), "huge": put([0, V - 1], 3e38), "first maximum": put([9, 20, V - 1], 40),
    }


@pytest.mark.parametrize("name", list(masked_rows(64)))
@pytest.mark.parametrize("T", [1.0, 0.0])
@pytest.mark.parametrize("V", [300, 16400])
def test_masked_rows(sampler, name, T, V):
    """Each kind of row as the target's, the draft's and the last position's."""
    rows = {k: np.asarray(v, np.float32) for k, v in masked_rows(V).items()}
    plain, odd = rows["half masked"], rows[name]
    rng = np.random.default_rng(11)
    lens = [2, 2, 1, 0, 2]
    t = np.stack([odd, plain, plain, plain, odd, plain, plain, plain, odd, odd, odd, odd])
    d = np.stack([plain, plain, odd, odd, plain, odd, odd])
    ids = np.array([V - 1, V // 2, V - 2, V - 1, 5, V // 2, V - 1], np.int32)
    for seed in range(3):
        u = rng.random(12) if seed else np.zeros(12)
        for draft in (d, None):
            b = Drafts(lens, ids, u)
            temps = np.full(5, T)
            live = verify(sampler, b, V, t, draft, temps=temps, dtemps=np.ones(5))
            hip.synchronize()
            b.check(expected(b, t, draft, temps=temps, dtemps=np.ones(5)), f"{name} {seed}")
            del live


def test_odd_probabilities(sampler):
    """Negative, NaN, infinite and unnormalised probabilities, and rows of
    nothing."""
    rng = np.random.default_rng(5)
    V, lens = 9000, [2, 2, 1, 0]
    p = rng.dirichlet(np.full(V, 0.05), 9).astype(np.float32) * 3
    p[:, ::5] = -p[:, ::5]
    p[:, 1::7] = NAN
    p[:, 2::11] = INF
    p[3] = 0
    p[8] = NAN
    q = rng.dirichlet(np.full(V, 0.05), 5).astype(np.float32)
    q[:, 3::5] = NAN
    q[4] = 0
    ids = np.array([3, 4, 8998, 13, 18], np.int32)
    for draft in (q, None):
        for seed in range(4):
            b = Drafts(lens, ids, rng.random(9))
            live = verify(sampler, b, V, p, draft, "probs", "probs")
            hip.synchronize()
            b.check(expected(b, p, draft, "probs", "probs"), f"{seed}")
            del live


@pytest.mark.parametrize("draft", [True, False])
def test_ids_outside_the_vocabulary(sampler, draft):
    rng = np.random.default_rng(6)
    t, d, ids, u = random_case(rng, [4, 4], 8200, draft)
    ids[[1, 6]] = [-1, 8200]
    ids[7] = 2**31 - 1
    u[:4] = u[5:7] = 0.0
    b = Drafts([4, 4], ids, u)
    live = verify(sampler, b, 8200, t, d)
    hip.synchronize()
    want = expected(b, t, d)
    assert len(want[0][0]) <= 2 and len(want[1][0]) <= 3
    b.check(want)
    del live


def test_nothing_beyond_the_draft(sampler):
    """The target is the draft (or all of it is the rejected id): a rejection
    can then only be forced, and the token is drawn from the target itself."""
    V = 8300
    rng = np.random.default_rng(8)
    p = rng.dirichlet(np.full(V, 0.1), 2).astype(np.float32)
    only = np.zeros((2, V), np.float32)
    only[:, 77] = 0.25
    hot = np.full((2, V), -INF, np.float32)
    hot[:, 8200] = 3.0
    for kind, rows, x in (("probs", p, 4), ("probs", p, int(p[0].argmax())), ("probs", only, 77),
                          ("logits", np.log(p + np.float32(1e-9)), 5), ("logits", hot, 8200)):
        for draft in (rows[:1].copy(), None):
            for u1 in (0.0, 0.3, 1 - 2.0 ** -53):
                # (the acceptance uniform is out of its range: rejected whatever p is)
                b = Drafts([1], [x], [2.0, u1])
                live = verify(sampler, b, V, rows, draft, kind, kind)
                hip.synchronize()
                b.check(expected(b, rows, draft, kind, kind))
                del live


def test_draws_at_the_steps(sampler):
    """Equal weights and uniforms that lie exactly on steps of the running sum
    (sums of powers of two, so exact in any order): the step belongs to the
    next id."""
    V = 1 << 14
    t = np.zeros((8, V), np.float32)
    steps = np.array([0, 1, 4095, 8191, 8192, 8193, 12288, V - 1])
    b = Drafts([0] * 8, [], steps / V, max_drafts=1, slack=2)
    live = verify(sampler, b, V, t, None)
    hip.synchronize()
    rows, counts, _ = b.outputs()
    assert [int(r[0]) for r in rows] == steps.tolist() and (counts == 1).all()
    # beside one certain draft that is rejected, its id has no step
    t = np.zeros((2, V), np.float32)
    for x, u, want in ((0, 0.0, 1), (100, 100.5 / (V - 1), 101), (V - 1, 1 - 2.0 ** -53, V - 2),
                       (3, NAN, V - 1)):
        b = Drafts([1], [x], [0.9, u])
        live = verify(sampler, b, V, t, None)
        hip.synchronize()
        assert b.outputs()[0][0].tolist() == [want, -1], (x, u)
    del live


def test_uniforms_at_the_acceptance(sampler):
    """u q < p is strict: p = q accepts every u below 1, p = 0 none."""
    V = 256
    p = np.full((3, V), 1 / 256, np.float32)
    p[1, 7] = 0
    for u, want in ((1 - 2.0 ** -53, 2), (0.0, 2)):
        b = Drafts([2], [9, 7], [u, 0.0, 0.5])
        live = verify(sampler, b, V, p, np.full((2, V), 1 / 256, np.float32), "probs", "probs")
        hip.synchronize()
        assert b.outputs()[1].tolist() == [want]
    b = Drafts([1], [9], [0.5, 0.5])                 # a half below a quarter: exactly at the step
    live = verify(sampler, b, V, np.full((2, V), 1 / 256, np.float32),
                  np.full((1, V), 1 / 128, np.float32), "probs", "probs")
    hip.synchronize()
    rows, counts, acc = b.outputs()
    assert counts.tolist() == [1] and acc.tolist() == [0.5]
    del live


def test_offsets_past_32_bits(sampler):
    """Rows more than 2^32 bytes apart."""
    V, stride = 1000, (1 << 29) + 3
    rng = np.random.default_rng(9)
    t, d, ids, u = random_case(rng, [2], V)
    big_t, big_d = hip.DeviceArray(2 * stride + V, np.float32), hip.DeviceArray(stride + V, np.float32)
    for arr, rows in ((big_t, t), (big_d, d)):
        for i, r in enumerate(rows):
            src = np.ascontiguousarray(r)
            hip.check(hip.runtime().hipMemcpy(arr.addr + 4 * i * stride, src.ctypes.data, src.nbytes,
                                              hip.H2D), "hipMemcpy")
    b = Drafts([2], ids, u)
    print("[gpu] verify far rows", flush=True)
    sampler.verify_drafts_device(hs.distribution(0, big_t.addr, stride),
                                 hs.distribution(0, big_d.addr, stride), V, b.desc)
    hip.synchronize()
    b.check(expected(b, t, d))


def test_bad_offsets_stay_inside(sampler):
    """Offsets that fall, are negative or run past the arrays are cut to what
    the arrays hold."""
    V = 300
    rng = np.random.default_rng(10)
    t, d, ids, u = random_case(rng, [2, 2, 2], V)
    b = Drafts([2, 2, 2], ids, u)
    b.d_off.upload(np.array([-5, 1 << 40, 3, -(1 << 50)], np.int64))
    live = verify(sampler, b, V, t, d)
    hip.synchronize()
    tok, c = b.tokens.download(), b.counts.download()
    assert (tok[9:] == -77).all() and (c[3:] == -77).all() and ((c[:3] >= 1) & (c[:3] <= 3)).all()
    run(sampler, [2, 2, 2], V, 10)     # and the next call finds its counters at zero
    del live


def test_histories(sampler):
    """Tokens join the rings up to a stop id, sequences done before stay."""
    V, lens = 9000, [3, 2, 4, 0, 3, 1]
    rng = np.random.default_rng(12)
    prompts = [list(rng.integers(0, V, n)) for n in (0, 5, 127, 128, 300, 2)]
    steps = [random_case(rng, lens, V, noise=0.4) for _ in range(4)]
    # stop ids that come up: drafts that are accepted at once
    stops = [int(steps[1][2][0]), int(steps[2][2][5])]
    steps[1][3][0] = steps[2][3][3 + 2 + 2] = 0.0
    st = DecodeState(sampler, prompts, stop_ids=stops, ring_cap=128)
    hist, done = [list(p) for p in prompts], [False] * 6
    st.done.upload(np.array([0, 0, 0, 0, 0, 7], np.int32))
    done[5] = True
    for i, (t, d, ids, u) in enumerate(steps):
        b = Drafts(lens, ids, u)
        want = expected(b, t, d)
        live = verify(sampler, b, V, t, d, state=st.descriptor())
        hip.synchronize()
        rows, counts, _ = b.outputs()
        for s in range(6):
            tok, done[s] = so.append(want[s][0], hist[s], done[s], stops)
            assert counts[s] == len(tok), (i, s)
            assert rows[s].tolist() == tok + [-1] * (lens[s] + 1 - len(tok)), (i, s)
        ring, length = st.ring.download(), st.lengths()
        assert ((st.done.download() != 0) == done).all()
        for s in range(6):
            assert length[s] == len(hist[s])
            for j in range(max(0, len(hist[s]) - 128), len(hist[s])):
                assert ring[s, j % 128] == hist[s][j], (i, s, j)
        del live
    assert sum(done) >= 2
    with pytest.raises(ValueError):
        st.verify_drafts(None, None, V, hs.draft_batch(5, 1, 5, None, 1, 1, 1, 1))
    st.free()


def test_streams_and_timing(sampler):
    """The workspace goes from one stream's call to the other's in order, and
    timed calls report their kernels."""
    V, lens = 60013, [3, 4, 2]
    rng = np.random.default_rng(13)
    a, b2 = hip.Stream(), hip.Stream()
    todo = []
    sampler.kernel_times()
    sampler.set_timing(True)
    for i in range(6):
        t, d, ids, u = random_case(rng, lens, V)
        b = Drafts(lens, ids, u)
        live = verify(sampler, b, V, t, d, stream=(a, b2)[i % 2])
        todo.append((b, t, d, live))
    hip.synchronize()
    sampler.set_timing(False)
    ms, calls = sampler.kernel_times()
    assert calls == 6 and ms["verify_stats_kernel"] > 0 and ms["verify_final_kernel"] > 0
    for b, t, d, _ in todo:
        b.check(expected(b, t, d))
    a.destroy()
    b2.destroy()


@pytest.mark.parametrize("draft", ["logits", "probs", None])
def test_captured(draft):
    """A context's first call captured, replayed on new inputs with eager calls
    of other sizes between: the graph keeps its workspace."""
    V, lens = 30011, [3, 1, 0, 4]
    rng = np.random.default_rng(14)
    cases = [random_case(rng, lens, V, draft is not None, dkind=draft or "logits") for _ in range(4)]
    st, kinds = hip.Stream(), dict(logits=0, probs=1)
    with Sampler(0) as ctx:
        t, d, ids, u = cases[0]
        b = Drafts(lens, ids, u)
        dt, dd = dev(t), dev(d) if draft else None
        td = hs.distribution(0, dt.addr, V)
        qd = hs.distribution(kinds[draft], dd.addr, V) if draft else None
        print(f"[gpu] captured verify {draft}", flush=True)
        g = Graph(st, lambda: ctx.verify_drafts_device(td, qd, V, b.desc, stream=st))
        for i, (t, d, ids, u) in enumerate(cases):
            dt.upload(t)
            if draft:
                dd.upload(d)
            b.drafts, b.u = ids, u
            b.d_drafts.upload(np.concatenate([ids, [0]]).astype(np.int32))
            b.d_u.upload(np.concatenate([u, [0.0]]))
            hip.synchronize()
            for _ in range(2):
                b.tokens.upload(np.full(b.tokens.shape, -77, np.int32))
                hip.synchronize()
                g.launch()
                st.synchronize()
                b.check(expected(b, t, d, dkind=draft or "logits"), f"replay {i}")
            run(ctx, [40] * (10 + 30 * i), 9000 + i, i)   # (the workspace grows)
        big = Drafts([60] * 400, np.zeros(24000, np.int32), np.zeros(24400))
        g.destroy()
    with Sampler(0) as ctx:
        # a capture allocates nothing: a larger call is refused, the graph stays empty
        def refused():
            with pytest.raises(SamplerError) as e:
                ctx.verify_drafts_device(hs.distribution(0, dt.addr, 0x7FFFFFFF), None, 1 << 20, big.desc,
                                         stream=st)
            assert e.value.status == 4 and "capture" in str(e.value)
        g = Graph(st, refused)
        g.destroy()
    st.destroy()


def test_contexts_side_by_side():
    """Two contexts on two streams, two graphs: each has its own workspace."""
    V, lens = 50021, [4, 2, 3]
    rng = np.random.default_rng(15)
    ctx, st = [Sampler(0), Sampler(0)], [hip.Stream(), hip.Stream()]
    cases = [random_case(rng, lens, V) for _ in range(2)]
    graphs, batches, live = [], [], []
    for i in range(2):
        t, d, ids, u = cases[i]
        b = Drafts(lens, ids, u)
        arr = dev(t), dev(d)
        td, qd = hs.distribution(0, arr[0].addr, V), hs.distribution(0, arr[1].addr, V)
        hip.synchronize()
        graphs.append(Graph(st[i], lambda i=i, td=td, qd=qd, b=b: ctx[i].verify_drafts_device(
            td, qd, V, b.desc, stream=st[i])))
        batches.append(b)
        live.append((arr, td, qd))
    for _ in range(5):
        for g in graphs:
            g.launch()
    hip.synchronize()
    for b, (t, d, _, _) in zip(batches, cases):
        b.check(expected(b, t, d))
    for g in graphs:
        g.destroy()
    for i in range(2):
        ctx[i].close()
        st[i].destroy()


def test_threads_share_a_context():
    """Calls of several threads on streams of their own, of sizes that make the
    workspace grow: one after another on the context's workspace."""
    import threading
    rng = np.random.default_rng(16)
    V, todo = 20021, []
    for lens, draft in (([3, 5], "logits"), ([2] * 30, "probs"), ([4], None)):
        t, d, ids, u = random_case(rng, lens, V, draft is not None, "logits", draft or "logits")
        arr = dev(t), dev(d) if draft else None
        td = hs.distribution(0, arr[0].addr, V)
        qd = hs.distribution(0 if draft == "logits" else 1, arr[1].addr, V) if draft else None
        todo.append((Drafts(lens, ids, u), t, d, draft, td, qd, hip.Stream(), arr))
    hip.synchronize()
    failed = []
    with Sampler(0) as ctx:
        def calls(b, td, qd, st):
            try:
                for _ in range(25):
                    ctx.verify_drafts_device(td, qd, V, b.desc, stream=st)
            except Exception as e:   # noqa: BLE001 (reported below)
                failed.append(e)
        threads = [threading.Thread(target=calls, args=(b, td, qd, st)) for b, _, _, _, td, qd, st, _ in todo]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        hip.synchronize()
        assert not failed, failed
        for b, t, d, draft, *_ in todo:
            b.check(expected(b, t, d, "logits", draft or "logits"))
    for *_, st, _ in todo:
        st.destroy()
