"""GPU parity of draft verification against candidate lists with its binary64
definition, on lists made here and on those that the sampler writes."""
import numpy as np
import pytest

from hachiue_amd import Sampler, hip
from hachiue_amd import sampler as hs
from hachiue_amd.decode import DecodeState
from hachiue_amd.sampler import make_configs
from oracle import serving_oracle as so
from tests.serving_util import Drafts, Graph, dev

pytestmark = pytest.mark.gpu

NAN, INF = np.nan, np.inf


class Lists:
    """Candidate lists on the device, entries behind each list garbage."""

    def __init__(self, ids, probs, kept, tokens=None):
        self.ids, self.probs = np.asarray(ids, np.int32), np.asarray(probs, np.float32)
        self.kept = np.asarray(kept, np.int32)
        self.tokens = None if tokens is None else np.asarray(tokens, np.int32)
        self.arr = [dev(self.ids), dev(self.probs), dev(self.kept)]
        if tokens is not None:
            self.arr.append(dev(self.tokens))
        self.desc = hs.candidates(self.ids.shape[1], *(a.addr for a in self.arr))

    def row(self, r):
        return (self.ids[r], self.probs[r], int(self.kept[r]),
                0 if self.tokens is None else int(self.tokens[r]))


def expected(b, t, d):
    out = []
    for s in range(b.seqs):
        o, n = int(b.off[s]), int(b.lens[s])
        tl = [t.row(o + s + i) for i in range(n + 1)]
        dl = [d.row(o + i) for i in range(n)] if d is not None else None
        out.append(so.verify_lists(tl, dl, b.drafts[o:o + n].tolist(), b.u[o + s:o + s + n + 1]))
    return out


def check(b, want):
    rows, counts, accept = b.outputs()
    for s, (tok, acc) in enumerate(want):
        n = int(b.lens[s])
        if tok is None:
            assert counts[s] == -1 and (rows[s] == -1).all(), s
            assert (accept[b.off[s]:b.off[s + 1]] == 0).all()
            continue
        assert counts[s] == len(tok) and rows[s].tolist() == tok + [-1] * (n + 1 - len(tok)), (s, tok, rows[s])
        got = accept[b.off[s]:b.off[s + 1]]
        assert np.all(np.abs(got - acc) <= 2.0 ** -24 * np.abs(acc) + 1e-13), (s, got, acc)


def random_lists(rng, rows, k, vocab, pools=None, garbage=True):
    """Sorted lists of up to k of `vocab` ids, cut short at random."""
    pool = max(2, min(vocab, 2 * k))
    if pools is None:
        pools = [rng.choice(vocab, pool, replace=False) for _ in range(rows)]
    ids, probs = np.full((rows, k), 12345, np.int32), np.full((rows, k), NAN, np.float32)
    kept = np.zeros(rows, np.int32)
    for r in range(rows):
        n = min(k, len(pools[r]))
        ids[r, :n] = rng.permutation(pools[r])[:n]
        p = np.sort(rng.dirichlet(np.full(n, 0.6)))[::-1]
        probs[r, :n] = p
        kept[r] = rng.integers(1, n + 1)
        if garbage:
            ids[r, kept[r]:] = rng.integers(-5, 99, k - kept[r])
            probs[r, kept[r]:] = NAN
    return Lists(ids, probs, kept, rng.integers(0, vocab, rows)), pools


def case(rng, lens, k, kd, vocab, draft=True):
    lens = np.asarray(lens)
    total, seqs = int(lens.sum()), len(lens)
    at = [int(lens[:b].sum()) + b + i for b, n in enumerate(lens) for i in range(n)]
    t, pools = random_lists(rng, total + seqs, k, vocab)
    d = random_lists(rng, total, kd, vocab, [pools[i] for i in at])[0] if draft and total else None
    x = []
    for i in range(total):
        l = d.row(i) if d is not None else t.row(at[i])
        x.append(int(l[0][rng.integers(0, l[2])]))
    return t, d, np.array(x, np.int32), rng.random(total + seqs)


@pytest.mark.parametrize("k,kd", [(1, 1), (2, 7), (20, 20), (64, 40), (65, 1), (255, 256), (257, 300),
                                  (1024, 1024), (4096, 4096), (4000, 3)])
@pytest.mark.parametrize("draft", [True, False])
def test_lists(sampler, k, kd, draft):
    for seed in range(3):
        rng = np.random.default_rng(k + kd + seed)
        lens = [3, 0, 5, 1] if seed else [2]
        t, d, x, u = case(rng, lens, k, kd, max(50, 3 * k), draft)
        b = Drafts(lens, x, u)
        print(f"[gpu] lists {k} {kd} {draft}", flush=True)
        sampler.verify_candidates_device(t.desc, d.desc if d else None, b.desc)
        hip.synchronize()
        check(b, expected(b, t, d))


@pytest.mark.parametrize("seqs,drafts", [(1, 63), (300, 3), (70, 0)])
def test_batches(sampler, seqs, drafts):
    rng = np.random.default_rng(seqs)
    t, d, x, u = case(rng, [drafts] * seqs, 12, 12, 100)
    b = Drafts([drafts] * seqs, x, u, offsets=False, max_drafts=drafts)
    sampler.verify_candidates_device(t.desc, d.desc if d else None, b.desc)
    hip.synchronize()
    check(b, expected(b, t, d))


def test_rows_without_lists(sampler):
    """Greedy rows (kept 0: their token), rows left unresolved, lists not kept
    whole, a null tokens array, probabilities that are none."""
    rng = np.random.default_rng(2)
    lens = [2] * 12
    t, d, x, u = case(rng, lens, 10, 10, 40)
    x[2] = t.tokens[3]
    t.kept[[0, 3, 8, 20]] = 0, 0, -3, 0
    t.kept[[12, 16]] = 11, 2 ** 31 - 1          # not kept whole
    t.tokens[20] = -1                           # unresolved
    d.kept[[4, 9, 14]] = 0, 11, 0
    d.tokens[14] = x[14]
    t.probs[27, :3] = [NAN, -1.0, INF]
    t.probs[30:33] = 0
    d.probs[22] = NAN
    for toks in (True, False):
        tt = Lists(t.ids, t.probs, t.kept, t.tokens if toks else None)
        dd = Lists(d.ids, d.probs, d.kept, d.tokens if toks else None)
        for draft in (dd, None):
            b = Drafts(lens, x, u)
            sampler.verify_candidates_device(tt.desc, draft.desc if draft else None, b.desc)
            hip.synchronize()
            want = expected(b, tt, draft)
            assert any(w[0] is None for w in want) and any(w[0] is not None for w in want)
            check(b, want)


def test_histories(sampler):
    rng = np.random.default_rng(3)
    lens = [2, 3, 0, 1, 2]
    st = DecodeState(sampler, [[1], [2] * 200, [], [3], [5]], stop_ids=[7, 9], ring_cap=130)
    hist, done = [[1], [2] * 200, [], [3], [5]], [False] * 5
    for step in range(8):
        t, d, x, u = case(rng, lens, 6, 6, 15)
        if step == 3:
            t.kept[-1] = 9                      # the last sequence's last position
            t = Lists(t.ids, t.probs, t.kept, t.tokens)
        b = Drafts(lens, x, u)
        st.verify_candidates(t.desc, d.desc, b.desc)
        hip.synchronize()
        rows, counts, _ = b.outputs()
        for s, (tok, _) in enumerate(expected(b, t, d)):
            if tok is None and not done[s]:
                assert counts[s] == -1 and (rows[s] == -1).all()
                continue
            tok, done[s] = so.append(tok or [], hist[s], done[s], [7, 9])
            assert counts[s] == len(tok) and rows[s].tolist() == tok + [-1] * (lens[s] + 1 - len(tok))
        ring, n = st.ring.download(), st.lengths()
        for s in range(5):
            assert n[s] == len(hist[s])
            assert all(ring[s, j % 130] == hist[s][j] for j in range(max(0, n[s] - 130), n[s]))
    assert any(done)
    st.free()


@pytest.mark.parametrize("topk", [1, 20, 64, 300, 1024])
def test_the_samplers_own_lists(sampler, topk):
    """Target and draft rows sampled with candidate outputs (penalties, top-k,
    top-p, greedy rows, masked rows), then verified on the lists that this
    left."""
    rng = np.random.default_rng(topk)
    V, seqs, n = 3001, 6, 3
    rows = seqs * (n + 1)
    logits = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    logits[5] = -INF
    at = [s * (n + 1) + i for s in range(seqs) for i in range(n)]
    near = (logits[at] + rng.standard_normal((len(at), V)) * 0.5).astype(np.float32)
    cfg = [dict(temperature=0.0 if s == 2 else 0.9, topK=topk, topP=0.9, repetitionPenalty=1.2)
           for s in range(seqs)]
    hist = rng.integers(0, V, 10 * rows).astype(np.int32)
    cap = min(4096, max(64, topk))

    def lists(x, cfgs):
        R = len(cfgs)
        arr = [dev(x), dev(hist[:10 * R]), dev(np.arange(R + 1, dtype=np.int64) * 10), dev(rng.random(R))]
        ids, probs = hip.DeviceArray((R, cap), np.int32), hip.DeviceArray((R, cap), np.float32)
        kept, tok = hip.DeviceArray(R, np.int32), hip.DeviceArray(R, np.int32)
        sampler.sample_device(arr[0].addr, R, V, V, arr[1].addr, arr[2].addr, make_configs(cfgs, R),
                              arr[3].addr, tok.addr, cand_stride=cap, d_cand_ids=ids.addr,
                              d_cand_probs=probs.addr, d_cutoff=kept.addr)
        hip.synchronize()
        return Lists(ids.download(), probs.download(), kept.download(), tok.download())

    t = lists(logits, [cfg[r // (n + 1)] for r in range(rows)])
    d = lists(near, [cfg[r // n] for r in range(seqs * n)])
    assert (t.kept[2 * (n + 1):3 * (n + 1)] == 0).all()
    b = Drafts([n] * seqs, d.tokens, rng.random(rows))
    sampler.verify_candidates_device(t.desc, d.desc, b.desc)
    hip.synchronize()
    want = expected(b, t, d)
    check(b, want)
    # a greedy sequence's tokens are the target's own greedy tokens
    tok = want[2][0]
    assert tok == t.tokens[2 * (n + 1):2 * (n + 1) + len(tok)].tolist()


def test_captured():
    rng = np.random.default_rng(5)
    lens = [2, 0, 4]
    cases = [case(rng, lens, 30, 30, 90) for _ in range(3)]
    st = hip.Stream()
    with Sampler(0) as ctx:
        t, d, x, u = cases[0]
        b = Drafts(lens, x, u)
        g = Graph(st, lambda: ctx.verify_candidates_device(t.desc, d.desc, b.desc, stream=st))
        for t2, d2, x, u in cases:
            for mine, new in ((t, t2), (d, d2)):
                for a, v in zip(mine.arr, (new.ids, new.probs, new.kept, new.tokens)):
                    a.upload(v)
            b.drafts, b.u = x, u
            b.d_drafts.upload(np.concatenate([x, [0]]).astype(np.int32))
            b.d_u.upload(np.concatenate([u, [0.0]]))
            hip.synchronize()
            for _ in range(2):
                g.launch()
                st.synchronize()
                check(b, expected(b, t2, d2))
            other = hip.Stream()               # an eager call on another stream goes on
            ctx.verify_candidates_device(t.desc, d.desc, b.desc, stream=other)
            other.synchronize()
            check(b, expected(b, t2, d2))
            other.destroy()
        g.destroy()
    st.destroy()
