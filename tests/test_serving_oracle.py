"""The binary64 forms of draft verification that the kernels are compared
with, against what verification promises: whatever the draft's distribution,
the token after a prefix is distributed as the target's.  Then the host checks
of the entry points, which come before a context is touched, so without a
GPU."""
import ctypes

import numpy as np
import pytest

from hachiue_amd import sampler as hs
from oracle import serving_oracle as so


def first_token_distribution(p, q, steps=4000):
    """The distribution of the first emitted token over a draft from q, an
    acceptance uniform and a final uniform (both integrated on a grid)."""
    out = np.zeros(p.size)
    grid = (np.arange(steps) + 0.5) / steps
    for x in range(p.size):
        share = q[x] if q is not None else (1.0 if x == 1 else 0.0)
        if share == 0:
            continue
        qx = q[x] if q is not None else 1.0
        a = np.mean(grid * qx < p[x])
        out[x] += share * a
        if a < 1:
            # any rejecting uniform, the final one over the grid
            for u in grid[::40]:
                t, _ = so.verify([p, p], None if q is None else [q], [x], [0.9999999, u])
                assert len(t) == 1
                out[t[0]] += share * (1 - a) / len(grid[::40])
    return out


@pytest.mark.parametrize("q", [[0.1, 0.2, 0.3, 0.4], [0.4, 0.3, 0.2, 0.1], [0.0, 1.0, 0.0, 0.0], None])
def test_the_tokens_are_the_targets(q):
    p = np.array([0.35, 0.05, 0.2, 0.4])
    got = first_token_distribution(p, None if q is None else np.array(q))
    # two grids: 1/4000 on each acceptance, 1/100 on each final draw's cuts
    assert np.abs(got - p).max() < 0.012


def test_lists_agree_with_whole_rows():
    rng = np.random.default_rng(4)
    for _ in range(50):
        V, n = 12, 3
        p, q = rng.dirichlet(np.ones(V), n + 1), rng.dirichlet(np.ones(V), n)
        x, u = rng.integers(0, V, n), rng.random(n + 1)
        ids = np.arange(V)
        want, acc = so.verify(list(p), list(q), x, u)
        got, acc2 = so.verify_lists([(ids, r, V, 0) for r in p], [(ids, r, V, 0) for r in q], x, u)
        assert got == want and np.allclose(acc, acc2)


def test_softmax_of_masked_rows():
    inf = np.inf
    assert so.softmax([-inf, np.nan]).tolist() == [0, 0]
    assert so.softmax([inf, 0, inf]).tolist() == [0.5, 0, 0.5]
    assert so.softmax([1, 3, 3], 0.0).tolist() == [0, 1, 0]
    low = np.finfo(np.float32).min
    assert np.allclose(so.softmax([low, low, -inf]), [0.5, 0.5, 0])


# ---- refusals (before the context is looked at)

P = 4096   # an address that no call below gets to use


def batch(**kw):
    d = dict(seqs=2, max_drafts=3, n_drafts=6, d_offsets=None, d_drafts=P, d_uniforms=P, d_tokens=P,
             d_counts=P)
    d.update(kw)
    return hs.draft_batch(*d.values())


def rows(**kw):
    d = dict(kind=0, d_data=P, row_stride=100)
    d.update(kw)
    return hs.distribution(*d.values())


def state(**kw):
    d = dict(d_ring=P, ring_cap=128, d_len=P, d_done=P)
    d.update(kw)
    return hs.decode_state(*d.values())


def refused(rc, text, status=1):
    assert rc == status and text in hs.lib().hs_last_error().decode(), (rc, hs.lib().hs_last_error())


BATCHES = [(dict(seqs=-1), "seqs", 1), (dict(max_drafts=-1), "max_drafts", 1),
           (dict(max_drafts=64, n_drafts=128), "max_drafts", 1), (dict(n_drafts=7), "n_drafts", 1),
           (dict(n_drafts=-1), "n_drafts", 1), (dict(n_drafts=5), "without offsets", 1),
           (dict(d_drafts=0), "drafts", 1), (dict(d_uniforms=0), "uniforms", 1),
           (dict(d_tokens=0), "tokens", 1), (dict(d_counts=0), "counts", 1),
           (dict(seqs=65536, max_drafts=0, n_drafts=0), "65535", 4)]
STATES = [(dict(d_ring=0), "ring"), (dict(d_len=0), "len"), (dict(d_done=0), "done"),
          (dict(ring_cap=127), "ring_cap"), (dict(ring_cap=(1 << 29) + 1), "ring_cap"),
          (dict(d_stop_ids=0, n_stop=1), "stop ids"), (dict(d_stop_ids=P, n_stop=1025), "n_stop")]


@pytest.mark.parametrize("kw,text,status", BATCHES)
def test_bad_batches(kw, text, status):
    L = hs.lib()
    refused(L.hs_verify_drafts_device(None, rows(), None, 100, batch(**kw), None, None), text, status)
    c = hs.candidates(8, P, P, P)
    refused(L.hs_verify_candidates_device(None, c, None, batch(**kw), None, None), text, status)


@pytest.mark.parametrize("kw,text", STATES)
def test_bad_states(kw, text):
    L = hs.lib()
    refused(L.hs_verify_drafts_device(None, rows(), None, 100, batch(), state(**kw), None), text)
    c = hs.candidates(8, P, P, P)
    refused(L.hs_verify_candidates_device(None, c, None, batch(), state(**kw), None), text)


def test_bad_rows():
    L, b = hs.lib(), batch()

    def call(t, d, vocab=100):
        return L.hs_verify_drafts_device(None, t, d, vocab, b, None, None)

    refused(call(None, None), "null target")
    refused(L.hs_verify_drafts_device(None, rows(), None, 100, None, None, None), "null draft batch")
    for v in (0, -1, (1 << 28) + 1):
        refused(call(rows(row_stride=1 << 40), None, v), "vocab")
    for kw, text in ((dict(kind=2), "kind"), (dict(kind=-1), "kind"), (dict(d_data=0), "rows"),
                     (dict(d_data=P + 2), "aligned"), (dict(row_stride=99), "stride")):
        refused(call(rows(**kw), None), text)
        refused(call(rows(), rows(**kw)), text)
    refused(call(rows(), rows()), "null context")
    assert L.hs_verify_drafts_device(None, rows(), None, 100, batch(seqs=0, n_drafts=0), None, None) == 0


def test_bad_lists():
    L, b = hs.lib(), batch()
    good = hs.candidates(8, P, P, P)

    def call(t, d):
        return L.hs_verify_candidates_device(None, t, d, b, None, None)

    refused(call(None, None), "null target")
    for c in (hs.candidates(0, P, P, P), hs.candidates(4097, P, P, P)):
        refused(call(c, None), "stride")
        refused(call(good, c), "stride")
    for c in (hs.candidates(8, 0, P, P), hs.candidates(8, P, 0, P), hs.candidates(8, P, P, 0)):
        refused(call(c, None), "must be given")
        refused(call(good, c), "must be given")
    refused(call(good, good), "null context")


def test_bad_adapters():
    L = hs.lib()

    def ad(**kw):
        d = dict(atype=30, count=2, rank=16, K=64, N=50, d_a=P, d_b=P)
        d.update(kw)
        return hs.adapters(*d.values())

    def call(a, M=3, ldx=64, slots=P, x=P, base=0, ldb=50, y=1 << 20, ldy=50):
        return L.hs_lora_device(None, x, M, ldx, a, slots, base or None, ldb, y, ldy, None)

    refused(call(None), "null adapters")
    refused(call(ad(atype=2)), "type 2", 4)
    for kw in (dict(count=-1), dict(rank=0), dict(K=0), dict(N=-1)):
        refused(call(ad(**kw)), "adapters of count")
    refused(call(ad(rank=257)), "rank 257", 4)
    for kw in (dict(K=(1 << 30) + 1), dict(N=2 ** 31 - 1)):
        refused(call(ad(**kw), ldx=1 << 31, ldy=1 << 31), "above 2^30", 4)
    refused(call(ad(), M=-1), "M must")
    refused(call(ad(), M=65536), "65535", 4)
    for kw in (dict(x=None), dict(slots=None), dict(y=None)):
        refused(call(ad(), **kw), "must not be null")
    for kw in (dict(d_a=0), dict(d_b=0)):
        refused(call(ad(**kw)), "must not be null")
    for kw in (dict(ldx=63), dict(ldy=49), dict(base=P, ldb=49)):
        refused(call(ad(), **kw), "strides")
    for kw in (dict(x=P + 2), dict(y=P + 1), dict(base=P + 2)):
        refused(call(ad(), **kw), "aligned")
    refused(call(ad(d_a=P + 1)), "aligned")
    refused(call(ad(atype=0, d_b=P + 2)), "aligned")
    y = 1 << 20
    refused(call(ad(), base=y, ldb=60, ldy=61), "row stride")
    refused(call(ad(), base=y - 4, ldb=50), "overlaps")
    refused(call(ad(), base=y + 4 * 149, ldb=50), "overlaps")
    refused(call(ad(), base=y + 4 * 150, ldb=50), "null context")
    refused(call(ad(), base=y, ldb=50), "null context")
    assert call(ad(), M=0) == 0 and call(ad(N=0), M=5, ldy=0) == 0
    # beside weights
    w = hs.weights(0, 50, 64, P)
    cfg = hs.make_configs(None, 3)

    def both(w, a, **kw):
        k = dict(cfg=cfg, u=P, tok=P, hist=None, off=None)
        k.update(kw)
        r1 = L.hs_gemv_lora_device(None, P, 3, 64, w, a, P, y, 50, None)
        e1 = hs.lib().hs_last_error()
        r2 = L.hs_lm_head_lora_sample_device(None, P, 3, 64, w, a, P, y, 50, k["hist"], k["off"],
                                             k["cfg"], k["u"], k["tok"], None)
        return (r1, e1), r2

    for w_, a_, text in ((None, ad(), b"null weights"), (w, ad(N=49), b"beside weights"),
                         (w, ad(K=32), b"beside weights"), (w, ad(rank=300), b"rank 300")):
        (r1, e1), r2 = both(w_, a_)
        assert r1 == r2 != 0 and text in e1 and text in hs.lib().hs_last_error()
    for kw, text in ((dict(u=None), "uniforms"), (dict(tok=None), "tokens"), (dict(hist=P), "history")):
        refused(both(w, ad(), **kw)[1], text)
    refused(both(w, ad())[1], "null context")


def test_structures_match_the_header():
    assert ctypes.sizeof(hs.DistributionC) == 32
    assert ctypes.sizeof(hs.DraftBatchC) == 64
    assert ctypes.sizeof(hs.DecodeStateC) == 48
    assert ctypes.sizeof(hs.CandidatesC) == 40
    assert ctypes.sizeof(hs.AdaptersC) == 56
