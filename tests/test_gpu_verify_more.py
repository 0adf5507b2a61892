"""Calls of the verification that its documentation allows: NaN of any bits,
neighbours of every kind in one call, rows read through one buffer."""
import numpy as np
import pytest

from hachiue_amd import hip
from hachiue_amd import sampler as hs
from tests.serving_util import Drafts, dev, expected, random_case, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [0x7F800001, 0xFF800001, 0x7FBFFFFF, 0x7FC00000, 0xFFFFFFFF])
@pytest.mark.parametrize("kind", ["logits", "probs"])
@pytest.mark.parametrize("T", [1.0, 0.0])
def test_nan_of_any_bits(sampler, bits, kind, T):
    """Signalling ones, negative ones: each weighs 0, wherever it stands."""
    rng = np.random.default_rng(bits & 0xFF)
    V, lens = 5000, [2, 0, 3, 1]
    for dkind in ("logits", "probs", None):
        t, d, ids, u = random_case(rng, lens, V, dkind is not None, kind, dkind or "logits")
        rows = [t] if d is None else [t, d]
        for r in rows:
            w = r.view(np.uint32)
            w[:, ::3] = bits
            w[:, 0] = w[:, V - 1] = bits
            w[1, :] = bits                       # a row of nothing else
            w[0, 1024:2048] = bits               # a part of nothing else
        b = Drafts(lens, ids, u)
        live = verify(sampler, b, V, t, d, kind, dkind or "logits", temps=np.full(4, T), dtemps=np.full(4, 0.8))
        hip.synchronize()
        with np.errstate(invalid="ignore"):
            want = expected(b, t, d, kind, dkind or "logits", np.full(4, T), np.full(4, 0.8))
        b.check(want, f"{bits:x} {dkind}")
        del live


def test_one_buffer_on_both_sides(sampler):
    """The draft's rows are the target's (a model that drafts for itself): every
    draft stands whatever its uniform below 1, at any temperature of both."""
    rng = np.random.default_rng(70)
    V, n, seqs = 9001, 4, 20
    t, _, _, u = random_case(rng, [n] * seqs, V)
    flat = t.reshape(seqs, n + 1, V)
    ids = flat[:, :n].argsort(-1)[:, :, -2].reshape(-1).astype(np.int32)
    # (rows of a sequence are n + 1 apart on the target's side, n on the draft's)
    d = np.ascontiguousarray(flat[:, :n].reshape(-1, V))
    u[:] = 1.0 - 2.0 ** -53
    b = Drafts([n] * seqs, ids, u)
    live = verify(sampler, b, V, t, d, temps=np.full(seqs, 0.7), dtemps=np.full(seqs, 0.7))
    hip.synchronize()
    assert (b.outputs()[1] == n + 1).all()
    b.check(expected(b, t, d, temps=np.full(seqs, 0.7), dtemps=np.full(seqs, 0.7)))
    del live
    # one sequence of one draft: the very same row
    one = Drafts([1], ids[:1], [1.0 - 2.0 ** -53, 0.5])
    buf = dev(np.stack([t[0], t[1]]))
    side = hs.distribution(hs.DIST_LOGITS, buf.addr, V)
    sampler.verify_drafts_device(side, side, V, one.desc)
    hip.synchronize()
    one.check(expected(one, t[:2], t[:1]))


def test_done_sequences_beside_all_others(sampler):
    """Sequences done before the call among running ones, in every kind of call,
    twice: nothing is left of one call in the next."""
    rng = np.random.default_rng(71)
    V, lens = 20011, [5, 3, 0, 8, 1, 8, 2]
    for dkind in ("logits", "probs", None):
        for kind in ("logits", "probs"):
            for _ in range(2):
                t, d, ids, u = random_case(rng, lens, V, dkind is not None, kind, dkind or "logits")
                b = Drafts(lens, ids, u)
                done = rng.integers(0, 2, 7).astype(np.int32)
                ring, ln, dn = dev(np.zeros((7, 128), np.int32)), dev(np.zeros(7, np.int64)), dev(done)
                st = hs.decode_state(ring.addr, 128, ln.addr, dn.addr)
                live = verify(sampler, b, V, t, d, kind, dkind or "logits", state=st)
                hip.synchronize()
                rows, counts, accept = b.outputs()
                for s, (tok, _) in enumerate(expected(b, t, d, kind, dkind or "logits")):
                    if done[s]:
                        assert counts[s] == 0 and (rows[s] == -1).all()
                        assert (accept[b.off[s]:b.off[s + 1]] == 0).all()
                    else:
                        assert rows[s].tolist() == tok + [-1] * (lens[s] + 1 - len(tok)), (kind, dkind, s)
                        assert ring.download()[s, :len(tok)].tolist() == tok
                    assert ln.download()[s] == (0 if done[s] else len(tok))
                del live
