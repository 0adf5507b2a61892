"""Draws and acceptance tests beside their steps: the weights are binary64 ones.

Rows of a few live ids, uniforms just below and just above the running sums' steps
(or p / q).  What the kernels can be off by, in units of 2^-53 of the row's
whole: a weight 2^d by 1.1 and by 3 |d| ln 2 (log2(e), its quotient by T and d are
rounded), by 4 more where it goes from its part's maximum to the row's; a
probability by 2 (the reciprocal, the product); sums of L live ids by 3 L on the
way to a part's, a row's and a thread's, and by L in the draw; u times the whole by
2.  With L = 6 and |d| <= 8 / 0.8 / ln 2 < 15: 64.3 * 1.11e-16 = 7.2e-15, and a
residual by two rows' errors over its own whole R, 1.5e-14 / R.  The uniforms are
2e-14 / R off the steps, which 80-bit arithmetic gives to 1e-18; u q < p is
tested 4e-14 of itself off, with two rows' errors between.
"""
import numpy as np
import pytest

from hachiue_amd import hip
from tests.serving_util import Drafts, verify

pytestmark = pytest.mark.gpu

OFF = 2e-14
W = np.longdouble
assert np.finfo(W).eps < 1e-18


def row(rng, V, live):
    x = np.full(V, -np.inf, np.float32)
    x[live] = rng.uniform(-4.0, 4.0, len(live)).astype(np.float32)
    return x


def softmax(x, T):
    x = x.astype(W)
    w = np.exp((x - x.max()) / W(T))
    return w / w.sum()


def steps(r):
    """(uniform, id) just below and above every inner step of a running sum."""
    ids = np.flatnonzero(r > 0)
    total = r.sum()
    at = np.cumsum(r[ids]) / total
    out = []
    for i in range(len(ids) - 1):
        if r[ids[i]] > 1e-6 * total and r[ids[i + 1]] > 1e-6 * total:
            out += [(float(at[i] - W(OFF) / total), int(ids[i])), (float(at[i] + W(OFF) / total), int(ids[i + 1]))]
    return out


@pytest.mark.parametrize("T", [1.0, 0.9, 1.7])
@pytest.mark.parametrize("V", [700, 9000])
def test_draws_beside_their_steps(sampler, V, T):
    """The one more token behind drafts that all stand (none here)."""
    rng = np.random.default_rng(int(V + 10 * T))
    rows, us, want = [], [], []
    for _ in range(40):
        x = row(rng, V, rng.choice(V, 6, replace=False))
        for u, v in steps(softmax(x, T)):
            rows.append(x)
            us.append(u)
            want.append(v)
    n = len(rows)
    b = Drafts([0] * n, [], us, max_drafts=1, slack=n)
    live = verify(sampler, b, V, np.stack(rows), None, temps=np.full(n, T))
    hip.synchronize()
    got = np.array([int(r[0]) for r in b.outputs()[0]])
    assert n > 200 and np.array_equal(got, want), (n, int((got != np.array(want)).sum()))
    del live


@pytest.mark.parametrize("T,dT", [(1.0, 1.0), (0.8, 1.3)])
@pytest.mark.parametrize("draft", [True, False])
def test_residuals_beside_their_steps(sampler, draft, T, dT):
    """One draft that is rejected, the token from what is left: p beyond q, or p
    without the draft."""
    rng = np.random.default_rng(int(10 * T + dT) + draft)
    V, t, d, ids, us, want = 5000, [], [], [], [], []
    for _ in range(60):
        live = rng.choice(V, 6, replace=False)
        x, y = row(rng, V, live), row(rng, V, live)
        p, q = softmax(x, T), softmax(y, dT)
        if draft:
            reject = live[np.argmin(p[live] - q[live])]
            r = np.maximum(p - q, 0)
        else:
            reject = live[0]
            r = p.copy()
            r[reject] = 0
        if r.sum() < 0.1:
            continue
        for u, v in steps(r):
            t += [x, x]
            d.append(y)
            ids.append(reject)
            us += [1.0 - 2.0 ** -53, u]
            want.append(v)
    n = len(ids)
    b = Drafts([1] * n, ids, us)
    keep = verify(sampler, b, V, np.stack(t), np.stack(d) if draft else None, temps=np.full(n, T),
                  dtemps=np.full(n, dT) if draft else None)
    hip.synchronize()
    rows, counts, _ = b.outputs()
    got = np.array([int(r[0]) for r in rows])
    assert n > 100 and (counts == 1).all() and np.array_equal(got, want), int((got != np.array(want)).sum())
    del keep


@pytest.mark.parametrize("draft", [True, False])
def test_acceptance_beside_its_step(sampler, draft):
    """u q < p just below and just above u = p / q."""
    rng = np.random.default_rng(3 + draft)
    V, t, d, ids, us, want = 3000, [], [], [], [], []
    for _ in range(300):
        live = rng.choice(V, 6, replace=False)
        x, y = row(rng, V, live), row(rng, V, live)
        p, q = softmax(x, 0.9), softmax(y, 1.1)
        i = live[0]
        ratio = p[i] / q[i] if draft else p[i]
        if not 1e-5 < ratio < 0.999:
            continue
        for sign in (-1, 1):
            t += [x, x]
            d.append(y)
            ids.append(i)
            us += [float(ratio * (1 + W(sign * 2 * OFF))), 0.5]
            want.append(2 if sign < 0 else 1)
    n = len(ids)
    b = Drafts([1] * n, ids, us)
    keep = verify(sampler, b, V, np.stack(t), np.stack(d) if draft else None, temps=np.full(n, 0.9),
                  dtemps=np.full(n, 1.1) if draft else None)
    hip.synchronize()
    counts = b.outputs()[1]
    assert n > 100 and np.array_equal(counts, want), int((counts != np.array(want)).sum())
    del keep


@pytest.mark.parametrize("draft", [None, 1500, 700, 2999])
def test_a_uniform_of_0_where_weights_underflow(sampler, draft):
    """A part whose sum is a denormal number while each of its ids' probabilities
    rounds to 0: u = 0 takes the first id that has one, never a masked id."""
    V, low = 3000, np.float32(-744.2)          # exp: 2^-1074, a third of which is 0
    x = np.full(V, -np.inf, np.float32)
    x[5:1024] = low
    x[1500:1503] = 0.0
    x[2990:] = low
    if draft is None:
        b, want, rows = Drafts([0, 0], [], [0.0, 0.0], max_drafts=1, slack=2), 1500, [x, x]
    else:      # a certain draft, rejected: what is left of p without it
        b, rows = Drafts([1, 1], [draft] * 2, [1.0 - 2.0 ** -53, 0.0] * 2), [x] * 4
        want = 1501 if draft == 1500 else 1500
    live = verify(sampler, b, V, np.stack(rows), None)
    hip.synchronize()
    assert [int(r[0]) for r in b.outputs()[0]] == [want] * 2
    del live
