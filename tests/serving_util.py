"""Helpers of the GPU tests of draft verification and adapters."""
from __future__ import annotations

import ctypes

import numpy as np

from hachiue_amd import hip
from hachiue_amd import sampler as hs
from oracle import serving_oracle as so

KINDS = {"logits": hs.DIST_LOGITS, "probs": hs.DIST_PROBS}
GUARD = 5


def dev(a):
    return hip.DeviceArray.from_numpy(np.ascontiguousarray(a))


class Graph:
    """A captured call (or several) and its replays."""

    def __init__(self, stream, enqueue, mode=0):
        R, vp = hip.runtime(), ctypes.c_void_p
        R.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
        R.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
        R.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
        R.hipGraphLaunch.argtypes = [vp, vp]
        R.hipGraphExecDestroy.argtypes = R.hipGraphDestroy.argtypes = [vp]
        self.stream, self.graph, self.ex = stream, vp(), vp()
        hip.check(R.hipStreamBeginCapture(stream.handle, mode), "hipStreamBeginCapture")
        try:
            enqueue()
        finally:
            hip.check(R.hipStreamEndCapture(stream.handle, ctypes.byref(self.graph)),
                      "hipStreamEndCapture")
        hip.check(R.hipGraphInstantiate(ctypes.byref(self.ex), self.graph, None, None, 0),
                  "hipGraphInstantiate")

    def launch(self):
        hip.check(hip.runtime().hipGraphLaunch(self.ex, self.stream.handle), "hipGraphLaunch")

    def destroy(self):
        R = hip.runtime()
        if self.ex.value:
            R.hipGraphExecDestroy(self.ex)
        R.hipGraphDestroy(self.graph)


class Drafts:
    """A ragged batch on the device, its outputs with a guard behind them."""

    def __init__(self, lens, drafts, u, max_drafts=None, slack=0, offsets=True):
        lens = np.asarray(lens)
        self.lens, self.seqs = lens, len(lens)
        self.off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
        self.total = int(self.off[-1])
        n = self.total + slack
        self.max_drafts = int(lens.max()) if max_drafts is None else max_drafts
        n = min(n, self.seqs * self.max_drafts)
        self.drafts, self.u = np.asarray(drafts, np.int32), np.asarray(u, np.float64)
        assert self.drafts.size == self.total and self.u.size == self.total + self.seqs
        pad = n - self.total
        self.d_off = dev(self.off) if offsets else None
        self.d_drafts = dev(np.concatenate([self.drafts, np.zeros(pad + 1, np.int32)]))
        self.d_u = dev(np.concatenate([self.u, np.zeros(pad + 1)]))
        self.tokens = dev(np.full(n + self.seqs + GUARD, -77, np.int32))
        self.counts = dev(np.full(self.seqs + GUARD, -77, np.int32))
        self.accept = dev(np.full(n + GUARD, -77.0, np.float32))
        self.desc = hs.draft_batch(self.seqs, self.max_drafts, n,
                                   self.d_off.addr if offsets else None, self.d_drafts.addr,
                                   self.d_u.addr, self.tokens.addr, self.counts.addr,
                                   self.accept.addr)

    def outputs(self):
        """(tokens per sequence, counts, acceptance probabilities); what lies
        behind the last sequence is as it was."""
        t, c, a = self.tokens.download(), self.counts.download(), self.accept.download()
        assert (t[self.total + self.seqs:] == -77).all() and (c[self.seqs:] == -77).all()
        assert (a[self.total:] == -77).all()
        rows = [t[self.off[b] + b:self.off[b + 1] + b + 1] for b in range(self.seqs)]
        return rows, c[:self.seqs], a[:self.total]

    def check(self, want, label=""):
        """want: per sequence (tokens, acceptance probabilities)."""
        rows, counts, accept = self.outputs()
        for b, (tok, acc) in enumerate(want):
            n = int(self.lens[b])
            assert counts[b] == len(tok), (label, b, counts[b], tok)
            assert rows[b].tolist() == tok + [-1] * (n + 1 - len(tok)), (label, b, rows[b], tok)
            # one rounding to binary32 of a binary64 quotient
            got = accept[self.off[b]:self.off[b + 1]]
            assert np.all(np.abs(got - acc) <= 2.0 ** -24 * np.abs(acc) + 1e-11), (label, b, got, acc)


def to_device(rows, pad=0, skew=0):
    """Rows of floats on the device, `pad` floats longer than they need (NaN)
    and `skew` floats off a 16-byte boundary: (array, address, stride)."""
    rows = np.asarray(rows, np.float32)
    R, V = rows.shape
    flat = np.full((R, V + pad), np.nan, np.float32)
    flat[:, :V] = rows
    d = dev(np.concatenate([np.zeros(skew, np.float32), flat.reshape(-1)]))
    return d, d.addr + 4 * skew, V + pad


def verify(sampler, batch, vocab, target, draft, kind="logits", dkind="logits", temps=None,
           dtemps=None, pad=0, skew=0, state=None, stream=None, keep=None):
    """Enqueues one call on host rows; returns what has to stay alive."""
    dt, at, ldt = to_device(target, pad, skew)
    live = [dt]
    tt = dev(np.asarray(temps, np.float64)) if temps is not None else None
    t = hs.distribution(KINDS[kind], at, ldt, tt.addr if tt else None)
    d = None
    if draft is not None:
        rows = draft if len(draft) else np.zeros((1, vocab), np.float32)
        dd, ad, ldd = to_device(rows, pad, skew)
        td = dev(np.asarray(dtemps, np.float64)) if dtemps is not None else None
        d = hs.distribution(KINDS[dkind], ad, ldd, td.addr if td else None)
        live += [dd, td]
    live += [tt, t, d]
    sampler.verify_drafts_device(t, d, vocab, batch.desc, state, stream)
    return live


def expected(batch, target, draft, kind="logits", dkind="logits", temps=None, dtemps=None):
    """The oracle's outcome per sequence."""
    out = []
    for b in range(batch.seqs):
        o, n = int(batch.off[b]), int(batch.lens[b])
        T = 1.0 if temps is None else float(temps[b])
        D = 1.0 if dtemps is None else float(dtemps[b])
        p = [so.softmax(target[o + b + i], T) if kind == "logits" else so.given(target[o + b + i])
             for i in range(n + 1)]
        q = None
        if draft is not None:
            q = [so.softmax(draft[o + i], D) if dkind == "logits" else so.given(draft[o + i])
                 for i in range(n)]
        out.append(so.verify(p, q, batch.drafts[o:o + n].tolist(), batch.u[o + b:o + b + n + 1]))
    return out


def random_case(rng, lens, vocab, draft=True, kind="logits", dkind="logits", temps=None, noise=1.0):
    """(target rows, draft rows, drafted ids, uniforms): drafts drawn from the
    draft's rows."""
    lens = np.asarray(lens)
    total, seqs = int(lens.sum()), len(lens)
    at = np.concatenate([np.arange(n) + int(lens[:b].sum()) + b for b, n in enumerate(lens)]).astype(int)
    t = (rng.standard_normal((total + seqs, vocab)) * 2.5).astype(np.float32)
    hot = rng.integers(0, vocab, (total + seqs, 4))
    np.add.at(t, (np.arange(total + seqs)[:, None], hot), np.float32(8.0))
    d = (t[at] + rng.standard_normal((total, vocab)) * noise).astype(np.float32)
    seq = np.repeat(np.arange(seqs), lens)
    T = np.ones(seqs) if temps is None else np.where(np.asarray(temps) > 0, temps, 0.5)
    ids = np.array([so.draw(so.softmax(d[i], T[seq[i]]), rng.random()) for i in range(total)], np.int32)
    u = rng.random(total + seqs)
    if kind == "probs":
        seq_t = np.repeat(np.arange(seqs), lens + 1)
        t = np.stack([so.softmax(t[i], T[seq_t[i]]) for i in range(total + seqs)]).astype(np.float32)
    if dkind == "probs" and total:
        d = np.stack([so.softmax(d[i], T[seq[i]]) for i in range(total)]).astype(np.float32)
    return t, d if draft else None, ids.reshape(-1), u
