"""Helpers of the tests of norms between blocks and 8-bit products."""
from __future__ import annotations

import numpy as np

from hachiue_amd import hip
from hachiue_amd import sampler as hs
from oracle import block_oracle as bo

I8 = 24
ACT_IDS = {k: i for i, k in enumerate(bo.ACTS)}
FILL = 0x5A


class Rows:
    """Rows on the device, `pad` elements of something else behind each and
    `skew` elements in front of the first."""

    def __init__(self, kind, M, C, host=None, pad=0, skew=0, one=False):
        self.kind, self.M, self.C, self.pad, self.skew = kind, M, C, pad, skew
        size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}[kind]
        self.dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i8": np.int8}[kind]
        self.ld = C + pad
        raw = np.full((skew + max(M, 1) * self.ld + 3) * size, FILL, np.uint8).view(self.dtype)
        if host is not None:
            raw[skew:skew + M * self.ld].reshape(M, self.ld)[:, :C] = host
        self.before = raw
        self.arr = hip.DeviceArray.from_numpy(raw)
        self.scales = None
        if kind == "i8":
            self.scales = hip.DeviceArray.from_numpy(np.full(max(M, 1) + 1, 123.0, np.float32))
        self.desc = hs.rows(bo.TYPES[kind], self.arr.addr + skew * size, 0 if one else self.ld,
                            self.scales.addr if self.scales else None)

    def get(self):
        """The rows; what surrounds them is as it was."""
        raw = self.arr.download()
        at = slice(self.skew, self.skew + self.M * self.ld)
        got = raw[at].reshape(self.M, self.ld)[:, :self.C].copy()
        kept = self.before.copy()
        kept[at].reshape(self.M, self.ld)[:, :self.C] = got
        assert np.array_equal(raw.view(np.uint8), kept.view(np.uint8)), "written outside of the rows"
        if self.kind != "i8":
            return got
        s = self.scales.download()
        assert s[self.M:] == 123.0 or self.M == 0
        return got, s[:self.M]

    @classmethod
    def of(cls, x, kind, pad=0, skew=0, one=False):
        """(rows of the values x rounded to `kind`, those values)"""
        raw, val = bo.store(x, kind)
        return cls(kind, x.shape[0], x.shape[1], raw, pad, skew, one), val


def quantised(q, scales, pad=0):
    r = Rows("i8", q.shape[0], q.shape[1], q, pad)
    r.scales.upload(np.concatenate([scales, [123.0]]).astype(np.float32))
    return r


class Weight:
    def __init__(self, rng, N, K, w=None, scales=None):
        self.w = rng.integers(-127, 128, (N, K)).astype(np.int8) if w is None else w
        self.s = (rng.uniform(0.5, 2, N) / (127 * np.sqrt(K))).astype(np.float32) if scales is None else scales
        self.arr = [hip.DeviceArray.from_numpy(np.ascontiguousarray(self.w).reshape(-1)),
                    hip.DeviceArray.from_numpy(self.s)]
        self.desc = hs.weights(I8, N, K, self.arr[0].addr, self.arr[1].addr)


def random_q(rng, M, K):
    """Integers of tokens as they come, extremes (-128 among them) and their scales."""
    q = np.clip(np.rint(rng.standard_normal((M, K)) * 30), -127, 127).astype(np.int8)
    q[rng.random((M, K)) < 0.01] = -128
    return q, rng.uniform(0.001, 0.1, M).astype(np.float32)
