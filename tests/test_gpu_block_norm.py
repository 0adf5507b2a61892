"""GPU parity of the norms between blocks with binary64, within what binary32
can be off (block_oracle); quantised rows to the bit where nothing is summed."""
import numpy as np
import pytest

from hachiue_amd import hip
from hachiue_amd import sampler as hs
from oracle import block_oracle as bo
from tests.block_util import ACT_IDS, Rows

pytestmark = pytest.mark.gpu
FLOATS = ["f32", "f16", "bf16"]


class Norm:
    def __init__(self, rng, kind, C, eps=1e-5, w=True, b=True):
        self.kind, self.eps = kind, eps
        self.w = rng.normal(1, 0.3, C).astype(np.float32) if w and kind else None
        self.b = rng.normal(0, 0.3, C).astype(np.float32) if b and kind else None
        self.arr = [None if v is None else hip.DeviceArray.from_numpy(v) for v in (self.w, self.b)]
        self.desc = hs.norm(kind, eps, *(None if a is None else a.addr for a in self.arr))

    @property
    def plain(self):
        return (self.kind, self.eps, *(None if v is None else v.astype(np.float64) for v in (self.w, self.b)))


def rows_like(rng, M, C, std=1.0):
    x = rng.standard_normal((M, C)) * std * np.exp(rng.standard_normal((M, 1)))
    x[:, rng.random(C) < 0.02] *= 15
    return x


def run(sampler, rng, M, C, x="f32", res="f32", out="f32", total="f32", gate=None, gate_kind="f32",
        act="none", after=bo.NONE, before=bo.RMS, scale=0.7, pad=0, skew=0, **norms):
    X, xv = Rows.of(rows_like(rng, M, C), x, pad, skew)
    R, rv = Rows.of(rows_like(rng, M, C, 3.0), res, pad, skew) if res else (None, None)
    G = gv = None
    if gate:
        G, gv = Rows.of(rows_like(rng, 1 if gate == "one" else M, C), gate_kind, pad, skew, gate == "one")
    S = Rows(total, M, C, None, pad, skew) if total else None
    O = Rows(out, M, C, None, pad, skew) if out else None
    A, B = Norm(rng, after, C, **norms), Norm(rng, before, C, **norms)
    print(f"[gpu] block norm {M} x {C} x={x} res={res} gate={gate} {gate_kind} act={act} after={after} "
          f"before={before} sum={total} out={out} pad={pad} skew={skew}", flush=True)
    block = hs.block_norm(M, C, X.desc, R.desc if R else None, scale, G.desc if G else None, ACT_IDS[act],
                          A.desc, S.desc if S else None, B.desc, O.desc if O else None)
    sampler.block_norm_device(block)
    hip.synchronize()
    s, ds, o, do = bo.block_norm(xv, A.plain, gv, act, scale, rv, B.plain)
    if S:
        near(bo.values(S.get(), total), s, bo.rounded(ds, s, total))
    if O and out == "i8":
        q, sc = O.get()
        quantised_near(q, sc, o, do)
    elif O:
        near(bo.values(O.get(), out), o, bo.rounded(do, o, out))


def near(got, want, bound):
    err = np.abs(got - want)
    assert np.all(err <= bound), (float((err / bound).max()), np.argwhere(~(err <= bound))[:4])


def quantised_near(q, scale, want, bound):
    """Scales and integers of results that are up to `bound` off."""
    most, db = np.abs(want).max(1), bound.max(1)
    assert np.all(np.abs(scale * 127.0 - most) <= db + 2 * bo.U * most)
    assert np.all(np.abs(q).max(1) == 127)
    off = np.abs(q * scale[:, None].astype(np.float64) - want)
    assert np.all(off <= 0.5 * scale[:, None] * (1 + 2.0 ** -10) + bound), float((off / scale[:, None]).max())


# a wave a row, a workgroup a row, the registers' limits; widths that 8 does not
# divide take the other form
@pytest.mark.parametrize("M,C", [(1, 1), (3, 7), (5, 8), (2, 63), (9, 257), (4, 512), (6, 520), (3, 2048),
                                 (2, 2049), (3, 4096), (2, 4104), (2, 8192), (1, 8193), (2, 16384),
                                 (1, 32760), (2, 32767), (1, 32768), (1030, 96)])
@pytest.mark.parametrize("before", [bo.RMS, bo.LAYER])
def test_widths(sampler, M, C, before):
    rng = np.random.default_rng(M + C + before)
    run(sampler, rng, M, C, after=3 - before, before=before, gate="each", act="sigmoid")


@pytest.mark.parametrize("C,pad,skew", [(1000, 0, 0), (1000, 3, 0), (1000, 8, 1), (1001, 0, 0), (64, 16, 8)])
@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("out", FLOATS)
def test_types_strides_and_alignment(sampler, x, out, C, pad, skew):
    rng = np.random.default_rng(C + pad + len(x) + len(out))
    other = {"f32": "bf16", "bf16": "f16", "f16": "f32"}
    run(sampler, rng, 70, C, x=x, res=other[x], total=other[out], out=out, gate="each", gate_kind=other[x],
        act="tanh", after=bo.RMS, before=bo.LAYER, pad=pad, skew=skew)


@pytest.mark.parametrize("act", bo.ACTS)
@pytest.mark.parametrize("gate", ["one", "each"])
def test_gates(sampler, act, gate):
    rng = np.random.default_rng(len(act))
    run(sampler, rng, 33, 264, gate=gate, gate_kind="bf16", act=act, after=bo.RMS)


@pytest.mark.parametrize("res", [None, "f32"])
@pytest.mark.parametrize("total,out", [(None, "f32"), ("f32", None), ("bf16", "f16")])
def test_what_may_be_absent(sampler, res, total, out):
    rng = np.random.default_rng(5)
    run(sampler, rng, 20, 320, res=res, total=total, out=out, w=False, b=False)
    run(sampler, rng, 20, 320, res=res, total=total, out=out, before=bo.NONE, after=bo.LAYER, w=True, b=False)
    run(sampler, rng, 20, 320, res=res, total=total, out=out, before=bo.RMS, w=False, b=True, eps=0.0)


@pytest.mark.parametrize("C", [16, 80, 1001, 2048, 4096, 12288])
@pytest.mark.parametrize("before", [bo.NONE, bo.RMS])
def test_quantised_behind_a_norm(sampler, C, before):
    rng = np.random.default_rng(C)
    run(sampler, rng, 37, C, out="i8", total="f32", x="bf16", before=before)


@pytest.mark.parametrize("kind", FLOATS)
@pytest.mark.parametrize("M,C,pad", [(1, 1, 0), (40, 33, 2), (300, 512, 0), (3, 4096, 0), (2, 12288, 8)])
def test_quantised_rows_are_exact(sampler, kind, M, C, pad):
    rng = np.random.default_rng(M + C)
    x = rows_like(rng, M, C) * np.exp2(rng.integers(-12, 12, (M, 1)))
    X, v = Rows.of(x, kind, pad)
    O = Rows("i8", M, C, None, pad)
    sampler.block_norm_device(hs.block_norm(M, C, X.desc, out=O.desc))
    hip.synchronize()
    q, s = O.get()
    wq, ws = bo.quantise(v.astype(np.float32))
    assert np.array_equal(s.view(np.uint32), ws.view(np.uint32))
    assert np.array_equal(q, wq), np.argwhere(q != wq)[:4]


def test_halves_go_to_even_and_their_neighbours_do_not(sampler):
    """Rows whose scale is a power of two hold every half exactly; with an odd
    scale, the binary32 values on either side of each half."""
    rows = []
    for scale in (np.float32(1.0), np.float32(2.0 ** -90), np.float32(1.1), np.float32(3e30)):
        half = np.arange(-126.5, 127, 1.0)
        v = (half * np.float64(scale)).astype(np.float32)
        near_by = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf))])
        top = np.float32(np.float64(scale) * 127)
        rows.append(np.concatenate([[top], near_by[np.abs(near_by) < top]]))
    C = min(len(r) for r in rows)
    x = np.stack([r[:C] for r in rows])
    X, _ = Rows.of(x, "f32")
    O = Rows("i8", len(rows), C)
    sampler.block_norm_device(hs.block_norm(len(rows), C, X.desc, out=O.desc))
    hip.synchronize()
    q, s = O.get()
    wq, ws = bo.quantise(x)
    assert np.array_equal(s, ws) and np.array_equal(q, wq)
    assert {0, 2, -126, 126} <= set(q[0].tolist())


@pytest.mark.parametrize("C", [24, 2048])
def test_rows_without_a_scale(sampler, C):
    """All zeros, below 2^-100, a NaN, an infinity: beside ordinary rows."""
    rng = np.random.default_rng(C)
    x = rng.standard_normal((9, C)).astype(np.float32)
    x[1], x[2] = 0.0, -0.0
    x[3] = 0.0
    x[3, 5] = 2.0 ** -101
    x[4] = 0.0
    x[4, C - 1] = -2.0 ** -100
    x[5, 3], x[6, C - 1], x[7, 0] = np.nan, np.inf, -np.inf
    X, _ = Rows.of(x, "f32")
    O = Rows("i8", 9, C)
    sampler.block_norm_device(hs.block_norm(9, C, X.desc, out=O.desc))
    hip.synchronize()
    q, s = O.get()
    wq, ws = bo.quantise(x)
    assert np.array_equal(q, wq) and np.array_equal(s, ws, equal_nan=True)
    assert s[1] == s[3] == 0 and s[4] > 0 and np.isnan(s[5:8]).all() and q[4, C - 1] == -127


def test_what_is_not_finite_stays_in_its_row(sampler):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 520)).astype(np.float32)
    r = rng.standard_normal((6, 520)).astype(np.float32)
    x[2, 7], r[4, 519] = np.nan, np.inf
    X, _ = Rows.of(x, "f32")
    R, _ = Rows.of(r, "f32")
    S, O = Rows("f32", 6, 520), Rows("f32", 6, 520)
    n = hs.norm(hs.NORM_RMS, 1e-6)
    sampler.block_norm_device(hs.block_norm(6, 520, X.desc, R.desc, after=n, before=n, sum=S.desc, out=O.desc))
    hip.synchronize()
    s, o = S.get(), O.get()
    fine = [0, 1, 3, 5]
    assert np.isfinite(s[fine]).all() and np.isfinite(o[fine]).all()
    assert np.isnan(s[2]).all() and np.isnan(o[2]).all()
    assert np.isinf(s[4, 519]) and np.isfinite(s[4, :519]).all() and np.isnan(o[4, 519])


@pytest.mark.parametrize("C", [72, 1003, 4096])
def test_in_place(sampler, C):
    """The stream's own rows hold the sum, the block's output the next block's input."""
    rng = np.random.default_rng(C)
    M, n = 50, hs.norm(hs.NORM_LAYER, 1e-5)
    got = []
    for place in (False, True):
        g = np.random.default_rng(C)
        X, xv = Rows.of(rows_like(g, M, C), "bf16")
        R, rv = Rows.of(rows_like(g, M, C), "f32")
        S, O = (R, X) if place else (Rows("f32", M, C), Rows("bf16", M, C))
        sampler.block_norm_device(hs.block_norm(M, C, X.desc, R.desc, 0.5, before=n, sum=S.desc, out=O.desc))
        hip.synchronize()
        got.append((S.get(), O.get()))
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_rows_between_each_other(sampler):
    """Inputs and outputs that are columns of one array."""
    rng = np.random.default_rng(8)
    M, C = 30, 64
    x = rng.standard_normal((M, 3 * C)).astype(np.float32)
    arr = hip.DeviceArray.from_numpy(x)
    part = [hs.rows(0, arr.addr + 4 * C * i, 3 * C) for i in range(3)]
    sampler.block_norm_device(hs.block_norm(M, C, part[0], part[2], out=part[1]))
    hip.synchronize()
    y = arr.download()
    assert np.array_equal(y[:, C:2 * C], x[:, :C] + x[:, 2 * C:])
    assert np.array_equal(y[:, :C], x[:, :C]) and np.array_equal(y[:, 2 * C:], x[:, 2 * C:])


def test_no_rows_and_no_columns(sampler):
    X = Rows("f32", 1, 8)
    for M, C in ((0, 8), (1, 0)):
        sampler.block_norm_device(hs.block_norm(M, C, X.desc, out=X.desc))
    sampler.block_norm_device(hs.block_norm(1, 8, X.desc))
    hip.synchronize()
    X.get()
