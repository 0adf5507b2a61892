"""Infinite elements in the adapters themselves: whatever type the adapters
are stored in, a product with an infinity is the infinity that it is in binary32,
also where x or x A^T has few significant bits (values that came from
bfloat16)."""
import numpy as np
import pytest

from hachiue_amd import hip  # noqa: F401 (the library is there)
from oracle import serving_oracle as so
from tests.test_gpu_lora import TYPES, Adapters, run, stored

pytestmark = pytest.mark.gpu
INF = np.inf

# rows, results, rank: the narrow second product (ranks in one and several
# steps, one and four tiles a wave), the one through LDS
SHAPES = [(3, 60, 4), (20, 200, 16), (5, 300, 40), (17, 66000, 20), (5, 99000, 64), (40, 33000, 130)]


def simple(rng, shape):
    """Values of one significant bit."""
    return (rng.choice([-1.0, 1.0], shape) * rng.choice([0.5, 1.0, 2.0], shape)).astype(np.float32)


def exact(ad, x, slots, base):
    with np.errstate(all="ignore"):
        return so.lora(x, ad.a, ad.b, ad.scales, ad.ranks, slots, base)


def check(got, want, bound, label):
    assert np.array_equal(np.isnan(got), np.isnan(want)), label
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf].astype(np.float32)), label
    fine = np.isfinite(want)
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine]), label
    return int(inf.sum())


def put(ad, kind):
    for arr, v in zip(ad.arr, (ad.a, ad.b)):
        arr.upload(stored(v, kind)[0])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,rank", SHAPES)
@pytest.mark.parametrize("K", [40, 600])
def test_infinite_elements(sampler, kind, M, N, rank, K):
    rng = np.random.default_rng(M + N + rank + K)
    for where in ("a", "b", "both signs"):
        ad = Adapters(rng, kind, 3, rank, K, N, scales=False)
        ad.a, ad.b = simple(rng, ad.a.shape), simple(rng, ad.b.shape)
        x, slots = simple(rng, (M, K)), rng.integers(-1, 3, M).astype(np.int32)
        slots[:2] = 0, 1
        if where == "a":
            ad.a[0, rank // 2, 7], ad.a[1, 0, K - 1] = INF, -INF
        elif where == "b":
            ad.b[0, N - 1, 0], ad.b[1, N // 3, rank - 1] = -INF, INF
        else:      # two of them: NaN where they meet with opposite signs
            ad.a[0, 1, [3, K - 2]] = [INF, -INF]
            ad.b[1, 5, [0, rank - 1]] = [INF, INF]
        put(ad, kind)
        y, base = run(sampler, ad, x, slots)
        # (t of whole halves may be 0, and 0 times an infinity is NaN: as in binary32)
        want, bound = exact(ad, x, slots, base)
        n = check(y, want, bound, where)
        assert n or where == "both signs"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,N,rank", [(3, 60, 4), (5, 300, 40), (5, 99000, 64)])
def test_infinities_on_both_sides(sampler, kind, M, N, rank):
    """An infinite x times an infinite element; a finite row of many bits beside
    it."""
    rng = np.random.default_rng(rank)
    ad = Adapters(rng, kind, 1, rank, 70, N, scales=False)
    ad.a, ad.b = simple(rng, ad.a.shape), np.ones_like(ad.b)
    ad.a[0, :, 9] = INF
    put(ad, kind)
    x = rng.standard_normal((M, 70)).astype(np.float32)
    x[:, 9] = np.abs(x[:, 9])
    x[0, 9] = INF
    y, _ = run(sampler, ad, x, [0] * M, None)
    assert (y == INF).all()
