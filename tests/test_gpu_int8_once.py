"""8-bit products over weights of more than 80 MiB that one tile of tokens reads:
each kernel's form that reads them non-temporally, against the exact integer sums, to
the bit, and the forms just below that size; gated pairs within the activations' bounds."""
import gc

import numpy as np
import pytest

from oracle import block_oracle as bo
from tests.block_util import Rows, Weight, quantised, random_q
from tests.test_gpu_int8 import gated, project, same

pytestmark = pytest.mark.gpu
LIMIT = 80 << 20      # bytes of weights: above it, if at most 64 tokens


@pytest.fixture(autouse=True)
def memory():
    yield
    gc.collect()


def weight(rng, N, K):
    return Weight(rng, N, K, rng.integers(-127, 128, (N, K), np.int8))


def sums(q, s, w):
    """bo.product, some thousand channels at a time."""
    return np.concatenate([bo.product(q, s, w.w[n:n + 4096], w.s[n:n + 4096]) for n in range(0, len(w.s), 4096)], 1)


# One token over several tiles a workgroup; K split among 8 waves (up to 4096
# channels) and 4, one tile of 16 tokens and two; 64 x 128 tiles of four stages and, above
# 256 of them, of two; tails of K of 16 and more, odd numbers of channels
ONE = [(1, 41001, 2064), (1, 40961, 2048), (1, 23000, 3696), (1, 8000, 10512), (2, 4090, 20528), (16, 4090, 20528),
       (16, 8001, 10512), (9, 12001, 7008), (17, 4000, 20992), (30, 4090, 20528), (32, 8190, 10256), (25, 8001, 10512),
       (7, 13000, 6480), (40, 16383, 5136), (64, 16384, 5136), (50, 40001, 2112), (64, 33001, 2560)]
TWO = [(1, 20501, 2064), (1, 12289, 4096), (5, 4090, 10272), (16, 8001, 5264), (17, 4000, 10512), (25, 8001, 5264),
       (33, 9001, 4672), (64, 16000, 2640), (50, 20001, 2112)]
# and what is not above: one byte-row less, or a second tile of tokens
BELOW = [(1, 40960, 2048), (2, 40960, 2048), (65, 16384, 5136)]


@pytest.mark.parametrize("M,N,K", ONE + BELOW)
def test_products(sampler, M, N, K):
    assert (N * K > LIMIT and M <= 64) == ((M, N, K) in ONE)
    rng = np.random.default_rng(M + N + K)
    w, (q, s) = weight(rng, N, K), random_q(rng, M, K)
    want = sums(q, s, w)
    same(project(sampler, quantised(q, s), w, M, N), want, "f32")
    same(project(sampler, quantised(q, s, 16), w, M, N, "bf16", pad=3), want, "bf16")


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 41001, 2064), (1, 21000, 4096), (6, 8001, 10512)])
def test_float_rows(sampler, M, N, K, x):
    """One row quantised by the product's workgroups, several by a launch before it."""
    rng = np.random.default_rng(N)
    w = weight(rng, N, K)
    X, v = Rows.of(rng.standard_normal((M, K)) * 3, x, 3, 1)
    same(project(sampler, X, w, M, N), sums(*bo.quantise(v.astype(np.float32)), w), "f32")


@pytest.mark.parametrize("M,N,K", TWO)
def test_pairs(sampler, M, N, K):
    assert 2 * N * K > LIMIT
    rng = np.random.default_rng(M * N + K)
    gate, up, (q, s) = weight(rng, N, K), weight(rng, N, K), random_q(rng, M, K)
    a, rel = bo.act("silu", sums(q, s, gate).astype(np.float64))
    u = sums(q, s, up).astype(np.float64)
    want, bound = a * u, np.abs(a * u) * (rel + 2 * bo.U) + 2.0 ** -126 * (1 + np.abs(u))
    for out, pad in (("f32", 0), ("f16", 5)):
        got = bo.values(gated(sampler, quantised(q, s, pad * 16), gate, up, "silu", M, N, out, pad), out)
        err, b = np.abs(got - want), bo.rounded(bound, want, out)
        assert np.all(err <= b), (float((err / b).max()), np.argwhere(~(err <= b))[:4])


def test_a_pair_of_one_float_row(sampler):
    """The bits that the row gives when it comes quantised."""
    rng = np.random.default_rng(3)
    N, K = 12289, 4096
    gate, up = weight(rng, N, K), weight(rng, N, K)
    X, v = Rows.of(rng.standard_normal((1, K)), "f16", 0, 3)
    got = [gated(sampler, x, gate, up, "gelu", 1, N) for x in (X, quantised(*bo.quantise(v.astype(np.float32))))]
    same(got[0], got[1], "f32")
