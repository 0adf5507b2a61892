"""Gated pairs whose 128 x 128 tiles are at most one for each compute unit (the form of
four stages), and the sizes on either side of that number."""
import numpy as np
import pytest

from oracle import block_oracle as bo
from tests.block_util import Weight, quantised, random_q
from tests.test_gpu_int8 import gated, gated_bound, same

pytestmark = pytest.mark.gpu


# up to 256 tiles of 128 tokens and 64 channels, but more of 64 tokens; K of less than
# the four stages, of them, and with a tail in each of their turns
@pytest.mark.parametrize("M,N,K", [(65, 16384, 144), (65, 16385, 144), (128, 16321, 48), (250, 8001, 400),
                                   (256, 8192, 512), (129, 8190, 1296), (257, 5400, 1040), (400, 4096, 1168),
                                   (500, 4033, 2064), (512, 4097, 656)])
def test_pairs(sampler, M, N, K):
    rng = np.random.default_rng(M * N + K)
    gate, up, (q, s) = Weight(rng, N, K), Weight(rng, N, K), random_q(rng, M, K)
    want, bound = gated_bound(q, s, gate, up, "silu")
    for out, pad in (("f32", 0), ("bf16", 3)):
        got = bo.values(gated(sampler, quantised(q, s, pad * 16), gate, up, "silu", M, N, out, pad), out)
        err, b = np.abs(got - want), bo.rounded(bound, want, out)
        assert np.all(err <= b), (float((err / b).max()), np.argwhere(~(err <= b))[:4])


@pytest.mark.parametrize("M,N,K", [(256, 8192, 1040), (300, 5001, 272)])
def test_rows_of_a_pair_do_not_depend_on_those_beside_them(sampler, M, N, K):
    """The same bits from the kernels that take fewer rows."""
    rng = np.random.default_rng(N)
    gate, up, (q, s) = Weight(rng, N, K), Weight(rng, N, K), random_q(rng, M, K)
    whole = gated(sampler, quantised(q, s), gate, up, "gelu", M, N)
    for rows in ([0], list(range(5, 21)), list(range(M - 64, M))):
        same(gated(sampler, quantised(q[rows], s[rows]), gate, up, "gelu", len(rows), N), whole[rows], "f32")
