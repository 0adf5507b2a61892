"""Norms between blocks in the forms that many rows take, two runs of eight
elements a thread, and on the other side of the numbers of rows where they begin:
binary64 within the same bounds as tests/test_gpu_block_norm.py."""
import numpy as np
import pytest

from oracle import block_oracle as bo
from tests.test_gpu_block_norm import FLOATS, run

pytestmark = pytest.mark.gpu

# a wave a row and two runs above 512 columns and rows, 256 threads above 2048 and 256,
# 512 above 4096 and 256: whole and with a tail, a thread's second run absent, begun
# and full, and the last number of rows (or columns) of the form before
SIZES = [(513, 520), (513, 600), (600, 1001), (513, 1017), (513, 1024), (512, 1001), (512, 1024), (700, 1025),
         (257, 2049), (257, 2056), (300, 3001), (257, 4095), (257, 4096), (256, 4095), (256, 4096),
         (257, 4097), (257, 4104), (270, 6001), (257, 8191), (257, 8192), (256, 8191), (256, 8192), (257, 8200)]


@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("before", [bo.RMS, bo.LAYER])
def test_many_rows(sampler, M, C, before):
    rng = np.random.default_rng(M * C + before)
    run(sampler, rng, M, C, after=3 - before, before=before, gate="each", act="sigmoid")


@pytest.mark.parametrize("M,C,pad,skew", [(513, 1000, 3, 1), (520, 777, 0, 0), (257, 3000, 8, 8), (260, 2999, 1, 1),
                                          (257, 7000, 3, 1), (259, 8001, 0, 0)])
@pytest.mark.parametrize("x", FLOATS)
def test_types_strides_and_alignment(sampler, x, M, C, pad, skew):
    """Every type in every place, one gate for all rows."""
    rng = np.random.default_rng(M + C + len(x))
    other = {"f32": "bf16", "bf16": "f16", "f16": "f32"}
    run(sampler, rng, M, C, x=x, res=other[x], total=other[other[x]], out=x, gate="one", gate_kind=other[x],
        act="gelu_tanh", after=bo.LAYER, before=bo.RMS, pad=pad, skew=skew)


@pytest.mark.parametrize("M,C,pad", [(513, 1024, 0), (513, 1003, 5), (257, 4096, 0), (257, 4001, 3), (257, 8192, 8),
                                     (257, 8189, 0), (300, 12289, 0), (40, 20001, 3)])
@pytest.mark.parametrize("before", [bo.NONE, bo.RMS, bo.LAYER])
def test_quantised_behind_a_norm(sampler, M, C, pad, before):
    rng = np.random.default_rng(C + before)
    run(sampler, rng, M, C, out="i8", total="bf16", x="bf16", after=bo.RMS, before=before, pad=pad)


@pytest.mark.parametrize("M,C", [(513, 1001), (257, 4096), (257, 8191)])
@pytest.mark.parametrize("w,b", [(True, False), (False, True), (False, False)])
def test_parameters_that_are_absent(sampler, M, C, w, b):
    rng = np.random.default_rng(C)
    run(sampler, rng, M, C, after=bo.LAYER, before=bo.RMS, w=w, b=b)
    run(sampler, rng, M, C, after=bo.RMS, before=bo.LAYER, w=w, b=b, res=None, total=None)
