"""Calls on I8 weights that have nothing to compute, or no room for their scales."""
import numpy as np
import pytest

from hachiue_amd import SamplerError, hip
from hachiue_amd import sampler as hs

pytestmark = pytest.mark.gpu


# (M, N, K): no rows or no channels, before anything else is looked at, as with
# every other type of weights
@pytest.mark.parametrize("wtype", [0, 24])
@pytest.mark.parametrize("M,N,K", [(0, 5, 64), (0, 5, 40), (0, 0, 40), (3, 0, 40), (0, 1 << 25, 1 << 17)])
def test_nothing_to_project(sampler, wtype, M, N, K):
    """Null rows, weights and scales, any K."""
    w = hs.weights(wtype, N, K, 0)
    print(f"[gpu] nothing to project: type {wtype}, {M} x {N} x {K}", flush=True)
    sampler.gemv_device_ex(0, M, K, w, 0, N)
    sampler.gemv_device(0, M, K, K, 0, wtype, N, 0, N)
    tok, u = hip.DeviceArray.from_numpy(np.full(4, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(4))
    greedy = [dict(temperature=0.0)] * M
    sampler.lm_head_sample_device_ex(0, M, K, w, 0, N, None, None, greedy, u.addr, tok.addr)
    ad = hs.adapters(0, 1, 8, K, N, 0, 0)
    sampler.gemv_lora_device(0, M, K, w, ad, 0, 0, N)
    sampler.lm_head_lora_sample_device(0, M, K, w, ad, 0, 0, N, None, None, greedy, u.addr, tok.addr)
    hip.synchronize()
    assert tok.download().tolist() == [0] * M + [-7] * (4 - M)   # (no id to draw: 0)


@pytest.mark.parametrize("M,N,K", [(-1, 5, 64), (0, -1, 64), (0, 5, 0), (3, 0, -16)])
def test_sizes_that_are_none(sampler, M, N, K):
    for wtype in (0, 24):
        with pytest.raises(SamplerError) as e:
            sampler.gemv_device_ex(0, M, 64, hs.weights(wtype, N, K, 0), 0, 64)
        assert e.value.status == 1


def test_calls_that_take_blocks_do_not_know_the_type(sampler):
    """They have no argument for the channels' scales: unsupported, as every type
    that is not in blocks of its own."""
    x, y, w = (hip.DeviceArray.from_numpy(np.zeros(64 * 64, np.float32)) for _ in range(3))
    tok, u = hip.DeviceArray.from_numpy(np.full(2, -7, np.int32)), hip.DeviceArray.from_numpy(np.zeros(2))
    for wtype in (7, 24):
        with pytest.raises(SamplerError) as e:
            sampler.gemv_device(x.addr, 2, 64, 64, w.addr, wtype, 5, y.addr, 64)
        assert e.value.status == 4 and str(wtype) in str(e.value)
        with pytest.raises(SamplerError) as e:
            sampler.lm_head_sample_device(x.addr, 2, 64, 64, w.addr, wtype, 5, y.addr, 64, None, None,
                                          dict(temperature=0.0), u.addr, tok.addr)
        assert e.value.status == 4 and str(wtype) in str(e.value)
        sampler.gemv_device(0, 0, 64, 64, 0, wtype, 5, 0, 64)
    hip.synchronize()
    assert (tok.download() == -7).all() and (y.download() == 0).all()
