"""Timed calls of which a HIP call fails: the times of the others stay right."""
import pytest

from hachiue_amd import SamplerError, hip
from hachiue_amd import sampler as hs
from tests.conftest import _context
from tests.test_gpu_block_calls import Block

pytestmark = pytest.mark.gpu
KERNELS = ("block_norm_kernel", "int8_kernel", "requant_kernel")


def calls_of(b, ctx):
    """The four calls of Block.enqueue, one by one; float rows, so that the products
    are up to three launches each."""
    return (lambda: ctx.block_norm_device(b.first),
            lambda: ctx.gated_int_device(b.M, b.q.desc, b.gate.desc, b.up.desc, hs.ACT_SILU, b.h.desc),
            lambda: ctx.matmul_int_device(b.M, b.h.desc, b.down.desc, None, b.y.desc),
            lambda: ctx.block_norm_device(b.last))


@pytest.fixture
def nothing_left_to_fail(sampler):     # (the device is prepared: no context's creation fails)
    yield
    _context({"HS_INJECT_HIP_FAILURE": "-1"}).close()


def test_a_timed_call_that_fails_has_no_times(nothing_left_to_fail):
    b = Block(40, x="f32")
    seen = 0
    for n in range(60):
        with _context({"HS_INJECT_HIP_FAILURE": str(n)}) as ctx:
            ctx.set_timing(True)
            made, failed = 0, 0
            for call in calls_of(b, ctx) * 2:
                try:
                    call()
                    made += 1
                except SamplerError as e:
                    assert e.status == 2
                    failed += 1
            hip.synchronize()
            _context({"HS_INJECT_HIP_FAILURE": "-1"}).close()
            print(f"[gpu] failure {n}: {made} calls made, {failed} failed", flush=True)
            ms, calls = ctx.kernel_times()
            assert calls == made and all(0 < ms[k] < 1000 for k in KERNELS)
            assert sum(ms.values()) == sum(ms[k] for k in KERNELS)
            assert ctx.kernel_times() == ({k: 0.0 for k in ms}, 0)
            for call in calls_of(b, ctx):
                call()
            ms, calls = ctx.kernel_times()
            assert calls == 4 and all(0 < ms[k] < 1000 for k in KERNELS)
            b.check()
        seen += failed
        if not failed:
            break
    assert seen >= 20     # (12 launches of the 8 calls, their events and those of the contexts)


def test_reading_the_times_anew_after_a_failure(sampler, nothing_left_to_fail):
    """Each of the query's HIP calls fails once: the next query has every call once."""
    b = Block(40, x="f32")
    failed = 0
    for n in range(60):
        with _context({"HS_INJECT_HIP_FAILURE": "-1"}) as ctx:
            ctx.set_timing(True)
            for call in calls_of(b, ctx):
                call()
            hip.synchronize()
            _context({"HS_INJECT_HIP_FAILURE": str(n)}).close()
            print(f"[gpu] query's failure {n}", flush=True)
            try:
                ms, calls = ctx.kernel_times()
            except SamplerError as e:
                assert e.status == 2
                failed += 1
                ms, calls = ctx.kernel_times()
            else:
                n = None
            assert calls == 4 and all(0 < ms[k] < 1000 for k in KERNELS)
        if n is None:
            break
    # a wait and a difference for each launch: 1 of a norm, 3 of the pair (its rows and
    # its results quantised), 1 of the product, 1 of a norm
    assert failed == 12
