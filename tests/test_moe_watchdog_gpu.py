"""A mixture-of-experts launch in which a CTA comes later to a grid barrier than the others wait: it ends by itself, the
failure is reported, and the instance then computes as before (GpuDevice.cs:337-374 failure kinds)."""
import time

import pytest

import onegpu_cuda as og
from test_moe_gpu import Layer, run

pytestmark = pytest.mark.gpu

LIMIT_US = 20000


def late_then_right(device, moe, size, barrier, **kw):
    layer = Layer(device, *size, **kw)
    try:
        moe.watchdog_selftest(barrier, LIMIT_US)
        enc = device.begin_commands()
        layer.encode(moe, enc)
        t0 = time.perf_counter()
        with pytest.raises(og.GpuCommandFailedException) as info:
            device.submit(enc)
            device.wait_idle()
        assert info.value.reason == "Watchdog"
        assert time.perf_counter() - t0 < 2.0
        device.wait_idle()  # the failure word was cleared
        for _ in range(2):
            enc = device.begin_commands()
            layer.encode(moe, enc)
            device.submit(enc)
            device.wait_idle()
            layer.check((size, barrier))
    finally:
        layer.dispose()


@pytest.mark.parametrize("barrier", [1, 2, 3, 4])
def test_a_late_cta_fails_the_launch_and_the_instance_stays_usable(device, barrier):
    with og.Int8MoeKernels(device) as moe:
        for size, half in [((1, 256, 512, 8, 2), True), ((8, 272, 144, 16, 4), True), ((5, 1001, 516, 12, 3), False)]:
            late_then_right(device, moe, size, barrier, half=half)


@pytest.mark.parametrize("barrier", [1, 2, 3, 4])
def test_blocks_of_tokens_ranked_by_one_cta_start_anew(device, barrier):
    """More than 8 tokens: the CTA that completes a block's logits ranks it, so what a late CTA still counts after others
    have left must not be found by the next launch."""
    with og.Int8MoeKernels(device) as moe:
        for size, half in [((16, 256, 128, 64, 8), True), ((30, 160, 96, 8, 2), False), ((100, 96, 272, 4, 3), True),
                           ((128, 160, 48, 512, 16), True)]:
            late_then_right(device, moe, size, barrier, half=half)


def test_self_test_arguments(device):
    with og.Int8MoeKernels(device) as moe:
        for barrier, limit in [(0, 1000), (5, 1000), (1, 0), (1, 500001)]:
            with pytest.raises(og.ArgumentOutOfRangeException):
                moe.watchdog_selftest(barrier, limit)
        run(device, moe, 2, 64, 48, 5, 2)  # nothing was set
