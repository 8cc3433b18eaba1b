"""An activated product of few rows whose load never comes: the launch ends by itself, the failure is reported, and the instance
then computes as before (GpuDevice.cs:337-374 failure kinds)."""
import time

import pytest

import onegpu_cuda as og
from test_activated_product_gpu import Product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (16, 300, 272), (40, 1000, 2048), (100, 256, 1024)])
def test_a_load_that_never_comes_fails_the_launch_and_the_instance_stays_usable(device, m, n, k):
    gemm = og.Int8Gemm(device)
    for za, zb in [(0, 0), (2, 2)]:  # without and with the warps that sum A's rows
        product = Product(device, m, n, k, transpose_b=True, za=za, zb=zb, act=og.ACTIVATION_SILU, residual="aligned")
        gemm.activated_watchdog_selftest(20000)
        enc = device.begin_commands()
        product.encode(gemm, enc)
        assert gemm.last_kernel.startswith("tensor-core-slim")
        t0 = time.perf_counter()
        with pytest.raises(og.GpuCommandFailedException) as info:
            device.submit(enc)
            device.wait_idle()
        assert info.value.reason == "Watchdog"
        assert time.perf_counter() - t0 < 2.0
        product.bufs["c"].write(product.init)
        for _ in range(2):
            enc = device.begin_commands()
            product.encode(gemm, enc)
            device.submit(enc)
            device.wait_idle()
            product.check((m, n, k))
        product.dispose()
    gemm.dispose()


def test_self_test_limit_is_checked(device):
    gemm = og.Int8Gemm(device)
    for limit in (0, 500001):
        with pytest.raises(og.ArgumentOutOfRangeException):
            gemm.activated_watchdog_selftest(limit)
    gemm.dispose()
