"""Products whose operands are copied into aligned rows first, on an instance that already holds byte-sum scratch: the
sums and the copies are separate buffers."""
import pytest

import onegpu_cuda as og
from cases import Case, problem
from gpu_rig import run_int32

pytestmark = pytest.mark.gpu


def test_staged_product_after_one_with_zero_points(device):
    """The first product allocates the byte sums' scratch; the second one's copy of B must not become that scratch."""
    with og.Int8Gemm(device) as gemm:
        bad, kernel = run_int32(device, gemm, Case("aligned", problem(300, 1008, 272), False, True, 1, 2), 1)
        assert bad == 0 and "staged" not in kernel
        for seed in (2, 3):
            bad, kernel = run_int32(device, gemm, Case("staged", problem(300, 1000, 272), False, True, 1, 2), seed)
            assert bad == 0 and "staged" in kernel
        gemm.reserve_scratch(100000)
        bad, kernel = run_int32(device, gemm, Case("staged", problem(310, 1001, 275), False, True, 2, 1), 4)
        assert bad == 0 and "staged" in kernel
