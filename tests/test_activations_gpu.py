"""The activations of the product's epilogue by themselves, relative to their results: a product of zeros whose bias is the
argument, on each kernel."""
import math

import numpy as np
import pytest

import onegpu_cuda as og

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step


def exact(v, kind):
    v = v.astype(np.float64)
    if kind == og.ACTIVATION_GELU:
        return 0.5 * v * np.vectorize(math.erfc)(-v * math.sqrt(0.5))
    u2 = v if kind == og.ACTIVATION_SILU else 2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)
    with np.errstate(over="ignore"):
        e = np.exp(-np.abs(u2))
    return np.where(u2 < 0, v * e, v) / (1.0 + e)


def bound(v, kind):
    """Relative, in halves of a float32 step. Documented errors: expf 1 unit in the last place (2 halves), the fast quotient 2
    units (4 halves); everything else rounds correctly (1 half each).
    SiLU: the exponential 2, its product 1, the sum 1 (less where e is small), the quotient 4: 8.
    GELU: fit 2.9; Horner 3, the products by t and e 2; t: a fused step 1 and a quotient 4, times the condition 2.6 of g t: 13;
    the exponential 2 and the square's rest put back 1, the last product 1: below 26.
    tanh GELU: the fast exponential 2 + 1.173 x units (4 + 2.35 x halves) of its argument x = |2 u|, which is off by its
    rounding (two constants, four operations) 6 x; with the product, sum and quotient as in SiLU, 10 + 8.4 x."""
    if kind == og.ACTIVATION_SILU:
        return np.full(v.shape, 8.0)
    if kind == og.ACTIVATION_GELU:
        return np.full(v.shape, 26.0)
    u2 = 2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.astype(np.float64) ** 3)
    return 10.0 + 8.4 * np.abs(u2)


def run(device, gemm, v, kind, m):
    n = v.size
    a, b = device.create_buffer(np.uint8, np.zeros(m * 16, np.uint8)), device.create_buffer(np.int8, np.zeros(16 * n, np.int8))
    one, bias = device.create_buffer(np.float32, np.ones(4, np.float32)), device.create_buffer(np.float32, v)
    c = device.create_buffer(np.float32, m * n)
    enc = device.begin_commands()
    gemm.encode_activated(enc, og.Int8GemmProblem(m, n, 16), a, b, c, og.Int8Operand(one, 0), og.Int8Operand(one, 0),
                          float_bias=og.Int8Operand(bias, 0, True), activation=kind)
    kernel = gemm.last_kernel
    device.submit(enc)
    got = c.read().reshape(m, n)
    for x in (a, b, one, bias, c):
        x.dispose()
    return got, kernel


@pytest.mark.parametrize("kind", [og.ACTIVATION_GELU, og.ACTIVATION_GELU_TANH, og.ACTIVATION_SILU])
def test_relative_error(device, kind):
    rng = np.random.default_rng(kind)
    v = np.concatenate([-np.linspace(0.001, 13, 1 << 14), np.linspace(0.001, 20, 1 << 13), rng.uniform(-6, -1, 1 << 14),
                        rng.standard_normal(1 << 13), -np.exp(rng.uniform(-60, 2, 1 << 13))]).astype(np.float32)
    if kind == og.ACTIVATION_SILU:
        v[:1 << 12] = -np.linspace(13, 87, 1 << 12)
    want = exact(v, kind)
    seen = set()
    for m, options in [(1, {}), (200, {}), (130, dict(tile=128)), (130, dict(tile=256)), (3, dict(kernel=og.KERNEL_PORTABLE))]:
        gemm = og.Int8Gemm(device, og.Int8GemmOptions(**options))
        got, kernel = run(device, gemm, v, kind, m)
        gemm.dispose()
        seen.add(kernel)
        big = np.abs(want) > 2.0 ** -120
        off = np.abs(got[0].astype(np.float64) - want) / np.abs(want) / U
        at = np.argmax(np.where(big, off / bound(v, kind), 0))
        assert np.all(off[big] <= bound(v, kind)[big]), (kernel, v[at], got[0, at], want[at], off[at])
        # Below, the exponential and what follows it may be denormal: three roundings of 2^-150, of what is times v.
        small = bound(v, kind) * U * np.abs(want) + 3 * 2.0 ** -150 * np.maximum(np.abs(v), 1)
        assert np.all((np.abs(got[0] - want) <= small)[~big])
        assert np.array_equal(got, np.broadcast_to(got[:1], got.shape))
    assert len(seen) >= 3, seen


@pytest.mark.parametrize("kind", [og.ACTIVATION_NONE, og.ACTIVATION_RELU, og.ACTIVATION_GELU, og.ACTIVATION_GELU_TANH,
                                  og.ACTIVATION_SILU])
def test_special_values(device, kind):
    """Zeros, the largest and infinite arguments, NaN: what the formulas give (-infinity times zero is NaN)."""
    big = np.float32(3.4e38)
    v = np.array([0.0, -0.0, big, -big, 1e5, -1e5, -100.0, -200.0, np.inf, -np.inf, np.nan, 1.0], np.float32)
    gemm = og.Int8Gemm(device)
    got = run(device, gemm, v, kind, 2)[0][0]
    gemm.dispose()
    assert np.all(got[:2] == 0) and got[2] == big and got[4] == np.float32(1e5) and got[8] == np.inf and np.isnan(got[10])
    if kind == og.ACTIVATION_NONE:
        assert np.array_equal(got[[3, 5, 6, 7, 9]], v[[3, 5, 6, 7, 9]])
    elif kind == og.ACTIVATION_RELU:
        assert np.all(got[[3, 5, 6, 7, 9]] == 0)
    else:
        assert np.all(np.abs(got[[3, 5, 6, 7]]) <= 2.0 ** -130) and np.isnan(got[9])
