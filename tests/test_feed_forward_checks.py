"""Refusals of the feed-forward operators (quantization by rows, the activated product, the mixture-of-experts layer),
without a GPU."""
import numpy as np
import pytest

import onegpu_cuda as og

U8, S8, I32, F32, F16 = np.uint8, np.int8, np.int32, np.float32, np.float16
spec, P, Op = og.buffer_spec, og.Int8GemmProblem, og.Int8Operand


def argument_of(fn, *args, **kw):
    with pytest.raises(og.GpuException) as e:
        fn(*args, **kw)
    return type(e.value), getattr(e.value, "argument", None)


shape, null = og.GpuKernelShapeException, og.ArgumentNullException


def test_activated_product():
    a, b, c, s = spec(U8, 64), spec(S8, 64), spec(F16, 64), spec(F32, 8)
    chk, p = og.check_activated, P(4, 8, 8)
    one, rows, cols = Op(s, 0), Op(s, 0, True), Op(s, 0, True)
    chk(p, a, b, c, rows, cols)
    chk(p, a, b, spec(F32, 32), one, one, Op(a, 0, True), Op(b, 0, True), cols, Op(spec(I32, 8), 0),
        og.ACTIVATION_SILU, Op(spec(F32, 32), 0))
    chk(p, a, b, c, one, one, residual=Op(c, 0))
    assert argument_of(chk, p, a, b, None, rows, cols) == (null, "c")
    assert argument_of(chk, p, a, b, spec(I32, 64), rows, cols) == (shape, "c")
    assert argument_of(chk, p, a, b, spec(F16, 31), rows, cols) == (shape, "c")
    assert argument_of(chk, p, a, b, c, None, cols) == (null, "aScale")
    assert argument_of(chk, p, a, b, c, rows, None) == (null, "bScale")
    assert argument_of(chk, P(9, 1, 1), a, b, c, rows, one) == (shape, "aScale")
    assert argument_of(chk, p, a, b, c, Op(s, 5, True), cols) == (shape, "aScale")
    assert argument_of(chk, p, a, b, c, Op(spec(F16, 8), 0), cols) == (shape, "aScale")
    assert argument_of(chk, p, a, b, c, rows, Op(s, 1, True)) == (shape, "bScale")
    assert argument_of(chk, p, a, b, c, rows, cols, float_bias=Op(spec(F32, 7), 0)) == (shape, "floatBias")
    assert argument_of(chk, p, a, b, c, rows, cols, int_bias=Op(s, 0)) == (shape, "intBias")
    assert argument_of(chk, p, a, b, c, rows, cols, activation=5) == (shape, "activation")
    assert argument_of(chk, p, a, b, c, rows, cols, activation=-1) == (shape, "activation")
    assert argument_of(chk, p, a, b, c, rows, cols, residual=Op(spec(F32, 64), 0)) == (shape, "residual")
    assert argument_of(chk, p, a, b, c, rows, cols, residual=Op(spec(F16, 64, null=True), 0)) == (null, "residual")
    far = og._BufferSpec(F16, 64, 0x9000)
    chk(p, a, b, c, rows, cols, residual=Op(far, 32))
    assert argument_of(chk, p, a, b, c, rows, cols, residual=Op(far, 33)) == (shape, "residual")
    assert argument_of(chk, p, a, b, c, rows, cols, residual=Op(c, 8)) == (shape, "residual")  # overlaps c, shifted
    assert argument_of(chk, P(4, 8, 8, offset_c=16), a, b, c, rows, cols, residual=Op(c, 0)) == (shape, "residual")
    chk(P(4, 8, 8, offset_c=32), a, b, c, rows, cols, residual=Op(c, 0))
    # the product's own checks come first, in its order
    assert argument_of(chk, P(9, 9, 9), a, b, c, rows, cols) == (shape, "OffsetA")
    assert argument_of(chk, p, a, b, c, rows, cols, Op(b, 0)) == (shape, "zpA")


def test_quantize_rows():
    x, y, s, z = spec(F16, 40), spec(U8, 40), spec(F32, 5), spec(U8, 5)
    chk = og.check_dynamic_quantize_rows
    chk(x, 0, 5, 8, 0, y, 0, s, 0, z, 0)
    chk(x, 0, 4, 8, 10, y, 0, s, 1, z, 1)
    chk(x, 0, 0, 8, 0, y, 0, s, 0, z, 0)
    assert argument_of(chk, None, 0, 5, 8, 0, y, 0, s, 0, z, 0) == (null, "x")
    assert argument_of(chk, x, 0, 5, 8, 0, spec(U8, 40, null=True), 0, s, 0, z, 0) == (null, "y")
    assert argument_of(chk, x, 0, 5, 8, 0, y, 0, None, 0, z, 0) == (null, "scale")
    assert argument_of(chk, x, 0, 5, 8, 0, y, 0, s, 0, None, 0) == (null, "zeroPoint")
    assert argument_of(chk, spec(I32, 40), 0, 5, 8, 0, y, 0, s, 0, z, 0) == (shape, "x")
    assert argument_of(chk, x, 0, 5, 8, 0, spec(S8, 40), 0, s, 0, z, 0) == (shape, "y")
    assert argument_of(chk, x, 0, -1, 8, 0, y, 0, s, 0, z, 0) == (shape, "rows")
    assert argument_of(chk, x, 0, 5, 0, 0, y, 0, s, 0, z, 0) == (shape, "columns")
    assert argument_of(chk, x, 0, 5, 8, 7, y, 0, s, 0, z, 0) == (shape, "rowStrideX")
    assert argument_of(chk, x, 0, 5, 8, -8, y, 0, s, 0, z, 0) == (shape, "rowStrideX")
    assert argument_of(chk, x, 0, 5, 8, 9, y, 0, s, 0, z, 0) == (shape, "x")
    assert argument_of(chk, x, 1, 5, 8, 0, y, 0, s, 0, z, 0) == (shape, "x")
    assert argument_of(chk, x, -1, 5, 8, 0, y, 0, s, 0, z, 0) == (shape, "xOffset")
    assert argument_of(chk, x, 0, 5, 8, 0, y, 1, s, 0, z, 0) == (shape, "y")
    assert argument_of(chk, x, 0, 5, 8, 0, y, 0, s, 1, z, 0) == (shape, "scale")
    assert argument_of(chk, x, 0, 5, 8, 0, y, 0, s, 0, z, 1) == (shape, "zeroPoint")
    assert argument_of(chk, x, 0, 65536, 65536, 0, y, 0, s, 0, z, 0) == (shape, "rows")
