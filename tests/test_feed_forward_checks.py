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


def _moe(**change):
    """Buffers of a small layer (5 tokens of 8, 4 experts of 6, 2 chosen), some of them replaced."""
    b = dict(x=spec(F16, 40), router=spec(F32, 32), w_in=spec(S8, 4 * 12 * 8), w_in_scale=spec(F32, 48),
             w_out=spec(S8, 4 * 8 * 6), w_out_scale=spec(F32, 32), y=og._BufferSpec(F16, 48, 0x9000))
    b.update(change)
    return b


def test_moe():
    chk, M = og.check_moe, og.MoeProblem
    p = M(5, 8, 6, 4, 2)
    chk(p, **_moe())
    chk(p, **_moe(residual=_moe()["y"], expert_ids=spec(I32, 10), expert_weights=spec(F32, 10), router=spec(F16, 32)))
    chk(p, **_moe(residual=_moe()["x"], y=_moe()["x"]))
    chk(M(0, 8, 6, 4, 2), **_moe())
    chk(M(5, 8, 12, 4, 2, gated=False, offset_y=8), **_moe(w_out=spec(S8, 384)))
    chk(M(5, 8, 6, 4, 4), **_moe())
    names = dict(x="x", router="router", w_in="wIn", w_in_scale="wInScale", w_out="wOut", w_out_scale="wOutScale", y="y")
    for key, name in names.items():
        assert argument_of(chk, p, **_moe(**{key: None})) == (null, name)
        full = _moe()[key]
        assert argument_of(chk, p, **_moe(**{key: spec(np.int16, full.length)})) == (shape, name)
        short = {"y": 39}.get(key, full.length - 1)
        assert argument_of(chk, p, **_moe(**{key: spec(full.dtype, short)})) == (shape, name)
    assert argument_of(chk, p, **_moe(y=spec(F32, 40))) == (shape, "y")
    assert argument_of(chk, p, **_moe(w_in=spec(U8, 384))) == (shape, "wIn")
    for bad, name in [(M(-1, 8, 6, 4, 2), "Tokens"), (M(129, 8, 6, 4, 2), "Tokens"), (M(5, 0, 6, 4, 2), "ModelSize"),
                      (M(5, 65537, 6, 4, 2), "ModelSize"), (M(5, 8, 0, 4, 2), "ExpertSize"),
                      (M(5, 8, 65537, 4, 2), "ExpertSize"), (M(5, 8, 6, 0, 1), "Experts"),
                      (M(5, 8, 6, 513, 2), "Experts"), (M(5, 8, 6, 4, 0), "TopK"), (M(5, 8, 6, 4, 5), "TopK"),
                      (M(5, 8, 6, 100, 17), "TopK"), (M(5, 8, 6, 4, 2, activation=5), "Activation"),
                      (M(5, 8, 6, 4, 2, activation=-1), "Activation")]:
        assert argument_of(chk, bad, **_moe()) == (shape, name)
    for field, name in [("offset_x", "x"), ("offset_router", "router"), ("offset_in", "wIn"),
                        ("offset_in_scale", "wInScale"), ("offset_out", "wOut"), ("offset_out_scale", "wOutScale"),
                        ("offset_y", "y")]:
        assert argument_of(chk, M(5, 8, 6, 4, 2, **{field: 9}), **_moe()) == (shape, name)
        assert argument_of(chk, M(5, 8, 6, 4, 2, **{field: -1}), **_moe()) == (shape, name + "Offset")
    far = og._BufferSpec(F16, 48, 0x20000)
    chk(M(5, 8, 6, 4, 2, offset_residual=8), **_moe(residual=far))
    assert argument_of(chk, M(5, 8, 6, 4, 2, offset_residual=9), **_moe(residual=far)) == (shape, "residual")
    assert argument_of(chk, p, **_moe(residual=spec(F32, 40))) == (shape, "residual")
    assert argument_of(chk, p, **_moe(residual=spec(F16, 40, null=True))) == (null, "residual")
    assert argument_of(chk, M(5, 8, 6, 4, 2, offset_residual=1), **_moe(residual=_moe()["y"])) == (shape, "residual")
    assert argument_of(chk, p, **_moe(expert_ids=spec(F32, 10))) == (shape, "expertIds")
    assert argument_of(chk, p, **_moe(expert_ids=spec(I32, 9))) == (shape, "expertIds")
    assert argument_of(chk, p, **_moe(expert_weights=spec(F16, 10))) == (shape, "expertWeights")
    assert argument_of(chk, M(5, 8, 6, 4, 2, offset_weights=1), **_moe(expert_weights=spec(F32, 10))) == (
        shape, "expertWeights")
