"""Int8Gemm.encode_activated (scale per row and column, bias, activation and residual in the product's epilogue) on every
kernel configuration, against the formula in 64 bits, with sentinels around every output."""
import math

import numpy as np
import pytest

import onegpu_cuda as og

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step
ACTS = [og.ACTIVATION_NONE, og.ACTIVATION_RELU, og.ACTIVATION_GELU, og.ACTIVATION_GELU_TANH, og.ACTIVATION_SILU]
_erf = np.vectorize(math.erf)


def activate64(v, kind):
    with np.errstate(all="ignore"):
        if kind == og.ACTIVATION_RELU:
            return np.where(np.isnan(v), v, np.maximum(v, 0.0))
        if kind == og.ACTIVATION_GELU:
            return 0.5 * v * (1.0 + _erf(v * math.sqrt(0.5)))
        if kind == og.ACTIVATION_GELU_TANH:
            return 0.5 * v * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
        if kind == og.ACTIVATION_SILU:
            return v / (1.0 + np.exp(-v))
        return v


def tolerance(p, b, v, out, half):
    """Rounding steps, each at most half a step: the sum's conversion, the scale product, the scaling and the bias (four,
    on at most |p| + |b|, times the activations' largest slope 1.13); the activation's own (erff: 2 float32 steps, the
    fast exponential and quotient 2^-22 each and |t| 2^-24 with |t| sigma(-t) < 0.28: below 24 halves of |v|); the
    residual's sum (one, of the result); and one rounding to float16, whose smallest step is 2^-24."""
    t = U * (1.13 * 4 * (np.abs(p) + np.abs(b)) + 24 * np.abs(v) + np.abs(out))
    return t + np.abs(out) * 2.0 ** -11 + 2.0 ** -25 if half else t + 1e-45


class Product:
    """One product: host data, buffers on the device, and the formula's result."""

    def __init__(self, device, m, n, k, *, batch=1, transpose_b=False, a_signed=False, za=0, zb=0, row_scale=True,
                 col_scale=True, bias=False, int_bias=False, act=og.ACTIVATION_NONE, residual="", half=False, seed=0,
                 pad_a=0, pad_b=0, offset_c=3, share_b=False):
        rng = np.random.default_rng(seed + 1000 * m + n + 7 * k)
        self.device, self.half, self.act, self.offset_c = device, half, act, offset_c
        lda, ldb = k + pad_a, (k if transpose_b else n) + pad_b
        a_type = np.int8 if a_signed else np.uint8
        rows_b = n if transpose_b else k
        a = rng.integers(-128 if a_signed else 0, 128 if a_signed else 256, (batch, m, max(lda, 1)), dtype=np.int16)
        b = rng.integers(-128, 128, (1 if share_b else batch, max(rows_b, 1), max(ldb, 1)), dtype=np.int16)
        a, b = a.astype(a_type), b.astype(np.int8)
        self.problem = og.Int8GemmProblem(m, n, k, batch, transpose_b, lda if pad_a else 0, ldb if pad_b else 0, 0, 0,
                                          offset_c, m * lda if batch > 1 else 0,
                                          0 if share_b or batch == 1 else rows_b * ldb)
        zav = rng.integers(0, 100, m if za == 2 else 1).astype(a_type) if za else None
        zbv = rng.integers(-50, 50, n if zb == 2 else 1).astype(np.int8) if zb else None
        sa = rng.uniform(0.01, 0.05, m if row_scale else 1).astype(np.float32)
        sb = (rng.uniform(0.5, 1.5, n if col_scale else 1) / (60.0 * math.sqrt(max(k, 1)))).astype(np.float32)
        fb = rng.standard_normal(n).astype(np.float32) if bias else None
        ib = rng.integers(-10000, 10000, n).astype(np.int32) if int_bias else None
        self.kind = np.float16 if half else np.float32
        res = rng.standard_normal(batch * m * n).astype(self.kind) if residual else None
        self.sentinel = np.full(offset_c + batch * m * n + 5, -77.0, self.kind)
        init = self.sentinel.copy()
        if residual == "own":
            init[offset_c:offset_c + res.size] = res
        self.init = init
        self.bufs = {}

        def buf(name, data, kind=None):
            if data is None:
                return None
            self.bufs[name] = device.create_buffer(kind or data.dtype, data.reshape(-1))
            return self.bufs[name]

        def opd(name, data, vector, offset=0):
            if data is None:
                return None
            return og.Int8Operand(buf(name, np.concatenate([np.zeros(offset, data.dtype), data])), offset, vector)

        self.args = [buf("a", a), buf("b", b), buf("c", init), opd("sa", sa, row_scale, 1), opd("sb", sb, col_scale, 2)]
        self.kw = dict(zero_point_a=opd("za", zav, za == 2, 3), zero_point_b=opd("zb", zbv, zb == 2, 1),
                       float_bias=opd("fb", fb, True, 3), int_bias=opd("ib", ib, True, 1), activation=act)
        if residual == "own":
            self.kw["residual"] = og.Int8Operand(self.bufs["c"], offset_c)
        elif residual:
            self.kw["residual"] = opd("res", res, False, 8 if residual == "aligned" else 1)
        # the formula
        af = a[:, :, :k].astype(np.float64)
        if zav is not None:
            af = af - zav.astype(np.float64).reshape(1, -1, 1)
        bf = b[:, :rows_b, :(k if transpose_b else n)].astype(np.float64)
        bf = bf.transpose(0, 2, 1) if transpose_b else bf
        if zbv is not None:
            bf = bf - zbv.astype(np.float64).reshape(1, 1, -1)
        s = np.matmul(af, bf) if k else np.zeros((batch, m, n))
        if ib is not None:
            s = s + ib
        p = s * sa.astype(np.float64).reshape(1, -1, 1) * sb.astype(np.float64).reshape(1, 1, -1)
        bias64 = np.zeros(n) if fb is None else fb.astype(np.float64)
        v = p + bias64
        out = activate64(v, act)
        if residual:
            out = out + res.astype(np.float64).reshape(batch, m, n)
        self.want = out.reshape(-1)
        self.tol = tolerance(p, bias64, v, out, half).reshape(-1)

    def encode(self, gemm, enc):
        gemm.encode_activated(enc, self.problem, *self.args, **self.kw)

    def check(self, what=""):
        got = self.bufs["c"].read()
        lo, hi = self.offset_c, self.offset_c + self.want.size
        assert np.array_equal(got[:lo], self.sentinel[:lo]) and np.array_equal(got[hi:], self.sentinel[hi:]), what
        if not self.want.size:
            return
        off = np.abs(got[lo:hi].astype(np.float64) - self.want)
        at = int(np.argmax(off - self.tol))
        assert np.all(off <= self.tol), (what, at, got[lo + at], self.want[at], off[at] / self.tol[at])

    def dispose(self):
        for b in self.bufs.values():
            b.dispose()


def run(device, gemm, *args, **kw):
    p = Product(device, *args, **kw)
    try:
        enc = device.begin_commands()
        p.encode(gemm, enc)
        kernel = gemm.last_kernel
        device.submit(enc)
        p.check((kernel, args, kw))
    finally:
        p.dispose()
    return kernel


SHAPES = [  # m, n, k: rows, one-SM and two-SM tiles, ragged edges, operands TMA cannot load
    (1, 1, 1), (1, 256, 128), (1, 130, 2048), (2, 1024, 4096), (7, 4096, 512), (16, 272, 1040), (17, 144, 128),
    (33, 31, 17), (128, 256, 128), (129, 257, 144), (200, 264, 400), (300, 1000, 272), (513, 520, 1024),
    (1100, 776, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes_and_types(device, m, n, k):
    with og.Int8Gemm(device) as gemm:
        for i, act in enumerate(ACTS):
            run(device, gemm, m, n, k, transpose_b=i % 2 == 0, a_signed=i % 2 == 1, za=i % 3, zb=(i + 1) % 3,
                row_scale=i != 1, col_scale=i != 2, bias=i % 2 == 0, int_bias=i == 3, act=act,
                residual=["", "own", "other", "", "aligned"][i], half=i % 2 == 0, offset_c=[0, 3, 8, 0, 8][i])
            run(device, gemm, m, n, k, transpose_b=i % 2 == 1, za=(i + 1) % 3, zb=i % 3, bias=i % 2 == 1, act=act,
                residual=["own", "aligned", "", "other", "own"][i], half=i % 2 == 1, offset_c=[8, 0, 1, 4, 0][i],
                seed=5)


@pytest.mark.parametrize("options", [dict(kernel=og.KERNEL_TENSOR_CORE, tile=128), dict(kernel=og.KERNEL_TENSOR_CORE,
                                     tile=256), dict(kernel=og.KERNEL_PORTABLE), dict(tile=256, stream_k=2),
                                     dict(tile=128, stream_k=2)])
def test_every_kernel_configuration(device, options):
    with og.Int8Gemm(device, og.Int8GemmOptions(**options)) as gemm:
        seen = set()
        for m, n, k in [(300, 528, 400), (256, 512, 1280), (2304, 2320, 256)]:
            for half in (False, True):
                for i, res in enumerate(("", "own", "aligned")):
                    seen.add(run(device, gemm, m, n, k, transpose_b=half, za=2, zb=1, bias=True, act=ACTS[2 + i],
                                 residual=res, half=half, offset_c=0 if i else 8))
        if options.get("stream_k"):
            assert any("stream-k" in s for s in seen), seen


def test_batches_strides_and_leading_dimensions(device):
    with og.Int8Gemm(device) as gemm:
        for m, n, k in [(5, 160, 96), (140, 272, 128), (300, 264, 144), (9, 31, 33)]:
            for half in (False, True):
                run(device, gemm, m, n, k, batch=3, za=2, zb=2, bias=True, act=og.ACTIVATION_SILU, residual="aligned",
                    half=half, pad_a=16, pad_b=32)
                run(device, gemm, m, n, k, batch=2, za=1, transpose_b=True, share_b=True, residual="own",
                    act=og.ACTIVATION_GELU, half=half, pad_a=3, pad_b=1)


def test_no_columns_no_rows_no_depth(device):
    with og.Int8Gemm(device) as gemm:
        for m, n, k in [(0, 8, 8), (8, 0, 8)]:
            assert run(device, gemm, m, n, k) == "none"
        # K = 0: every sum is empty, the bias and the residual remain.
        run(device, gemm, 5, 40, 0, bias=True, act=og.ACTIVATION_GELU, residual="other")
        run(device, gemm, 5, 40, 0, bias=True, residual="own", half=True, int_bias=True)


def test_values_that_are_not_finite(device):
    """A row scale, a bias or a residual that is infinite or NaN stays in its row, column or element; float16 results past
    the type's range are infinite."""
    m, n, k = 130, 272, 128
    for half in (False, True):
        for tile, act in [(0, og.ACTIVATION_NONE), (128, og.ACTIVATION_RELU), (0, og.ACTIVATION_SILU)]:
            for rows in (3, m):
                rng = np.random.default_rng(1)
                a = rng.integers(0, 256, (rows, k)).astype(np.uint8)
                b = rng.integers(-128, 128, (k, n)).astype(np.int8)
                sa = np.full(rows, 1e-3, np.float32)
                sa[1] = np.nan
                sa[2] = 3e6
                sb = np.ones(n, np.float32)
                fb = np.zeros(n, np.float32)
                fb[5], fb[7] = np.inf, np.nan
                kind = np.float16 if half else np.float32
                res = np.zeros((rows, n), kind)
                res[0, 9], res[0, 11] = -np.inf, np.nan
                bufs = [device.create_buffer(x.dtype, x.reshape(-1)) for x in (a, b, sa, sb, fb, res)]
                c = device.create_buffer(kind, rows * n)
                with og.Int8Gemm(device, og.Int8GemmOptions(tile=tile)) as gemm:
                    enc = device.begin_commands()
                    gemm.encode_activated(enc, og.Int8GemmProblem(rows, n, k), bufs[0], bufs[1], c,
                                          og.Int8Operand(bufs[2], 0, True), og.Int8Operand(bufs[3], 0, True),
                                          float_bias=og.Int8Operand(bufs[4]), activation=act,
                                          residual=og.Int8Operand(bufs[5]))
                    device.submit(enc)
                    got = c.read().reshape(rows, n).astype(np.float64)
                with np.errstate(all="ignore"):
                    v = (a.astype(np.float64) @ b.astype(np.float64)) * sa.astype(np.float64)[:, None] + fb
                    want = activate64(v, act) + res.astype(np.float64)
                    want = want.astype(kind).astype(np.float64)
                for buf in bufs + [c]:
                    buf.dispose()
                assert np.array_equal(np.isnan(got), np.isnan(want)), (half, tile, act)
                assert np.array_equal(np.isposinf(got), np.isposinf(want)), (half, tile, act)
                assert np.array_equal(np.isneginf(got), np.isneginf(want)), (half, tile, act)


def test_captured_and_replayed(device):
    """Two captured graphs of one instance, replayed in turn with new inputs, share its workspaces in stream order."""
    with og.Int8Gemm(device) as gemm:
        ps = [Product(device, m, n, k, za=2, zb=2, bias=True, act=og.ACTIVATION_SILU, residual="aligned", half=True,
                      offset_c=0) for m, n, k in [(4, 512, 2048), (300, 520, 256)]]
        graphs = []
        for p in ps:
            for capture in (False, True):
                enc = device.begin_commands()
                p.encode(gemm, enc)
                if capture:
                    device.capture_begin()
                device.submit(enc)
            graphs.append(device.capture_end())
        for _ in range(3):
            for p, g in zip(ps, graphs):
                p.bufs["c"].fill(0)
                g.launch()
        for p in ps:
            p.sentinel[:] = 0
            p.check("replayed")
        for g in graphs:
            g.dispose()
        for p in ps:
            p.dispose()


def test_results_do_not_change_from_call_to_call(device):
    with og.Int8Gemm(device) as gemm:
        for m, n, k in [(2, 1024, 4096), (300, 1032, 512)]:
            p = Product(device, m, n, k, za=1, zb=2, bias=True, act=og.ACTIVATION_GELU)
            first = None
            for _ in range(4):
                enc = device.begin_commands()
                p.encode(gemm, enc)
                p.encode(gemm, enc)
                device.submit(enc)
                got = p.bufs["c"].read()
                first = got if first is None else first
                assert np.array_equal(first, got)
            p.dispose()
