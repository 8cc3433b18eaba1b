"""The feed-forward operators run one after another as a decoder block uses them: the tokens quantized row by row, the up
projection with its activation, its result quantized, the down projection added to the stream in place, and a
mixture-of-experts layer on the stream. Each stage is held against its formula in 64 bits from the stage's own inputs, run
as it is and captured into a graph that is replayed on new tokens."""
import numpy as np
import pytest

import og_oracle as oracle
import onegpu_cuda as og
import test_activated_product_gpu as products
import test_moe_gpu as layers

pytestmark = pytest.mark.gpu


class Block:
    """tokens x model; the plain half has `wide` hidden units, the mixture `expert` in each of `experts`."""

    def __init__(self, device, tokens, model, wide, expert, experts, top_k, half, shift):
        rng = np.random.default_rng(tokens + 31 * model + wide)
        self.device, self.tokens, self.model, self.wide, self.half = device, tokens, model, wide, half
        self.kind = np.float16 if half else np.float32
        self.w_up = rng.integers(-128, 128, (wide, model), dtype=np.int16).astype(np.int8)
        self.w_down = rng.integers(-128, 128, (model, wide), dtype=np.int16).astype(np.int8)
        self.s_up = (rng.uniform(0.5, 1.5, wide) / (74 * np.sqrt(model))).astype(np.float32)
        self.s_down = (rng.uniform(0.5, 1.5, model) / (74 * np.sqrt(wide))).astype(np.float32)
        self.bias = (rng.standard_normal(wide) * 0.1).astype(np.float32)
        self.layer = layers.Layer(device, tokens, model, expert, experts, top_k, half=half, shift=shift, residual=True)
        make = device.create_buffer
        self.stream = self.layer.bufs["x"]  # the mixture reads what the down projection left there
        self.at = shift
        self.b = {"w_up": make(np.int8, self.w_up.reshape(-1)), "w_down": make(np.int8, self.w_down.reshape(-1)),
                  "s_up": make(np.float32, self.s_up), "s_down": make(np.float32, self.s_down),
                  "bias": make(np.float32, self.bias), "up": make(self.kind, np.zeros(tokens * wide, self.kind))}
        for name, columns in (("x", model), ("h", wide)):
            self.b[name + "_codes"] = make(np.uint8, np.zeros(tokens * columns, np.uint8))
            self.b[name + "_scale"] = make(np.float32, np.zeros(tokens, np.float32))
            self.b[name + "_zero"] = make(np.uint8, np.zeros(tokens, np.uint8))

    def write(self, x):
        self.x = x.astype(self.kind)
        full = self.stream.read()
        full[self.at:self.at + x.size] = self.x.reshape(-1)
        self.stream.write(full)

    def encode(self, enc, dq, gemm, moe):
        b, t, d, f = self.b, self.tokens, self.model, self.wide
        row = lambda name: og.Int8Operand(b[name], 0, True)  # noqa: E731
        dq.encode_rows(enc, self.stream, self.at, t, d, 0, b["x_codes"], 0, b["x_scale"], 0, b["x_zero"], 0)
        gemm.encode_activated(enc, og.Int8GemmProblem(t, f, d, transpose_b=True), b["x_codes"], b["w_up"], b["up"],
                              row("x_scale"), row("s_up"), zero_point_a=row("x_zero"), float_bias=row("bias"),
                              activation=og.ACTIVATION_SILU)
        dq.encode_rows(enc, b["up"], 0, t, f, 0, b["h_codes"], 0, b["h_scale"], 0, b["h_zero"], 0)
        gemm.encode_activated(enc, og.Int8GemmProblem(t, d, f, transpose_b=True, offset_c=self.at), b["h_codes"],
                              b["w_down"], self.stream, row("h_scale"), row("s_down"), zero_point_a=row("h_zero"),
                              residual=og.Int8Operand(self.stream, self.at))
        self.layer.encode(moe, enc)

    def _rows(self, x, name):
        for r in range(self.tokens):
            y, s, z = oracle.dynamic_quantize(x[r].astype(np.float32))
            assert np.array_equal(self.codes(name, x.shape[1])[r], y), name
            assert self.b[name + "_scale"].read()[r] == s and self.b[name + "_zero"].read()[r] == z, name

    def codes(self, name, columns):
        return self.b[name + "_codes"].read().reshape(self.tokens, columns)

    def _product(self, name, columns, w, scale, bias, act, residual, got):
        a = self.codes(name, columns).astype(np.float64) - self.b[name + "_zero"].read().astype(np.float64)[:, None]
        p = (a @ w.T.astype(np.float64)) * self.b[name + "_scale"].read().astype(np.float64)[:, None] * scale
        v = p + bias
        out = products.activate64(v, act) + residual
        tol = products.tolerance(p, bias, v, out, self.half)
        assert np.all(np.abs(got.astype(np.float64) - out) <= tol), (name, np.max(np.abs(got - out) / tol))

    def check(self):
        t, d, f = self.tokens, self.model, self.wide
        up = self.b["up"].read().reshape(t, f)
        down = self.stream.read()[self.at:self.at + t * d].reshape(t, d)
        self._rows(self.x, "x")
        self._product("x", d, self.w_up, self.s_up.astype(np.float64), self.bias.astype(np.float64), og.ACTIVATION_SILU,
                      0.0, up)
        self._rows(up, "h")
        self._product("h", f, self.w_down, self.s_down.astype(np.float64), np.zeros(d), og.ACTIVATION_NONE,
                      self.x.astype(np.float64), down)
        self.layer.x = down
        self.layer._formula(og.ACTIVATION_SILU, True, True, self.layer.problem.expert_size)
        self.layer.check()

    def outputs(self):
        return self.layer.bufs["y"].read().tobytes() + self.stream.read().tobytes()

    def dispose(self):
        self.layer.dispose()
        for b in self.b.values():
            b.dispose()


@pytest.mark.parametrize("tokens,model,wide,expert,experts,top_k,half,shift", [
    (1, 1024, 4096, 512, 16, 2, True, 0), (9, 512, 1408, 256, 8, 2, False, 0), (5, 333, 777, 101, 7, 3, True, 1),
    (70, 640, 1280, 320, 12, 4, True, 0), (128, 130, 257, 66, 5, 2, False, 3)])
def test_block(device, tokens, model, wide, expert, experts, top_k, half, shift):
    rng = np.random.default_rng(5)
    with og.DynamicQuantizeKernels(device) as dq, og.Int8Gemm(device) as gemm, og.Int8MoeKernels(device) as moe:
        block = Block(device, tokens, model, wide, expert, experts, top_k, half, shift)
        inputs = [rng.standard_normal((tokens, model)) for _ in range(3)]
        eager = []
        for x in inputs:
            block.write(x)
            enc = device.begin_commands()
            block.encode(enc, dq, gemm, moe)
            device.submit(enc)
            block.check()
            eager.append(block.outputs())
        enc = device.begin_commands()
        block.encode(enc, dq, gemm, moe)
        device.capture_begin()
        device.submit(enc)
        graph = device.capture_end()
        for x, want in zip(inputs, eager):  # a replay has the same bits
            block.write(x)
            graph.launch()
            assert block.outputs() == want
        graph.dispose()
        block.dispose()


@pytest.mark.parametrize("m,n,k,kernel", [
    (1, 33, 129, "slim-staged"), (2, 333, 6001, "slim-staged"), (9, 1001, 40, "slim-staged"), (64, 1024, 4096, "slim"),
    (65, 1030, 1100, "slim-staged"), (130, 2064, 1536, "slim"), (300, 520, 2048, "slim-staged"), (1024, 528, 1040, "slim"),
    (257, 4100, 512, "slim-staged"), (129, 144, 640, "slim"), (300, 272, 272, "1sm"), (301, 65, 33, "1sm")])
def test_products_of_few_rows(device, m, n, k, kernel):
    """K shared by clusters of every size, several chunks of rows, and operands copied to 16-byte boundaries first."""
    with og.Int8Gemm(device) as gemm:
        for form in (dict(za=2, zb=2, bias=True, act=og.ACTIVATION_GELU, residual="own", half=True),
                     dict(zb=1, a_signed=True, row_scale=False, transpose_b=True), dict(za=1, int_bias=True, residual="off"),
                     dict()):
            used = products.run(device, gemm, m, n, k, **form)
            if "za" in form and "zb" in form:
                assert used == "tensor-core-" + kernel if "slim" in kernel else "slim" not in used


def test_batched_products_of_few_rows(device):
    with og.Int8Gemm(device) as gemm:
        for m, n, k in [(3, 130, 1000), (200, 144, 1040), (33, 1024, 512)]:
            for share in (False, True):
                products.run(device, gemm, m, n, k, batch=3, za=2, zb=2, half=True, share_b=share, residual="own")


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("tokens,model,expert,experts,top_k,shift", [
    (1, 2049, 1025, 6, 3, 0), (2, 1000, 1361, 9, 2, 1), (7, 999, 500, 5, 2, 0), (20, 515, 333, 30, 3, 1),
    (70, 260, 131, 6, 3, 0), (128, 64, 48, 4, 4, 1), (3, 5, 3, 2, 1, 0), (17, 127, 129, 3, 2, 3)])
def test_layers_of_any_alignment(device, tokens, model, expert, experts, top_k, shift, half):
    """Weights whose rows start anywhere."""
    with og.Int8MoeKernels(device) as moe:
        for gated in (True, False):
            assert layers.run(device, moe, tokens, model, expert, experts, top_k, half=half, shift=shift, gated=gated,
                              residual=True) == "fused-unaligned"


def test_unaligned_layers_that_keep_dram_busy(device):
    layers.test_layers_that_keep_dram_busy(device, 12, 2049, 2047, 40, 4, False)
    layers.test_layers_that_keep_dram_busy(device, 2, 4095, 4097, 10, 6, True)
    layers.test_layers_that_keep_dram_busy(device, 64, 2047, 1409, 40, 6, True)


@pytest.mark.parametrize("counts", [[1, 1, 5, 9, 17, 2], [33, 1, 1, 1, 1, 1], [6, 7, 8, 9, 16, 0]])
def test_layers_of_uneven_experts(device, counts):
    """Experts with one token, a few and several tiles of them: the CTAs' shares end anywhere in a group's units."""
    tokens, experts, model = sum(counts), len(counts), 320
    x = np.zeros((tokens, model), np.float32)
    x[np.arange(tokens), np.repeat(np.arange(experts), counts)] = 4.0
    x[:, experts:] = np.random.default_rng(tokens).standard_normal((tokens, model - experts))
    router = np.zeros((experts, model), np.float32)
    router[np.arange(experts), np.arange(experts)] = 3.0
    with og.Int8MoeKernels(device) as moe:
        for half in (True, False):
            layers.run(device, moe, tokens, model, 1408, experts, 1, half=half, x=x, router=router)
