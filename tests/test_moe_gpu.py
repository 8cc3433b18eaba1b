"""Int8MoeKernels (a mixture-of-experts layer for a few tokens) against its formula in 64 bits, with sentinels around
every output."""
import numpy as np
import pytest

import onegpu_cuda as og
from test_activated_product_gpu import ACTS, activate64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step


class Layer:
    """One layer: host data, buffers on the device, and the formula's result."""

    def __init__(self, device, tokens, model, expert, experts, top_k, *, act=og.ACTIVATION_SILU, gated=True,
                 normalize=True, half=True, router_half=False, residual="", in_place=False, seed=0, shift=0, routing=True,
                 x=None, router=None, out_gain=1.0):
        rng = np.random.default_rng(seed + tokens * 1000003 + model * 1009 + expert * 31 + experts)
        self.device, self.half, self.tokens, self.model, self.top_k = device, half, tokens, model, top_k
        kind = self.kind = np.float16 if half else np.float32
        up = (2 if gated else 1) * expert
        self.x = (rng.standard_normal((tokens, model)) if x is None else x).astype(kind)
        self.router = (rng.standard_normal((experts, model)) * 2 / np.sqrt(model) if router is None else router).astype(
            np.float16 if router_half else np.float32)
        self.w_in = rng.integers(-128, 128, (experts, up, model), dtype=np.int16).astype(np.int8)
        self.w_out = rng.integers(-128, 128, (experts, model, expert), dtype=np.int16).astype(np.int8)
        self.in_scale = (rng.uniform(0.5, 1.5, (experts, up)) / (74 * np.sqrt(model))).astype(np.float32)
        self.out_scale = (rng.uniform(0.5, 1.5, (experts, model)) / (74 * np.sqrt(expert)) * out_gain).astype(np.float32)
        self.residual = rng.standard_normal((tokens, model)).astype(kind) if residual else None
        self.bufs = {}
        off = dict(offset_x=shift, offset_router=2 * shift, offset_in=3 * shift, offset_in_scale=shift,
                   offset_out=5 * shift, offset_out_scale=2 * shift, offset_y=3 * shift, offset_residual=shift,
                   offset_ids=shift, offset_weights=shift)

        def buf(name, data, lead, tail=0):
            flat = np.concatenate([np.full(lead, -77, data.dtype), data.reshape(-1), np.full(tail, -77, data.dtype)])
            self.bufs[name] = device.create_buffer(data.dtype, flat)
            return self.bufs[name]

        self.y0 = 3 * shift
        x_buf = buf("x", self.x, off["offset_x"], 5)
        self.args = [x_buf, buf("router", self.router, off["offset_router"]), buf("w_in", self.w_in, off["offset_in"]),
                     buf("in_scale", self.in_scale, off["offset_in_scale"]), buf("w_out", self.w_out, off["offset_out"]),
                     buf("out_scale", self.out_scale, off["offset_out_scale"])]
        if in_place:  # y is x
            off["offset_y"] = off["offset_x"]
            self.y0 = off["offset_x"]
            self.bufs["y"] = x_buf
            if residual == "own":
                self.residual = self.x
        else:
            buf("y", self.residual if residual == "own" else np.full((tokens, model), -77, kind), off["offset_y"], 5)
        self.args.append(self.bufs["y"])
        self.kw = {}
        if residual == "own":
            off["offset_residual"] = off["offset_y"]
            self.kw["residual"] = self.bufs["y"]
        elif residual:
            self.kw["residual"] = buf("residual", self.residual, off["offset_residual"])
        if routing:
            self.kw["expert_ids"] = buf("ids", np.full((tokens, top_k), -77, np.int32), shift, 3)
            self.kw["expert_weights"] = buf("weights", np.full((tokens, top_k), -77, np.float32), shift, 3)
        self.shift = shift
        self.problem = og.MoeProblem(tokens, model, expert, experts, top_k, act, gated, normalize, **off)
        self._formula(act, gated, normalize, expert)

    def _formula(self, act, gated, normalize, expert):
        x = self.x.astype(np.float64)
        with np.errstate(all="ignore"):
            logits = x @ self.router.astype(np.float64).T
            rank = np.where(np.isnan(logits), -np.inf, logits)
            self.ids = np.argsort(-rank, axis=1, kind="stable")[:, :self.top_k]
            p = np.exp(logits - logits.max(1, keepdims=True))
            p = p / p.sum(1, keepdims=True)
            w = np.take_along_axis(p, self.ids, 1)
            self.weights = w / w.sum(1, keepdims=True) if normalize else w
        y = np.zeros((self.tokens, self.model))
        tol = np.zeros_like(y)
        # float32 sums (pieces of the operands below a float32 step are dropped): 8 steps of the sum of the products'
        # root mean square by their count, times the constant 6 of the largest of some 1e5 such errors.
        for t in range(self.tokens):
            for k in range(self.top_k):
                e, wt = self.ids[t, k], self.weights[t, k]
                wi = self.w_in[e].astype(np.float64)
                u = (wi @ x[t]) * self.in_scale[e]
                du = 8 * 6 * U * np.sqrt(wi ** 2 @ x[t] ** 2) * self.in_scale[e] + 8 * U * np.abs(u)
                if gated:
                    h = activate64(u[:expert], act) * u[expert:]
                    dh = 1.13 * du[:expert] * np.abs(u[expert:]) + np.abs(activate64(u[:expert], act)) * du[expert:]
                    dh = dh + 32 * U * np.abs(u[:expert] * u[expert:])
                else:
                    h = activate64(u, act)
                    dh = 1.13 * du + 32 * U * np.abs(u)
                if self.half:  # hidden values may be held to 16 significant bits
                    dh = dh + np.abs(h) * 2.0 ** -17
                wo = self.w_out[e].astype(np.float64)
                y[t] += wt * (wo @ h) * self.out_scale[e]
                tol[t] += wt * self.out_scale[e] * (np.sqrt(wo ** 2 @ dh ** 2) * 6 +
                                                    8 * 6 * U * np.sqrt(wo ** 2 @ h ** 2))
                tol[t] += 64 * U * np.abs(wt * (wo @ h) * self.out_scale[e])
        if self.residual is not None:
            y = y + self.residual.astype(np.float64)
        self.y = y
        self.tol = tol + (np.abs(y) * 2.0 ** -11 + 2.0 ** -25 if self.half else np.abs(y) * 4 * U + 1e-30)

    def encode(self, moe, enc):
        moe.encode(enc, self.problem, *self.args, **self.kw)

    def check(self, what=""):
        if "ids" in self.bufs:
            n = self.tokens * self.top_k
            for name, want in (("ids", self.ids), ("weights", self.weights)):
                got = self.bufs[name].read()
                assert np.all(got[:self.shift] == -77) and np.all(got[self.shift + n:] == -77), (what, name)
                got = got[self.shift:self.shift + n].reshape(self.tokens, self.top_k)
                if name == "ids":
                    assert np.array_equal(got, want), (what, got, want)
                else:  # a logit off by 2^-21 of the largest summand shifts a weight by as much; expf 2 steps
                    assert np.allclose(got, want, rtol=1e-5, atol=1e-7, equal_nan=True), (what, got, want)
        got = self.bufs["y"].read()
        lo, hi = self.y0, self.y0 + self.tokens * self.model
        assert np.all(got[:lo] == -77) and np.all(got[hi:] == -77), what
        got = got[lo:hi].reshape(self.tokens, self.model).astype(np.float64)
        with np.errstate(all="ignore"):
            rounded = self.y.astype(self.kind).astype(np.float64)  # past the type's range: infinite
        bad = ~(np.abs(got - self.y) <= self.tol) & ~(np.isnan(got) & np.isnan(self.y)) & ~(got == rounded)
        if bad.any():
            i = np.unravel_index(np.nanargmax(np.where(bad, np.abs(got - self.y) / self.tol, 0)), bad.shape)
            assert False, (what, int(bad.sum()), i, got[i], self.y[i], np.abs(got - self.y)[i] / self.tol[i])

    def dispose(self):
        for b in {id(b): b for b in self.bufs.values()}.values():
            b.dispose()


def run(device, moe, *args, **kw):
    layer = Layer(device, *args, **kw)
    try:
        enc = device.begin_commands()
        layer.encode(moe, enc)
        device.submit(enc)
        layer.check((args, kw))
    finally:
        layer.dispose()
    return moe.last_kernel


# tokens, model, expert, experts, top_k: one token to 128, one expert to many, odd sizes, sizes that end inside a tile
SIZES = [(1, 1, 1, 1, 1), (1, 16, 16, 2, 1), (1, 256, 128, 8, 2), (2, 64, 48, 5, 5), (3, 100, 37, 7, 2),
         (1, 1024, 512, 64, 8), (4, 272, 144, 16, 4), (5, 1001, 516, 12, 3), (8, 512, 256, 8, 2), (9, 208, 80, 3, 2),
         (16, 384, 1040, 4, 1), (17, 64, 64, 1, 1), (31, 144, 96, 33, 7), (40, 256, 112, 2, 2), (64, 128, 176, 60, 6),
         (65, 80, 32, 2, 1), (100, 96, 272, 4, 3), (128, 64, 64, 1, 1), (128, 160, 48, 512, 16), (2, 4112, 2064, 2, 1)]


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("tokens,model,expert,experts,top_k", SIZES)
def test_sizes(device, tokens, model, expert, experts, top_k, half):
    with og.Int8MoeKernels(device) as moe:
        run(device, moe, tokens, model, expert, experts, top_k, half=half)
        run(device, moe, tokens, model, expert, experts, top_k, half=half, gated=False, normalize=False, seed=1,
            act=og.ACTIVATION_GELU, residual="other", shift=1, router_half=True)
        run(device, moe, tokens, model, expert, experts, top_k, half=half, seed=2, residual="own", shift=16,
            act=og.ACTIVATION_GELU_TANH, routing=False)


def test_activations_and_forms(device):
    with og.Int8MoeKernels(device) as moe:
        for act in ACTS:
            for gated in (True, False):
                for half in (True, False):
                    run(device, moe, 6, 96, 80, 5, 2, act=act, gated=gated, half=half, normalize=not gated,
                        residual="" if half else "other")


def test_in_place(device):
    """y may be x, with x as the residual too."""
    with og.Int8MoeKernels(device) as moe:
        for half in (True, False):
            for size in [(1, 256, 128, 8, 2), (24, 272, 144, 6, 2)]:
                run(device, moe, *size, half=half, in_place=True)
                run(device, moe, *size, half=half, in_place=True, residual="own")


def test_equal_logits_choose_the_lowest_experts(device):
    with og.Int8MoeKernels(device) as moe:
        for experts, top_k in [(40, 5), (8, 8), (70, 3)]:
            router = np.zeros((experts, 64))
            run(device, moe, 3, 64, 32, experts, top_k, router=router)
            router[experts // 2:] = 1.0 / 64  # two groups of equal logits
            run(device, moe, 3, 64, 32, experts, top_k, router=router)


def test_every_token_on_one_expert(device):
    """The largest group of one expert, the others idle; and every expert with the same number of tokens."""
    with og.Int8MoeKernels(device) as moe:
        for half in (True, False):
            x = np.random.default_rng(0).standard_normal((128, 64))
            x[:, 0] = 8.0
            router = np.zeros((9, 64))
            router[7, 0] = 1.0
            run(device, moe, 128, 64, 48, 9, 1, x=x, router=router, half=half)
            x[:, 1:9] = 0.0
            x[np.arange(128), 1 + np.arange(128) % 8] = 8.0
            router = np.zeros((8, 64))
            router[np.arange(8), 1 + np.arange(8)] = 1.0
            run(device, moe, 128, 64, 48, 8, 1, x=x, router=router, half=half)


def test_logits_that_are_not_finite(device):
    """A -infinite logit is an expert that is never chosen while others are left; NaN ranks below every number and makes
    the token's weights NaN; no token reaches another's outputs."""
    with og.Int8MoeKernels(device) as moe:
        for half in (True, False):
            rng = np.random.default_rng(3)
            x = rng.standard_normal((6, 32))
            router = rng.standard_normal((6, 32))
            x[:, 0] = 1.0
            x[2, 1], x[3, 1] = np.nan, np.inf
            router[:, 1] = rng.uniform(0.5, 1.5, 6)
            router[4] = 0.0
            router[4, 0] = -np.inf
            layer = Layer(device, 6, 32, 16, 6, 2, x=x, router=router, half=half)
            enc = device.begin_commands()
            layer.encode(moe, enc)
            device.submit(enc)
            ids = layer.bufs["ids"].read()[:12].reshape(6, 2)
            w = layer.bufs["weights"].read()[:12].reshape(6, 2)
            y = layer.bufs["y"].read()[:6 * 32].reshape(6, 32).astype(np.float64)
            fine = [0, 1, 4, 5]
            assert np.array_equal(ids[fine], layer.ids[fine])
            assert np.all((ids >= 0) & (ids < 6))
            assert np.isnan(w[[2, 3]]).all() and np.isnan(y[[2, 3]]).all()
            assert np.all(np.abs(y[fine] - layer.y[fine]) <= layer.tol[fine])
            layer.dispose()


def test_values_past_the_range_of_float16(device):
    """float16 activations that are infinite, and float32 ones of any magnitude."""
    with og.Int8MoeKernels(device) as moe:
        for half, scale in [(True, 3e4), (False, 1e18), (False, 1e-18)]:
            x = np.random.default_rng(5).standard_normal((4, 64)) * scale
            router = np.random.default_rng(6).standard_normal((4, 64)) / scale
            layer = Layer(device, 4, 64, 32, 4, 2, x=x, router=router, half=half, act=og.ACTIVATION_RELU, gated=False)
            enc = device.begin_commands()
            layer.encode(moe, enc)
            device.submit(enc)
            layer.check((half, scale))
            layer.dispose()


def test_hidden_values_past_the_range_of_float16(device):
    """Hidden values of some 1e8 with float16 results inside the range."""
    with og.Int8MoeKernels(device) as moe:
        x = np.random.default_rng(5).standard_normal((9, 64)) * 1e4
        router = np.random.default_rng(6).standard_normal((4, 64)) * 1e-4
        layer = Layer(device, 9, 64, 32, 4, 2, x=x, router=router, act=og.ACTIVATION_RELU, out_gain=1e-5)
        assert np.all(np.isfinite(layer.y)) and 1 < np.abs(layer.y).max() < 6e4
        enc = device.begin_commands()
        layer.encode(moe, enc)
        device.submit(enc)
        layer.check()
        layer.dispose()


def test_no_tokens(device):
    with og.Int8MoeKernels(device) as moe:
        layer = Layer(device, 1, 16, 16, 2, 1)
        layer.problem.tokens = 0
        enc = device.begin_commands()
        layer.encode(moe, enc)
        assert enc.dispatch_count == 0 and moe.last_kernel == "none"
        device.submit(enc)
        assert np.all(layer.bufs["y"].read() == -77)
        layer.dispose()


def test_captured_replayed_and_repeated(device):
    """Two captured layers of one instance replayed in turn, and recorded twice in one encoder: the same bits every time."""
    with og.Int8MoeKernels(device) as moe:
        layers = [Layer(device, 1, 512, 256, 16, 4), Layer(device, 30, 160, 96, 8, 2, half=False)]
        first, graphs = [], []
        for layer in layers:
            enc = device.begin_commands()
            layer.encode(moe, enc)
            layer.encode(moe, enc)
            device.submit(enc)
            layer.check()
            first.append(layer.bufs["y"].read())
        for layer in layers:
            enc = device.begin_commands()
            layer.encode(moe, enc)
            device.capture_begin()
            device.submit(enc)
            graphs.append(device.capture_end())
        for _ in range(5):
            for layer, graph in zip(layers, graphs):
                layer.bufs["y"].write(np.full(layer.bufs["y"].length, -77, layer.kind))
                graph.launch()
            for layer, want in zip(layers, first):
                assert np.array_equal(layer.bufs["y"].read(), want)
        for g in graphs:
            g.dispose()
        for layer in layers:
            layer.dispose()


@pytest.mark.parametrize("tokens,model,expert,experts,top_k,half", [(40, 2048, 1408, 48, 6, True),
                                                                    (1, 4096, 4096, 12, 8, True),
                                                                    (6, 2048, 2048, 24, 4, False)])
def test_layers_that_keep_dram_busy(device, tokens, model, expert, experts, top_k, half):
    """Weights far larger than L2, so that every load waits behind others: some tokens against the formula, and the same
    bits in every run."""
    rng = np.random.default_rng(tokens)
    kind = np.float16 if half else np.float32
    x = rng.standard_normal((tokens, model)).astype(kind)
    router = (rng.standard_normal((experts, model)) * 2 / np.sqrt(model)).astype(np.float32)
    w_in = rng.integers(-128, 128, (experts, 2 * expert, model), dtype=np.int8)
    w_out = rng.integers(-128, 128, (experts, model, expert), dtype=np.int8)
    in_scale = (rng.uniform(0.5, 1.5, (experts, 2 * expert)) / (74 * np.sqrt(model))).astype(np.float32)
    out_scale = (rng.uniform(0.5, 1.5, (experts, model)) / (74 * np.sqrt(expert))).astype(np.float32)
    bufs = [device.create_buffer(a.dtype, a.reshape(-1)) for a in (x, router, w_in, in_scale, w_out, out_scale)]
    y, ids = device.create_buffer(kind, tokens * model), device.create_buffer(np.int32, tokens * top_k)
    with og.Int8MoeKernels(device) as moe:
        first = None
        for _ in range(12):
            y.fill(0xFF)
            enc = device.begin_commands()
            moe.encode(enc, og.MoeProblem(tokens, model, expert, experts, top_k), *bufs, y, expert_ids=ids)
            device.submit(enc)
            got = y.read()
            first = got if first is None else first
            assert np.array_equal(first.view(np.uint8), got.view(np.uint8))
    chosen = ids.read().reshape(tokens, top_k)
    for b in bufs + [y, ids]:
        b.dispose()
    logits = x.astype(np.float64) @ router.astype(np.float64).T
    assert np.array_equal(chosen, np.argsort(-logits, axis=1, kind="stable")[:, :top_k])
    for t in sorted({0, tokens // 2, tokens - 1}):
        p = np.exp(logits[t, chosen[t]] - logits[t].max())
        p /= p.sum()
        want, size = np.zeros(model), np.zeros(model)
        for k, e in enumerate(chosen[t]):
            u = (w_in[e].astype(np.float32) @ x[t].astype(np.float64)) * in_scale[e]
            h = activate64(u[:expert], og.ACTIVATION_SILU) * u[expert:]
            part = p[k] * (w_out[e].astype(np.float32) @ h) * out_scale[e]
            want += part
            size += np.abs(part)
        # below 2^-20 of the parts and of their root mean square, and one rounding of the result
        tol = 2.0 ** -20 * (size + np.sqrt(np.mean(size ** 2))) + np.abs(want) * 2.0 ** (-11 if half else -24)
        assert np.all(np.abs(first.reshape(tokens, model)[t].astype(np.float64) - want) <= tol + 1e-7), t
