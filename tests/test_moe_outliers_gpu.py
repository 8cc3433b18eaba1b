"""Int8MoeKernels on rows with values far above the others: a few loud channels of x, or of the hidden values, whose weights
are zero, so that the result rests on the quiet ones alone."""
import numpy as np
import pytest

import onegpu_cuda as og
from test_activated_product_gpu import activate64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step


def held(values, weights, half):
    """How far sum_k weights[j][k] values[k] may be off: values are held to a step of 2^-30 of the largest (2^-38 for
    float32 layers; up to a factor of 2^0.02 more, where the largest did not fit the digits' range), each rounded to half a
    step, and the products of the lowest digit of 128 values are rounded to a multiple of 256 steps. The exact sum then
    becomes a float32."""
    step = np.abs(values).max() * 2.0 ** (-29.98 if half else -37.98)
    w = np.abs(weights)
    return step * (w.sum(-1) / 2 + 128 * ((values.size + 127) // 128)) + U * np.abs(weights @ values)


@pytest.mark.parametrize("half,loud", [(True, 3e3), (True, 6e4), (False, 1e3), (False, 1e5)])
@pytest.mark.parametrize("where", ["x", "hidden"])
@pytest.mark.parametrize("tokens,model,expert,experts,top_k", [(1, 512, 256, 8, 2), (6, 1024, 384, 4, 2), (5, 333, 259, 5, 2),
                                                               (24, 256, 512, 16, 4), (48, 272, 144, 4, 2)])
def test_loud_channels_without_weights(device, tokens, model, expert, experts, top_k, where, half, loud):
    rng = np.random.default_rng(model + tokens)
    kind = np.float16 if half else np.float32
    x = rng.standard_normal((tokens, model))
    router = (rng.standard_normal((experts, model)) * 2 / np.sqrt(model)).astype(np.float32)
    w_in = rng.integers(-128, 128, (experts, 2 * expert, model), dtype=np.int16).astype(np.int8)
    w_out = rng.integers(-128, 128, (experts, model, expert), dtype=np.int16).astype(np.int8)
    in_scale = (rng.uniform(0.5, 1.5, (experts, 2 * expert)) / (74 * np.sqrt(model))).astype(np.float32)
    out_scale = (rng.uniform(0.5, 1.5, (experts, model)) / (74 * np.sqrt(expert))).astype(np.float32)
    if where == "x":
        channels = rng.choice(model, 5, replace=False)
        x[:, channels] *= loud / np.abs(x[:, channels]).max()
        w_in[:, :, channels] = 0
        router[:, channels] = 0.0
    else:
        channels = rng.choice(expert, 5, replace=False)
        in_scale[:, channels] *= np.sqrt(loud)
        in_scale[:, expert + channels] *= np.sqrt(loud)
        w_out[:, :, channels] = 0
    x = x.astype(kind)
    bufs = [device.create_buffer(a.dtype, a.reshape(-1)) for a in (x, router, w_in, in_scale, w_out, out_scale)]
    y, ids = device.create_buffer(kind, tokens * model), device.create_buffer(np.int32, tokens * top_k)
    with og.Int8MoeKernels(device) as moe:
        enc = device.begin_commands()
        moe.encode(enc, og.MoeProblem(tokens, model, expert, experts, top_k), *bufs, y, expert_ids=ids)
        device.submit(enc)
        got, chosen = y.read().reshape(tokens, model).astype(np.float64), ids.read().reshape(tokens, top_k)
    for b in bufs + [y, ids]:
        b.dispose()
    x = x.astype(np.float64)
    logits = x @ router.astype(np.float64).T
    assert np.array_equal(chosen, np.argsort(-logits, axis=1, kind="stable")[:, :top_k])
    for t in range(tokens):
        p = np.exp(logits[t, chosen[t]] - logits[t].max())
        p /= p.sum()
        want, tol = np.zeros(model), np.zeros(model)
        for k, e in enumerate(chosen[t]):
            wi, wo = w_in[e].astype(np.float64), w_out[e].astype(np.float64)
            u = (wi @ x[t]) * in_scale[e]
            du = held(x[t], wi, half) * in_scale[e] + U * np.abs(u)
            act = activate64(u[:expert], og.ACTIVATION_SILU)
            h = act * u[expert:]
            # SiLU's slope is at most 1.1, its own error 24 halves of a step of its argument; one more for the product
            dh = (1.1 * du[:expert] + 24 * U * np.abs(u[:expert])) * (np.abs(u[expert:]) + du[expert:]) + np.abs(act) * du[
                expert:] + U * np.abs(h)
            part = p[k] * out_scale[e] * (wo @ h)
            want += part
            # independent errors of the hidden values: six times their root sum of squares
            tol += p[k] * out_scale[e] * (6 * np.sqrt(wo ** 2 @ dh ** 2) + held(h, wo, half)) + 36 * U * np.abs(part)
        tol += np.abs(want) * (2.0 ** -11 if half else (top_k + 1) * U) + (2.0 ** -25 if half else 0)
        off = np.abs(got[t] - want)
        assert np.all(off <= tol), (t, (off / tol).max(), off.max())
