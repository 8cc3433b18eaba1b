"""The router of Int8MoeKernels holds its logits in 64 bits: large common offsets and logits that float32 cannot tell apart
change neither the choice of the experts nor their weights."""
import numpy as np
import pytest

import onegpu_cuda as og
from test_moe_gpu import Layer

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a float32 step


def weights_of(device, moe, **kw):
    layer = Layer(device, **kw)
    try:
        enc = device.begin_commands()
        layer.encode(moe, enc)
        device.submit(enc)
        layer.check(kw)  # the ids equal those of the 64-bit logits
        n = layer.tokens * layer.top_k
        return layer.bufs["weights"].read()[:n].reshape(layer.tokens, -1).astype(np.float64), layer.weights
    finally:
        layer.dispose()


# Roundings of a weight: expf (2 halves of a step), the rest of its argument (1), the sum of up to 16 chosen terms, each off
# by as much (3, and 15 additions) or of 16 + 5 partial sums over all experts (3 and 21), the quotient (1): below 32 halves.
RTOL = 32 * U


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("offset", [30.0, 300.0, 1000.0])
def test_a_common_offset_of_all_logits(device, offset, half):
    with og.Int8MoeKernels(device) as moe:
        for tokens, model, experts, top_k, normalize in [(1, 1024, 128, 8, True), (6, 256, 64, 4, False), (70, 512, 200, 16, True),
                                                         (2, 100, 512, 3, False)]:
            rng = np.random.default_rng(experts)
            x = rng.standard_normal((tokens, model))
            x[:, 0] = offset
            router = rng.standard_normal((experts, model)) * 2 / np.sqrt(model)
            router[:, 0] = 1.0
            got, want = weights_of(device, moe, tokens=tokens, model=model, expert=16, experts=experts, top_k=top_k,
                                   half=half, normalize=normalize, x=x, router=router)
            assert np.all(np.abs(got - want) <= RTOL * want), (np.abs(got / want - 1).max() / U)


@pytest.mark.parametrize("tokens", [1, 5, 33])
def test_logits_closer_than_a_float32_step(device, tokens):
    """Logits of 1000 + i 2^-20, where float32's step is 2^-14, in any order: the largest are chosen, not the first."""
    with og.Int8MoeKernels(device) as moe:
        for experts, top_k in [(64, 8), (300, 16)]:
            router = np.zeros((experts, 48))
            router[:, 0] = 1000.0
            router[:, 1] = np.random.default_rng(experts).permutation(experts) * 2.0 ** -20
            x = np.zeros((tokens, 48))
            x[:, :2] = 1.0
            for half in (True, False):
                got, want = weights_of(device, moe, tokens=tokens, model=48, expert=16, experts=experts, top_k=top_k,
                                       half=half, x=x, router=router)
                assert np.all(np.abs(got - want) <= RTOL * want)


def test_weights_of_experts_far_below_the_first(device):
    """Terms down to float32's smallest normal number keep their relative precision."""
    with og.Int8MoeKernels(device) as moe:
        router = np.zeros((16, 32))
        router[:, 0] = -5.7 * np.arange(16)
        x = np.zeros((3, 32))
        x[:, 0] = 1.0
        got, want = weights_of(device, moe, tokens=3, model=32, expert=16, experts=16, top_k=16, half=False, x=x, router=router)
        assert want.min() > 2.0 ** -126
        assert np.all(np.abs(got - want) <= RTOL * want), (np.abs(got / want - 1).max() / U)
