"""The experts' products of up to 16 tokens over rows of several groups of 512 columns, on gfx950 against the plain 64-bit form:
tolerances as in test_gpu_experts."""

import pytest

from test_gpu_experts import Layer, choice, randn

pytestmark = pytest.mark.gpu


def check(dev, layer, tokens, top_k, size, skew=1.0):
    ids, weights = choice(dev, tokens, tokens, layer.e.experts, top_k, skew)
    x = randn(dev, tokens, tokens, layer.e.hidden, dtype=layer.e.dtype, scale=size)
    layer.check(layer.e.apply(x, ids, weights), x, ids, weights)


@pytest.mark.parametrize("fmt", ["fp4_e2m1", "fp6_e2m3", "fp6_e3m2", "int4", "uint4"])
@pytest.mark.parametrize("hidden,ffn", [(640, 1152), (2176, 640)])
def test_unscaled_experts_of_several_groups(dev, fmt, hidden, ffn):
    print(f"unscaled {fmt} {hidden} {ffn}", flush=True)
    layer = Layer(dev, fmt, 3, hidden, ffn, None)
    for tokens, top_k in ((1, 1), (1, 3), (5, 2), (16, 2)):
        check(dev, layer, tokens, top_k, 0.002)
