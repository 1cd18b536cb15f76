"""The experts' products of up to 16 tokens over rows of several groups of 512 columns, on gfx950 against the plain 64-bit form:
tolerances as in test_gpu_experts."""

import pytest
import torch

from test_gpu_experts import BF16, F16, F32, FORMATS, Layer, choice, randn

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


@pytest.mark.parametrize("fmt,scales,block", [f for f in FORMATS if f[1] is not None])
@pytest.mark.parametrize("hidden,ffn", [(640, 1152), (2176, 640), (3712, 256)])
def test_experts_of_several_groups(dev, fmt, scales, block, hidden, ffn):
    """Rows of 2 to 8 groups, whose last one is not full, whole and in two and four slices of waves."""
    print(f"groups {fmt} {scales} {block} {hidden} {ffn}", flush=True)
    layer = Layer(dev, fmt, 3, hidden, ffn, scales, block)
    for tokens, top_k in ((1, 1), (1, 3), (5, 2), (16, 2)):
        check(dev, layer, tokens, top_k, 0.3)


@pytest.mark.parametrize("fmt,scales,block", [("fp4_e2m1", "e8m0", 32), ("fp6_e2m3", "e8m0", 32), ("fp6_e3m2", "e8m0", 32), ("int4", F16, 32),
                                              ("int4", F32, 32), ("uint4", BF16, 64), ("uint4", F32, 64), ("int4", F32, 128)])
def test_waves_of_many_groups(dev, fmt, scales, block):
    """More rows than waves: each goes through several units, with the next groups always on their way."""
    print(f"many groups {fmt} {scales} {block}", flush=True)
    layer = Layer(dev, fmt, 8, 2176, 2176, scales, block)
    for tokens, top_k in ((16, 4), (15, 8), (16, 1)):
        check(dev, layer, tokens, top_k, 0.3)


@pytest.mark.parametrize("tokens", [3, 40])
def test_outputs_over_the_weights_are_refused(dev, tokens):
    """A token's output is written while another's weights are read."""
    layer = Layer(dev, "fp4_e2m1", 4, 128, 128)
    ids, weights = choice(dev, 1, tokens, 4, 2)
    x = randn(dev, 2, tokens, 128, dtype=layer.e.dtype, scale=0.5)
    held = torch.zeros(tokens * 128 + 2 * tokens, device=dev)
    out, behind = held[:tokens * 128].view(tokens, 128), held[tokens * 128:].view(tokens, 2)
    behind.copy_(weights)
    want = layer.e.apply(x, ids, weights, out=torch.empty_like(out))
    assert torch.equal(layer.e.apply(x, ids, behind, out=out), want)  # next to each other
    for at in (0, 7, tokens * 128 - 1):
        over = held[at:at + 2 * tokens].view(tokens, 2)
        over.copy_(weights)
        with pytest.raises(ValueError):
            layer.e.apply(x, ids, over, out=out)
    rows = torch.zeros((tokens, 130), device=dev)  # weights in the gaps of out's rows, all in one row
    gaps = rows.view(-1)[128:128 + 2].view(1, 2)
    gaps.copy_(weights[:1])
    got = layer.e.apply(x[:1], ids[:1], gaps, out=rows[:1, :128])
    assert torch.equal(gaps, weights[:1])
    layer.check(got, x[:1], ids[:1], weights[:1])
