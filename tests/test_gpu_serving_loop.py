"""The serving loop in states that a program can bring it into."""

from dataclasses import replace

import pytest
import torch

from tinygrad_mi355x.decoder import random_weights
from tinygrad_mi355x.serving import ServingDecoder
from test_gpu_serving_decoder import SMALL, prompts_of

pytestmark = pytest.mark.gpu


def test_prompts_need_the_prefix(dev):
    """Pages of a prefix that was never run through the model are not attended to."""
    d = ServingDecoder(random_weights(SMALL, dev, seed=20), SMALL, 2, 192, 16, prefix=64)
    u = torch.rand((2, 3), device=dev)
    for call in (lambda: d.prefill(prompts_of(dev, 2, 4)), lambda: d.generate(prompts_of(dev, 2, 4), 3, u)):
        with pytest.raises(RuntimeError, match="load_prefix"):
            call()
    with pytest.raises(ValueError):
        d.load_prefix(prompts_of(dev, 1, 64)[0] + SMALL.vocab)
    with pytest.raises(RuntimeError, match="load_prefix"):
        d.prefill(prompts_of(dev, 2, 4))
    d.load_prefix(prompts_of(dev, 1, 64)[0])
    first = d.generate(prompts_of(dev, 2, 4), 3, u)
    assert torch.equal(d.generate(prompts_of(dev, 2, 4), 3, u), first)  # loaded once


def test_a_held_graph_follows_the_filters(dev):
    """A step captured once and replayed behind a later generate draws with that one's filters, as an eager step does."""
    d = ServingDecoder(random_weights(SMALL, dev, seed=21), SMALL, 3, 128, 16)
    prompts, u = prompts_of(dev, 3, 20, 22), torch.rand((3, 2), generator=torch.Generator().manual_seed(23)).to(dev)
    d.generate(prompts, 2, u)
    graph = d.capture()
    drawn = []
    for filters in (dict(temperature=0.0), dict(temperature=1.5), dict(temperature=torch.tensor([2.0, 0.0, 1.0]), top_k=1),
                    dict(temperature=1.5, top_k=torch.tensor([0, 40, 3]), top_p=0.9, min_p=0.02), dict(temperature=1.5, top_p=0.3)):
        for i in range(2):
            d.generate(prompts, 2, u, **filters)
            junk = [torch.full((3,), 7.0, device=dev) for _ in range(64)]  # what a freed parameter would read as
            d.u.fill_(0.7 - 0.3 * i)
            tokens, pos = d.tokens[:3].clone(), d.pos.clone()
            d.step()
            want, logits = d.tokens[:3].clone(), d.logits.clone()
            d.tokens[:3], d.pos[:] = tokens, pos
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(d.logits, logits) and torch.equal(d.tokens[:3], want), filters
            drawn.append(want.tolist())
            del junk
    assert len(set(map(str, drawn))) > 3  # they do differ


def test_traces_of_a_prefix_in_short_chunks(dev):
    """Chunks of 5 to 7 tokens of one sequence in a decoder of 8: the traced feed-forward output is the one that the next
    layer adds, in whatever form the down projection computes it (fp32 sums in another order: 2^-20 of the norm)."""
    cfg = replace(SMALL, ffn=4096)
    w = random_weights(cfg, dev, seed=24)
    d = ServingDecoder(w, cfg, 8, 64, 6, prefix=16, page_size=16)
    assert d.down_slices == 2
    tokens, traces = prompts_of(dev, 1, 16, 25)[0], []
    for slices in (2, 1):
        d.down_slices, d.layer_trace = slices, []
        d.load_prefix(tokens)
        traces.append(d.layer_trace[:cfg.layers])  # of the first chunk; its first layer sees the same input both times
    a, b = traces[0][0], traces[1][0]
    assert torch.equal(a["act"], b["act"])
    assert (a["delta"] - b["delta"]).norm() <= 2.0 ** -20 * b["delta"].norm()
