"""A decoder whose feed-forward blocks are a mixture of experts, and the probabilities that the serving loop tells."""

from dataclasses import replace

import numpy as np
import pytest
import torch

import experts_oracle as X
from tinygrad_mi355x.codegen.decomp.mi355x import PackedTensor
from tinygrad_mi355x.decoder import Decoder, DecoderConfig, load_weights, random_weights, save_weights
from tinygrad_mi355x.experts import PackedExperts
from tinygrad_mi355x.sampling import log_probs
from tinygrad_mi355x.serving import ServingDecoder
from test_gpu_experts import np64, routes

pytestmark = pytest.mark.gpu
DENSE = DecoderConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000, layers=2)
MIXED = replace(DENSE, experts=6, experts_per_token=3)


def prompts_of(dev, rows, n, seed=0):
    return torch.randint(0, DENSE.vocab, (rows, n), generator=torch.Generator().manual_seed(seed)).to(dev)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (2, 3), (3, 40)])
def test_layers_of_experts(dev, score, batch, tokens):
    """Every layer's choice and output from the traced input: the router's logits within 32-bit sums of 256 products, the
    choice of those logits, and the experts' products within the bound that their own tests derive."""
    cfg = replace(MIXED, router_score=score)
    w = random_weights(cfg, dev, seed=1)
    d = Decoder(w, cfg, batch, 64, 48)
    d.layer_trace = []
    d.prefill(prompts_of(dev, batch, tokens))
    d.step()
    for i, tr in enumerate(d.layer_trace):
        L = w.layers[i % cfg.layers]
        x, r = np64(tr["xb"]), np64(L.router)
        off = np.abs(np64(tr["router"]) - x @ r.T) - 256 * 2.0 ** -24 * (np.abs(x) @ np.abs(r).T)
        assert (off <= 0).all()
        ids, weights = X.route(np64(tr["router"]), 3, score)

        class Choice:
            pass

        got = Choice()
        got.ids, got.weights = tr["ids"], tr["expert_weights"]
        routes(got, (ids, weights))
        gate_up, down = (np64(t.unpack(torch.float32)) for t in (L.w_gate_up, L.w_down))
        want, tol = X.experts(x, ids, np64(tr["expert_weights"]), gate_up, down, torch.finfo(torch.bfloat16).eps)
        assert (np.abs(np64(tr["delta"]) - want) <= tol + 2.0 ** -24 * np.abs(want)).all()
    assert len(d.layer_trace) == 2 * cfg.layers and d.layer_trace[0]["act"] is None


def test_equal_experts_are_one_block(dev):
    """Experts that are all alike give what the block itself gives: the weights sum to 1 within 2^-22, the hidden values are
    rounded at the same place, and sums in another order move some of them by a step (2^-8), as in the block's own forms:
    2^-6 of the logits' norm bounds a shift of several."""
    w = random_weights(DENSE, dev, seed=2)
    cfg = replace(DENSE, experts=4, experts_per_token=2)

    def repeated(t):
        return PackedTensor(t.data.repeat(4), t.format, (4, *t.shape), t.scales.view(torch.uint8).repeat(4, 1, 1).view(
            torch.float8_e8m0fnu), t.block_size)

    layers = [replace(L, w_gate_up=repeated(L.w_gate_up), w_down=repeated(L.w_down),
                      router=torch.randn((4, 256), device=dev).to(torch.bfloat16)) for L in w.layers]
    prompts = prompts_of(dev, 2, 20)
    one, many = Decoder(w, DENSE, 2, 64, 32), Decoder(replace(w, layers=layers), cfg, 2, 64, 32)
    for d in (one, many):
        d.prefill(prompts)
    assert (one.logits - many.logits).norm() <= 2.0 ** -6 * one.logits.norm()
    one.tokens.copy_(many.tokens)
    for d in (one, many):
        d.step()
    assert (one.logits - many.logits).norm() <= 2.0 ** -6 * one.logits.norm()


@pytest.mark.parametrize("batch", [1, 5])
def test_generate_replays_what_it_runs(dev, batch):
    """Replayed steps give the eager ones' tokens, with memory allocated and freed in between, in both decoders."""
    w = random_weights(MIXED, dev, seed=3)
    prompts, u = prompts_of(dev, batch, 9), torch.rand((batch, 10), generator=torch.Generator().manual_seed(1)).to(dev)
    d = Decoder(w, MIXED, batch, 64, 16)
    eager = d.generate(prompts, 10, graph=False)
    for _ in range(3):
        junk = [torch.full((1 << 16,), float("nan"), device=dev) for _ in range(8)]
        assert torch.equal(d.generate(prompts, 10), eager)
        del junk
    s = ServingDecoder(w, MIXED, batch, 64, 16)
    eager, told = s.generate(prompts, 10, u, temperature=0.9, top_k=40, graph=False, logprobs=5)
    for _ in range(3):
        tokens, again = s.generate(prompts, 10, u, temperature=0.9, top_k=40, logprobs=5)
        assert torch.equal(tokens, eager) and all(torch.equal(a, b) for a, b in zip(told, again))
    assert torch.equal(s.generate(prompts, 10, u, temperature=0.9, top_k=40), eager)
    assert told.logprobs.shape == told.ranks.shape == told.entropy.shape == (batch, 10) and told.top_ids.shape == (batch, 10, 5)
    assert int(told.ranks.max()) < 40 and torch.isfinite(told.logprobs).all()


def test_told_probabilities_are_the_logits(dev):
    d = ServingDecoder(random_weights(MIXED, dev, seed=4), MIXED, 3, 64, 16)
    u = torch.rand((3, 1), generator=torch.Generator().manual_seed(2)).to(dev)
    tokens, told = d.generate(prompts_of(dev, 3, 12), 1, u, temperature=1.3, logprobs=7)
    want = log_probs(d.logits, tokens[:, 0].contiguous(), top=7)
    assert all(torch.equal(a[:, 0], b) for a, b in zip(told, want))
    exact = X.log_probs(np64(d.logits), tokens[:, 0].cpu().numpy(), 7)
    np.testing.assert_allclose(np64(told.logprobs[:, 0]), exact[0], atol=2.0 ** -17, rtol=2.0 ** -22)


def test_weights_of_experts_go_to_disk(dev, tmp_path):
    w = random_weights(MIXED, dev, seed=5)
    save_weights(tmp_path / "m.safetensors", w, MIXED)
    v, cfg = load_weights(tmp_path / "m.safetensors", dev)
    assert cfg == MIXED
    prompts = prompts_of(dev, 2, 5)
    assert torch.equal(Decoder(v, cfg, 2, 32, 16).generate(prompts, 6), Decoder(w, cfg, 2, 32, 16).generate(prompts, 6))


def test_decoders_of_experts_refuse(dev):
    w = random_weights(MIXED, dev, seed=6)
    for cfg in (replace(MIXED, experts=5), replace(MIXED, experts_per_token=7), replace(MIXED, experts_per_token=0),
                replace(MIXED, router_score="relu"), replace(MIXED, ffn=256)):
        with pytest.raises(ValueError):
            Decoder(w, cfg, 1, 32, 16)
    for L in (replace(w.layers[0], router=None), replace(w.layers[0], router=w.layers[0].router.float())):
        with pytest.raises(ValueError):
            Decoder(replace(w, layers=[L, w.layers[1]]), MIXED, 1, 32, 16)
    d = ServingDecoder(w, MIXED, 1, 32, 16)
    with pytest.raises(ValueError):
        d.generate(prompts_of(dev, 1, 4), 2, torch.rand((1, 2), device=dev), logprobs=65)


def test_workspaces_of_fewer_tokens_are_no_larger(dev):
    L = random_weights(MIXED, dev, seed=7).layers[0]
    e = PackedExperts(L.w_gate_up, L.w_down)
    sizes = [e.workspace_bytes(t, 3) for t in (1, 2, 15, 16, 17, 42, 43, 200, 5000)]
    assert sizes == sorted(sizes)
