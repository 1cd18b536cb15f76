"""Prompts of a few tokens for several sequences: rows between the batch and the GEMV's 16."""

import pytest
import torch

from tinygrad_mi355x.decoder import Decoder, DecoderConfig, random_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,tokens", [(5, 2), (8, 2), (5, 3)])
def test_short_prompts_of_large_batches(dev, batch, tokens):
    """Prompts whose rows are more than the batch and at most 16: the down projection's K-slice parts hold `batch` rows,
    so they are not used there; the logits are those of one sequence at a time (fp32 sums in another order: an activation
    next to a border moves by a step of f16 or bf16, 2^-8 of it, and a logit is a sum over 256 such values: 2^-6 of the
    logits' norm bounds a shift of several of them)."""
    cfg = DecoderConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=4096, vocab=1000, layers=2)
    w = random_weights(cfg, dev, seed=10)
    prompts = torch.randint(0, cfg.vocab, (batch, tokens), generator=torch.Generator().manual_seed(11)).to(dev)
    many = Decoder(w, cfg, batch, 32, 8)
    assert many.down_slices == 2
    many.prefill(prompts)
    one = Decoder(w, cfg, 1, 32, 8)
    for b in range(batch):
        one.prefill(prompts[b:b + 1])
        assert (many.logits[b] - one.logits[0]).norm() <= 2.0 ** -6 * one.logits[0].norm()
