"""The serving loop (quantised paged cache, common prefix, sampling) on gfx950."""

import math

import pytest
import torch

from tinygrad_mi355x.decoder import Decoder, DecoderConfig, random_weights
from tinygrad_mi355x.rotary import Rotary
from tinygrad_mi355x.serving import ServingDecoder

pytestmark = pytest.mark.gpu
SMALL = DecoderConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000, layers=2)


def prompts_of(dev, rows, n, seed=0):
    return torch.randint(0, SMALL.vocab, (rows, n), generator=torch.Generator().manual_seed(seed)).to(dev)


def plain_attend(cache, q, table, lengths, shared=0, scale=None, out=None):
    """Attention over what ``cache.read`` gives, in 64 bits."""
    b, t, h, hd = q.shape
    n = table.shape[1] * cache.page_size
    k, v = (x.double() for x in cache.read(table, torch.zeros_like(lengths), n, torch.float32))
    k, v = (x.repeat_interleave(h // cache.kv_heads, 2).transpose(1, 2).contiguous() for x in (k, v))
    s = torch.matmul(q.double().transpose(1, 2).contiguous(), k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    last = lengths[:, None] - t + torch.arange(t, device=q.device)
    s = s.masked_fill((torch.arange(n, device=q.device) > last[..., None])[:, None], -math.inf)
    return torch.matmul(torch.softmax(s, -1), v).transpose(1, 2).contiguous().to(q.dtype)


@pytest.mark.parametrize("prefix,k_format,v_format", [(0, "fp8_e4m3", "fp8_e4m3"), (128, "fp8_e4m3", "fp4_e2m1"),
                                                      (64, "fp4_e2m1", "fp8_e4m3")])
def test_serving_attends_over_its_cache(dev, prefix, k_format, v_format):
    """Every token's logits are those of a 64-bit attention over the stored keys and values.

    The two differ by fp32 summation in the attention (below 2^-17 of the outputs' scale), which the two layers' f16 and
    bf16 activations round anew: a value next to a border moves by a step, 2^-11 and 2^-8 of it, and a logit is a sum over
    256 such values: 2^-6 of the logits' norm bounds a shift of several of them."""
    w = random_weights(SMALL, dev, seed=1)
    d = ServingDecoder(w, SMALL, 3, 320, 48, prefix=prefix, k_format=k_format, v_format=v_format)
    d._filters = dict(temperature=torch.ones(3, device=dev))
    prompts = prompts_of(dev, 3, 100)

    def run():
        out = []
        d.load_prefix(prompts_of(dev, 1, max(prefix, 1), 5)[0][:prefix])
        d.u.fill_(0.5)
        d.prefill(prompts)
        out.append(d.logits.clone())
        for i in range(3):
            d.tokens[:3] = torch.tensor([i, 7, 11 * i], dtype=torch.int32, device=dev)  # the same tokens both times
            d._decode_step()
            out.append(d.logits.clone())
        return out

    got = run()
    for c in d.caches:
        c.attend = lambda q, table, lengths, c=c, **kw: plain_attend(c, q, table, lengths, **kw)
    want = run()
    for a, b in zip(got, want):
        assert torch.isfinite(a).all()
        assert (a - b).norm() <= 2.0 ** -6 * b.norm()


def test_serving_close_to_the_bf16_decoder(dev):
    """With fp8 keys and values the logits stay near those of the bf16 cache: each stored value is off by at most 2^-4 of
    itself (2^-5 on average), independently, so an attention output by about 2^-5 of its scale, and the residual stream,
    which the embedding (norm 1 a value) leads, by less."""
    w = random_weights(SMALL, dev, seed=2)
    prompts = prompts_of(dev, 2, 60, 3)
    base = Decoder(w, SMALL, 2, 128, 64)
    base.prefill(prompts)
    d = ServingDecoder(w, SMALL, 2, 128, 64)
    d._filters = dict(temperature=torch.zeros(2, device=dev))
    d.prefill(prompts)
    assert (d.logits - base.logits).norm() <= 2.0 ** -4 * base.logits.norm()


def test_generate_graph_prefix_and_filters(dev):
    """Replayed steps give the eager ones' tokens; greedy rows take the first maximum; a prefix held in common gives what
    the same tokens in front of every prompt give."""
    w = random_weights(SMALL, dev, seed=4)
    common, own = prompts_of(dev, 1, 128, 6)[0], prompts_of(dev, 4, 21, 7)
    u = torch.rand((4, 12), generator=torch.Generator().manual_seed(8)).to(dev)
    filters = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.3]), top_k=torch.tensor([0, 20, 0, 50]),
                   top_p=torch.tensor([1.0, 0.9, 0.95, 1.0]), min_p=0.01)
    d = ServingDecoder(w, SMALL, 4, 256, 40, prefix=128, v_format="fp4_e2m1",
                       rotary=Rotary(64, layout="interleaved", scaling=dict(kind="yarn", factor=4.0, trained=64)))
    d.load_prefix(common)
    eager = d.generate(own, 12, u, graph=False, **filters)
    for _ in range(2):
        assert torch.equal(d.generate(own, 12, u, **filters), eager)
        torch.cuda.synchronize()
    assert int(d.pos[0]) == 128 + 21 + 11
    assert eager.shape == (4, 12) and int(eager.min()) >= 0 and int(eager.max()) < SMALL.vocab
    alone = ServingDecoder(w, SMALL, 4, 256, 40, v_format="fp4_e2m1", rotary=d.rotary)
    d._filters = alone._filters = {k: v for k, v in d._filters.items()}
    d.prefill(own)
    with_common = d.logits.clone()
    alone.prefill(torch.cat((common.expand(4, -1), own), 1))
    assert (alone.logits - with_common).norm() <= 2.0 ** -6 * with_common.norm()


def test_serving_refuses(dev):
    w = random_weights(SMALL, dev, seed=9)
    for kw in (dict(prefix=63), dict(prefix=128), dict(page_size=24), dict(k_format="fp16"),
               dict(rotary=Rotary(128, device=dev))):
        with pytest.raises(ValueError):
            ServingDecoder(w, SMALL, 2, 128, 16, **kw)
    d = ServingDecoder(w, SMALL, 2, 128, 16, prefix=64)
    u = torch.rand((2, 4), device=dev)
    for call in (lambda: d.load_prefix(prompts_of(dev, 1, 63)[0]), lambda: d.prefill(prompts_of(dev, 3, 4)),
                 lambda: d.prefill(prompts_of(dev, 2, 65)), lambda: d.generate(prompts_of(dev, 2, 62), 4, u),
                 lambda: d.generate(prompts_of(dev, 2, 4), 5, u), lambda: d.prefill(prompts_of(dev, 2, 4) + 1000)):
        with pytest.raises(ValueError):
            call()
