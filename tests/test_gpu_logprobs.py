"""Log probabilities on gfx950 against their plain 64-bit form (oracle/experts_oracle.py).

Tolerances.  A logit's distance d from the largest is rounded once in 32 bits, its exponential is off by 2^-22 and by d's own
rounding and that of d log2(e), 2^-23 |d|; sums of n such terms in 32 bits (32 a thread, 6 steps in a wave, 16 waves, stretches)
add 64 roundings.  exp(d) (1 + |d|) is at most 1, so of a sum both errors are at most (2^-22 + 2^-18), taken as 2^-17 here;
the results' own roundings are half a step of d and of the logarithm.
"""

import math

import numpy as np
import pytest
import torch

import experts_oracle as X
from tinygrad_mi355x.sampling import log_probs, sample

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def np64(t):
    return t.double().cpu().numpy()


def randn(dev, seed, *shape, dtype=F32, scale=1.0):
    x = np.random.default_rng(seed).standard_normal(shape) * scale
    return torch.from_numpy(x).to(dtype).to(dev)


def near(got, want, entropy=1.0):
    with np.errstate(over="ignore"):  # in 32 bits, where what is below -2^128 (logits of 3e38 and -3e38) is -infinity
        want = want.astype(np.float32)
    np.testing.assert_allclose(np64(got), want, rtol=2.0 ** -22, atol=2.0 ** -17 * entropy)


def check(logits, tokens, top):
    got = log_probs(logits, tokens, top=top)
    want = X.log_probs(np64(logits), tokens.cpu().numpy(), top)
    np.testing.assert_array_equal(got.ranks.cpu().numpy(), np.where(np.isnan(want[0]), got.ranks.cpu().numpy(), want[1]))
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), want[3])
    near(got.logprobs, want[0])
    # log S - T / S: T is up to S log n
    near(got.entropy, want[2], 2 + np.log(logits.shape[1]))
    near(got.top_logprobs, want[4])
    return got


def tokens_of(dev, seed, rows, vocab):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)).to(dev)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,top", [(1, 1), (2, 2), (7, 0), (63, 63), (64, 64), (65, 5), (500, 20), (1000, 64), (2047, 1), (4097, 17),
                                       (8191, 5), (16411, 64), (31999, 20), (32000, 5), (32768, 16), (32769, 16), (50257, 20), (131072, 5),
                                       (131073, 64), (200001, 33)])
def test_log_probs(dev, dtype, vocab, top):
    print(f"log_probs {dtype} {vocab} {top}", flush=True)
    for rows, scale in ((1, 3.0), (5, 0.01), (3, 30.0)):
        check(randn(dev, rows, rows, vocab, dtype=dtype, scale=scale), tokens_of(dev, rows, rows, vocab), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [300, 32000, 70000])
def test_log_probs_of_rows_of_their_own(dev, dtype, vocab):
    """Equal logits, sorted ones either way, one that outweighs all, few that are not -infinity, large ones side by side."""
    rng = np.random.default_rng(1)
    rows = [np.zeros(vocab), np.arange(vocab) / vocab * 5, -np.arange(vocab) / vocab * 5, np.where(np.arange(vocab) == 123, 90.0, 0.0),
            np.where(np.arange(vocab) % 97 == 5, rng.standard_normal(vocab), -np.inf), np.where(np.arange(vocab) < 250, 5.0, -5.0),
            np.round(rng.standard_normal(vocab) * 2), np.where(np.arange(vocab) == vocab - 1, 0.0, -np.inf),
            rng.standard_normal(vocab) * 1e4, np.where(np.arange(vocab) == 0, 3e38, -3e38)]
    logits = torch.from_numpy(np.stack(rows)).to(dtype).to(dev)
    for token in (0, 123, 124, vocab - 1):
        check(logits, torch.full((len(rows),), token, dtype=torch.int32, device=dev), 20)


@pytest.mark.parametrize("vocab", [70, 32000, 100000])
def test_log_probs_of_what_is_not_finite(dev, vocab):
    inf, nan = float("inf"), float("nan")
    x = randn(dev, 1, 5, vocab)
    x[0, 5] = nan
    x[1, vocab - 1] = inf
    x[2] = -inf
    x[3] = nan
    x[4, :vocab - 3] = -inf
    tokens = torch.tensor([1, 2, 3, 4, vocab - 2], dtype=torch.int32, device=dev)
    got = log_probs(x, tokens, top=8)
    for t in (got.logprobs, got.entropy, got.top_logprobs):
        assert torch.isnan(t[:4]).all()
    assert ((got.top_ids >= 0) & (got.top_ids < vocab)).all()
    assert got.top_ids[1, 0] == vocab - 1 and got.top_ids[2].tolist() == list(range(8)) == got.top_ids[3].tolist()
    check(x[4:], tokens[4:], 8)


def test_log_probs_of_no_token(dev):
    x = randn(dev, 1, 4, 32000)
    tokens = torch.tensor([-1, 32000, 5, -2 ** 31], dtype=torch.int32, device=dev)
    got = check(x, tokens, 3)
    assert got.logprobs[[0, 1, 3]].tolist() == [0.0] * 3 and got.ranks[[0, 1, 3]].tolist() == [-1] * 3
    assert log_probs(x[:0], tokens[:0], top=3).top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_of_views(dev, dtype):
    """Rows that are apart and of every alignment, of one stretch and of several; what lies around them does not count."""
    for vocab in (501, 32003, 32766, 65531):
        flat = torch.full((4 * (vocab + 13) + 9,), 1e4, dtype=dtype, device=dev)
        for off in (0, 1, 3, 6, 7):
            x = flat[off:off + 4 * (vocab + 13)].view(4, vocab + 13)[:, 2:2 + vocab]
            x.copy_(randn(dev, off, 4, vocab, dtype=dtype))
            check(x, tokens_of(dev, off, 4, vocab), 9)
            x.fill_(1e4)


def test_log_probs_again_and_captured(dev):
    for rows, vocab in ((6, 32000), (2, 131072)):
        x, tokens = randn(dev, 1, rows, vocab), tokens_of(dev, 1, rows, vocab)
        want = log_probs(x, tokens, top=20)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = log_probs(x, tokens, top=20)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = log_probs(x, tokens, top=20)
        for seed in (5, 6, 7):
            x.copy_(randn(dev, seed, rows, vocab))
            tokens.copy_(tokens_of(dev, seed, rows, vocab))
            want = log_probs(x, tokens, top=20)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_log_probs_of_sampled_tokens(dev):
    """As a serving step uses them: the greedy token ranks first, a token of the k largest before k."""
    logits = randn(dev, 1, 16, 32000, scale=3.0)
    u = torch.rand(16, device=dev)
    got = check(logits, sample(logits, u, temperature=0.0), 5)
    assert not got.ranks.any() and torch.equal(got.top_logprobs[:, 0], got.logprobs)
    got = check(logits, sample(logits, u, top_k=7), 7)
    assert int(got.ranks.max()) < 7


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_ranks_of_tokens_that_are_ruled_out(dev, dtype):
    """-infinity ranks by index behind what is finite, in rows of every alignment, of one stretch and of several."""
    for vocab in (40, 32001, 66000):
        flat = torch.zeros(vocab + 16, dtype=dtype, device=dev)
        for off in (0, 1, 5, 7):
            x = flat[off:off + vocab].view(1, vocab)
            x.copy_(randn(dev, off, 1, vocab, dtype=dtype))
            x[0, ::3] = -float("inf")
            for token in (0, 3, 9, 36, vocab - 1 - (vocab - 1) % 3):
                check(x, torch.tensor([token], dtype=torch.int32, device=dev), 5)


def test_log_probs_past_four_gib(dev):
    """Rows on both sides of 2^32 bytes are what they are alone."""
    rows, vocab = 70000, 32000
    logits = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=dev)
    some = torch.tensor([0, 33553, 33554, 67107, 67108, 67109, rows - 1], device=dev)
    logits[some] = torch.randn((7, vocab), device=dev, generator=torch.Generator(dev).manual_seed(0)).to(torch.bfloat16) * 3
    tokens = torch.arange(rows, dtype=torch.int32, device=dev) % vocab
    got = log_probs(logits, tokens, top=5)
    alone = log_probs(logits[some].contiguous(), tokens[some].contiguous(), top=5)
    assert torch.equal(got.ranks[some], alone.ranks) and torch.equal(got.top_ids[some], alone.top_ids)
    for a, b in ((got.logprobs, alone.logprobs), (got.entropy, alone.entropy), (got.top_logprobs, alone.top_logprobs)):
        assert torch.allclose(a[some], b, rtol=1e-5, atol=1e-5)  # two orders of 32000 terms summed in 32 bits
    flat = torch.full_like(got.logprobs, -math.log(vocab))
    flat[some] = got.logprobs[some]
    assert torch.allclose(got.logprobs, flat, rtol=1e-5, atol=0)


@pytest.mark.parametrize("vocab", [32769, 65537, 70001, 131072, 400000, 1 << 20])
@pytest.mark.parametrize("top", [1, 7, 64])
def test_lists_of_stretches(dev, vocab, top):
    """Rows in several stretches whose likeliest tokens lie in one of them, are all alike, are few, or are masked but for a few."""
    print(f"stretches {vocab} {top}", flush=True)
    x = torch.randn((6, vocab), device=dev, generator=torch.Generator(dev).manual_seed(vocab + top))
    x[1, vocab // 2:vocab // 2 + 100] += 20
    x[2] = 1.25
    x[3] = float("-inf")
    x[3, [5, vocab - 1]] = 2.0
    x[4, :vocab - 40] = float("-inf")
    x[5] = torch.arange(vocab, device=dev) / vocab  # rising: all of them in the last stretch
    tokens = torch.tensor([0, vocab // 2, vocab - 1, 5, vocab - 2, 17], dtype=torch.int32, device=dev)
    check(x, tokens, top)
