"""Ranks of log_probs in rows that hold NaN or infinities, on gfx950 against the plain form (oracle/experts_oracle.py): whole
numbers, equal in every row."""

import numpy as np
import pytest
import torch

import experts_oracle as X
from test_gpu_logprobs import BF16, F16, F32, np64
from tinygrad_mi355x.sampling import log_probs

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def rows_of(vocab):
    """Rows that are not finite, and the tokens that are looked at in each."""
    rng = np.random.default_rng(vocab)
    base = np.round(rng.standard_normal(vocab) * 4) / 4  # many equal ones
    a, b, last = vocab // 3, vocab // 2, vocab - 1

    def row(**at):
        x = base.copy()
        for value, where in at.items():
            x[where] = dict(nan=NAN, inf=INF, low=-INF, zero=0.0, minus=-0.0)[value]
        return x

    some = rng.integers(0, vocab, max(1, vocab // 10))
    return [row(nan=[a]), row(nan=[0, last]), row(nan=some), row(nan=slice(None)), row(nan=slice(1, None)), row(inf=[b]),
            row(inf=[0, a, last]), row(inf=[b], nan=[a, last]), row(low=slice(None, None, 3), nan=[1, a, last]), row(low=slice(None)),
            row(low=slice(None), nan=some), row(low=slice(None), inf=[b]), row(zero=slice(None, None, 2), minus=slice(1, None, 2), nan=[a]),
            row(low=slice(2, None))]


def check(x, tokens, top):
    got = log_probs(x, tokens, top=top)
    want = X.log_probs(np64(x), tokens.cpu().numpy(), top)
    np.testing.assert_array_equal(got.ranks.cpu().numpy(), want[1])
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), want[3])
    np.testing.assert_array_equal(np.isnan(np64(got.logprobs)), np.isnan(want[0]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 70, 4099, 32000, 70001])
def test_ranks_of_what_is_not_finite(dev, dtype, vocab):
    print(f"ranks {dtype} {vocab}", flush=True)
    x = torch.from_numpy(np.stack(rows_of(vocab)) if vocab > 2 else np.array([[NAN] * vocab, [INF] * vocab, [-INF] * vocab, [0.0] * vocab]))
    x = x.to(dtype).to(dev)
    for token in sorted({0, 1, 2, 5, 9, vocab // 3, vocab // 3 + 1, vocab // 2, vocab - 2, vocab - 1} & set(range(vocab))):
        check(x, torch.full((len(x),), token, dtype=torch.int32, device=dev), min(3, vocab))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [37, 4099, 66001])
def test_ranks_in_rows_of_every_alignment(dev, dtype, vocab):
    """What lies beside a row, NaN or infinities, does not count."""
    rows = rows_of(vocab)
    for off in (0, 1, 3, 6, 7):
        for around in (NAN, INF, -INF):
            flat = torch.full((len(rows) * (vocab + 11) + 16,), around, dtype=dtype, device=dev)
            x = flat[off:off + len(rows) * (vocab + 11)].view(len(rows), vocab + 11)[:, 1:1 + vocab]
            x.copy_(torch.from_numpy(np.stack(rows)).to(dtype))
            for token in (0, 8, vocab // 3, vocab - 1):
                check(x, torch.full((len(rows),), token, dtype=torch.int32, device=dev), 2)


def test_ranks_in_many_rows(dev):
    """Rows of 64 logits a thread."""
    x = torch.randn((600, 5003), device=dev, generator=torch.Generator(dev).manual_seed(1)).to(BF16)
    x[::3, 77] = NAN
    x[1::3, 100:900] = -INF
    tokens = torch.arange(600, dtype=torch.int32, device=dev) * 8
    tokens[::6] = 77
    check(x, tokens, 4)


def test_ranks_again_and_captured(dev):
    rows = torch.from_numpy(np.stack(rows_of(40000))).to(F32).to(dev)
    x, tokens = rows.clone(), torch.full((len(rows),), 13333, dtype=torch.int32, device=dev)
    log_probs(x, tokens, top=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = log_probs(x, tokens, top=3)
    for shift in (0, 3, 7):
        x.copy_(rows.roll(shift, 0))
        tokens.fill_(13333 + shift)
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(got.ranks.cpu().numpy(), X.log_probs(np64(x), tokens.cpu().numpy(), 3)[1])
