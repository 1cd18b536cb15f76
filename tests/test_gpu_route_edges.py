"""Routing where scores are small or rows are not finite, on gfx950 against the plain 64-bit form (oracle/experts_oracle.py).

Tolerances are those of test_gpu_experts: chosen logits lie within 20 of each other, and those that do not have weights
below 1e-8 or are compared by a bound of their own.
"""

import numpy as np
import pytest
import torch

import experts_oracle as X
from test_gpu_experts import BF16, F32, np64, routes
from tinygrad_mi355x.experts import route

pytestmark = pytest.mark.gpu


def check(dev, x, top_k, bias=None, dtype=F32, **kw):
    x = torch.from_numpy(np.asarray(x)).to(dtype).to(dev)
    b = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).to(dev)
    got = route(x, top_k, bias=b, **kw)
    routes(got, X.route(np64(x), top_k, bias=None if b is None else np64(b), **kw))
    return got


# ----------------------------------------------------------------------------- scores far below the largest
def test_weights_of_small_scores(dev):
    """Two chosen logits one apart are 0.731 and 0.269 wherever they lie; a single one is the scale."""
    want = np.array([1 / (1 + np.exp(-1.0)), 1 / (1 + np.exp(1.0))])
    for low in (1.0, 60.0, 88.0, 95.0, 103.0, 150.0, 700.0):
        got = check(dev, [[0.0, -low, -low - 1, -2.0]], 2, [0, 10, 10, 0])
        np.testing.assert_allclose(np64(got.weights)[0], want, rtol=3e-6)
    for low in (10.0, 80.0, 88.2, 100.0, 103.5, 120.0, 700.0):
        if low >= 80.0:  # the quotient of two sigmoids is that of the exponentials
            got = check(dev, [[-low, -low - 1]], 2, score="sigmoid")
            np.testing.assert_allclose(np64(got.weights)[0], want, rtol=3e-6)
        got = check(dev, [[-low, -low - 1]], 1, score="sigmoid", scale=2.5)
        assert abs(float(got.weights) - 2.5) <= 2.5 * 3e-6


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,groups,top_k", [(8, 1, 3), (64, 1, 20), (64, 8, 6), (96, 3, 8), (256, 8, 8), (1024, 1, 8)])
def test_route_of_small_scores(dev, dtype, experts, groups, top_k):
    """Softmax rows whose bias picks experts far below the largest logit, and sigmoid rows of low logits."""
    rng = np.random.default_rng(experts)
    top_groups = (groups + 1) // 2
    for low in (30.0, 89.0, 97.0, 104.0, 200.0, 600.0):
        x = rng.standard_normal((21, experts)) * 1.5 - low
        x[::2, experts // 2] = 0.5  # the largest, which the bias leaves out
        bias = rng.standard_normal(experts) * 0.01 + 10
        bias[experts // 2] = -10
        for renormalize in (True, False):
            kw = dict(groups=groups, top_groups=top_groups, renormalize=renormalize, scale=2.5)
            check(dev, x, top_k, bias, dtype, **kw)
            check(dev, x - 0.5, top_k, bias, dtype, score="sigmoid", **kw)
            check(dev, x - 0.5, top_k, None, dtype, score="sigmoid", renormalize=renormalize, scale=2.5)


def test_weights_of_scores_far_apart(dev):
    """Chosen scores of e^0 to e^-90 side by side: d = x - largest is off by half a step of up to 128, 128 2^-24 = 7.7e-6 of e^d,
    and 30 roundings as elsewhere."""
    x = np.array([[0.0, -20.25, -41.5, -63.125, -80.75, -5.0]] * 3) - np.array([[0.0], [3.0], [300.0]])
    for score in ("softmax", "sigmoid"):
        t = torch.from_numpy(x.astype(np.float32)).to(dev)
        got = route(t, 5, score=score, bias=torch.tensor([8.0, 7, 6, 5, 4, -9], device=dev), scale=0.5)
        ids, weights = X.route(np64(t), 5, score, np.array([8.0, 7, 6, 5, 4, -9]), scale=0.5)
        np.testing.assert_array_equal(got.ids.cpu().numpy(), ids)
        np.testing.assert_allclose(np64(got.weights), weights, rtol=1e-5, atol=1e-37)


def test_weights_without_a_score(dev):
    """Chosen logits of -infinity have no score: zero, beside others and alone."""
    inf = float("inf")
    x = [[-inf, -inf, 1.0, 2.0], [-inf] * 4, [-200.0, -inf, 5.0, -201.0], [-inf, -inf, -inf, 0.0]]
    for score in ("softmax", "sigmoid"):
        got = check(dev, x, 2, [5, 5, 0, 0], score=score)
        assert got.weights[[0, 1, 3]].eq(0).all() and got.weights[2].tolist() == [1.0, 0.0]


# ----------------------------------------------------------------------------- rows that are not finite
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_k", [(8, 1, 4), (64, 1, 14), (64, 1, 15), (64, 8, 14), (96, 3, 13), (256, 8, 12), (512, 1, 30),
                                                  (1024, 4, 40)])
def test_route_of_rows_with_a_nan(dev, score, experts, groups, top_k):
    """Rows with a NaN or +infinity beside rows whose keys lie next to a border: their experts too are those of 64-bit keys,
    each named once; under a softmax every key of such a row is NaN, and the experts come by index."""
    rng = np.random.default_rng(experts + top_k)
    x = rng.standard_normal((60, experts))
    x[15:45] = np.round(x[15:45])  # many equal ones
    x[::3, rng.integers(0, experts, 20)] = np.nan
    x[1::7, experts // 3] = np.inf
    x[4::9, rng.integers(0, experts, 7)] = -np.inf
    undone = -(1 / (1 + np.exp(-np.nan_to_num(x[1].astype(np.float32).astype(np.float64), posinf=0, neginf=0))))
    for bias in (undone + rng.standard_normal(experts) * 1e-9, np.zeros(experts), np.round(rng.standard_normal(experts)) * 1000,
                 np.where(np.arange(experts) % 3 == 0, -np.inf, 0.25), None):
        for top_groups in sorted({groups, (groups + 1) // 2}):
            got = check(dev, x, top_k, bias, score=score, groups=groups, top_groups=top_groups)
            assert all(len(set(row)) == top_k for row in got.ids.tolist())


def test_rows_with_a_nan_next_to_a_border(dev):
    """Rows with a NaN whose keys differ in 64 bits alone: all of them, and four around the last chosen one beside rows of the
    same wave that have them earlier."""
    for seed in range(12):
        rng = np.random.default_rng(seed)
        for experts, top_k in ((8, 3), (64, 9), (256, 8)):
            x = np.repeat(rng.standard_normal((1, experts)), 24, 0).astype(np.float32)
            bias = rng.standard_normal(experts) * 1e-9 - 1 / (1 + np.exp(-x[0].astype(np.float64)))
            x[::2, 2] = x[1::2, experts - 1] = np.nan
            check(dev, x, top_k, bias, score="sigmoid")
        route(torch.randn((64, 64), device=dev), 1, groups=64, top_groups=63)
        x = np.repeat(rng.standard_normal((1, 64)), 40, 0).astype(np.float32)
        x[:, :3] = 8
        keys = 2 - 0.01 * np.arange(64)
        keys[13:17] = keys[13] - 1e-7 * rng.permutation(4)
        bias = keys - 1 / (1 + np.exp(-x[0].astype(np.float64)))
        x[::2, :3] = -np.inf
        x[1::2, 63] = np.nan
        got = check(dev, x, 14, bias, score="sigmoid")
        assert all(len(set(row)) == 14 for row in got.ids.tolist())
