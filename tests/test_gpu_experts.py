"""The mixture-of-experts operators on gfx950 against their plain 64-bit forms (oracle/experts_oracle.py).

Tolerances.  A rounding to type t is off by at most half a step, eps(t) / 2 of the value.  A sum of n products in 32 bits is
off by at most n eps(f32) / 2 of the products' sizes summed.
"""

import numpy as np
import pytest
import torch

import experts_oracle as X
from tinygrad_mi355x.experts import route

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# weights in 32 bits: a score is e^d / sum, d off by half a step of up to 20 (1.2e-6 of e^d), 30 roundings of half a step
ROUTE_TOL = 3e-6


def np64(t: torch.Tensor) -> np.ndarray:
    return t.double().cpu().numpy()


def randn(dev, seed, *shape, dtype=F32, scale=1.0) -> torch.Tensor:
    x = np.random.default_rng(seed).standard_normal(shape) * scale
    return torch.from_numpy(x).to(dtype).to(dev)


def routes(got, want, tol=ROUTE_TOL):
    ids, weights = want
    np.testing.assert_array_equal(got.ids.cpu().numpy(), ids)
    np.testing.assert_allclose(np64(got.weights), weights, rtol=tol, atol=1e-37)


# ----------------------------------------------------------------------------- routing
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 1), (7, 7), (8, 2), (9, 3), (16, 4), (31, 5), (64, 6), (65, 8), (128, 8),
                                           (130, 1), (256, 8), (300, 12), (512, 8), (513, 3), (1000, 64), (1024, 8)])
def test_route(dev, dtype, experts, top_k):
    print(f"route {dtype} {experts} {top_k}", flush=True)
    for tokens, score, bias, renormalize in ((1, "softmax", False, True), (37, "sigmoid", True, True), (9, "softmax", True, False),
                                             (3, "sigmoid", False, False)):
        x = randn(dev, tokens, tokens, experts, dtype=dtype, scale=1.5)
        b = randn(dev, 5, experts, scale=0.1) if bias else None
        got = route(x, top_k, score=score, bias=b, renormalize=renormalize, scale=2.5)
        routes(got, X.route(np64(x), top_k, score, None if b is None else np64(b), 1, 1, renormalize, 2.5))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(256, 8, 4, 8), (64, 8, 3, 6), (6, 2, 1, 3), (12, 12, 5, 5), (60, 4, 2, 7),
                                                             (96, 3, 2, 64), (1024, 64, 7, 8), (320, 64, 64, 8), (10, 5, 1, 2)])
def test_route_of_groups(dev, dtype, experts, groups, top_groups, top_k):
    print(f"groups {dtype} {experts} {groups} {top_groups}", flush=True)
    for tokens, score, bias in ((33, "sigmoid", True), (5, "softmax", False), (4, "softmax", True)):
        x = randn(dev, tokens, tokens, experts, dtype=dtype, scale=1.5)
        b = randn(dev, 5, experts, scale=0.1) if bias else None
        got = route(x, top_k, score=score, bias=b, groups=groups, top_groups=top_groups)
        routes(got, X.route(np64(x), top_k, score, None if b is None else np64(b), groups, top_groups))


@pytest.mark.parametrize("experts,groups", [(8, 1), (64, 8), (256, 8)])
def test_route_next_to_a_border(dev, experts, groups):
    """Keys that differ in the 64-bit values alone, and keys that do not differ: biases that undo the scores but for a part
    in 10^9, and equal logits."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((40, experts)).astype(np.float32)
    x[20:] = np.round(x[20:])  # many equal ones
    bias = -(1 / (1 + np.exp(-x[0].astype(np.float64))))
    bias = (bias + rng.standard_normal(experts) * 1e-9).astype(np.float32)
    for b in (bias, np.zeros(experts, np.float32), None):
        got = route(torch.from_numpy(x).to(dev), 4, score="sigmoid", bias=None if b is None else torch.from_numpy(b).to(dev),
                    groups=groups, top_groups=max(1, groups // 2))
        routes(got, X.route(x, 4, "sigmoid", b, groups, max(1, groups // 2)))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_what_is_not_finite(dev, score):
    inf, nan = float("inf"), float("nan")
    rows = [[1, -inf, 2, -inf, 0, -inf, -inf, 3], [-inf] * 8, [nan, 1, 2, 3, nan, 5, 6, 7], [nan] * 8, [0, inf, 1, 2, 3, 4, 5, 6],
            [-3e38, 3e38, 0, 1, 2, 3, -0.0, 0.0], [-0.0, 0.0] * 4]
    x = torch.tensor(rows, dtype=F32, device=dev)
    got = route(x, 6, score=score)
    ids, weights = X.route(np64(x), 6, score)
    if score == "softmax":
        weights[4] = np.nan  # +infinity
    routes(got, (ids, weights))


def test_route_of_views(dev):
    """Rows that are apart, and not aligned to vectors of four."""
    flat = randn(dev, 1, 20 * 70 + 1)
    for x in (flat[:-1].view(20, 70)[:, :64], flat[1:].view(20, 70)[:, 3:67], flat[:1280].view(20, 64)[3::4]):
        routes(route(x, 6), X.route(np64(x), 6))
    assert route(flat[:0].view(0, 64), 6).ids.shape == (0, 6)


def test_route_again_and_on_another_stream(dev):
    x, b = randn(dev, 1, 4096, 256), randn(dev, 2, 256, scale=0.1)
    want = route(x, 8, score="sigmoid", bias=b, groups=8, top_groups=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route(x, 8, score="sigmoid", bias=b, groups=8, top_groups=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.ids, want.ids) and torch.equal(got.weights, want.weights)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = route(x, 8, score="sigmoid", bias=b, groups=8, top_groups=4)
    for seed in (5, 6, 7):
        x.copy_(randn(dev, seed, 4096, 256))
        want = route(x, 8, score="sigmoid", bias=b, groups=8, top_groups=4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.ids, want.ids) and torch.equal(got.weights, want.weights)
