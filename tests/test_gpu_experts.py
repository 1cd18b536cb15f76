"""The mixture-of-experts operators on gfx950 against their plain 64-bit forms (oracle/experts_oracle.py).

Tolerances.  A rounding to type t is off by at most half a step, eps(t) / 2 of the value.  A sum of n products in 32 bits is
off by at most n eps(f32) / 2 of the products' sizes summed.
"""

import numpy as np
import pytest
import torch

import experts_oracle as X
import packed_oracle as O
from tinygrad_mi355x.codegen.decomp.mi355x import PackedTensor
from tinygrad_mi355x.experts import PackedExperts, route

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
@pytest.mark.parametrize("experts,groups,top_k", [(64, 8, 6), (64, 1, 30), (256, 8, 8), (12, 4, 2), (96, 1, 17), (512, 16, 8), (1024, 2, 60)])
def test_route_by_large_biases(dev, score, experts, groups, top_k):
    """Biases that are much larger than the scores, many of them equal: experts in runs of equal 32-bit keys, groups whose
    two best keys cancel."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((30, experts)).astype(np.float32) * 2
    for bias in (np.round(rng.standard_normal(experts)) * 1000, np.where(np.arange(experts) % 2 == 0, 5000.0, -5000.0) +
                 rng.standard_normal(experts), np.full(experts, 3e4), np.where(np.arange(experts) % 3 == 0, -np.inf, 0.25)):
        bias = bias.astype(np.float32)
        got = route(torch.from_numpy(x).to(dev), top_k, score=score, bias=torch.from_numpy(bias).to(dev), groups=groups,
                    top_groups=(groups + 1) // 2)
        routes(got, X.route(x, top_k, score, bias, groups, (groups + 1) // 2))


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


# ----------------------------------------------------------------------------- the experts' products
BITS = {"fp4_e2m1": 4, "fp6_e2m3": 6, "fp6_e3m2": 6, "int4": 4, "uint4": 4}


def packed(dev, rng, fmt, shape, scales, block):
    """A packed weight of values of about 0.1, and the values."""
    codes = rng.integers(0, 1 << BITS[fmt], shape).astype(np.uint8)
    data = O.pack_codes(codes.reshape(-1, shape[-1]), BITS[fmt])
    if scales is None:
        sc = numbers = None
    elif scales == "e8m0":
        e = rng.integers(120, 124, shape[:-1] + (shape[-1] // block,)).astype(np.uint8)
        sc, numbers = torch.from_numpy(e).to(dev).view(torch.float8_e8m0fnu), O.e8m0_decode(e)
    else:
        sc = torch.from_numpy(rng.random(shape[:-1] + (shape[-1] // block,)) * 0.02 + 0.005).to(scales).to(dev)
        numbers = np64(sc)
    w = PackedTensor(torch.from_numpy(data).to(dev), fmt, shape, sc, block)
    flat = (int(np.prod(shape[:-1])), shape[-1])
    values = O.dequant_f64(data, fmt, flat, None if numbers is None else numbers.reshape(flat[0], -1), block)
    return w, np.asarray(values, np.float64).reshape(shape)


class Layer:
    """Experts, and their values in 64 bits."""

    def __init__(self, dev, fmt, experts, hidden, ffn, scales="e8m0", block=32, seed=0):
        rng = np.random.default_rng(seed)
        gate_up, self.gate_up = packed(dev, rng, fmt, (experts, 2 * ffn, hidden), scales, block)
        down, self.down = packed(dev, rng, fmt, (experts, hidden, ffn), scales, block)
        self.e = PackedExperts(gate_up, down)

    def check(self, got, x, ids, weights):
        want, tol = X.experts(np64(x), ids.cpu().numpy(), np64(weights), self.gate_up, self.down, torch.finfo(x.dtype).eps)
        tol = tol + torch.finfo(got.dtype).eps / 2 * (np.abs(want) + tol) + 2.0 ** -25
        off = np.abs(np64(got) - want) - tol
        assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.size} off, by up to {off.max():.3g} over the tolerance"


def choice(dev, seed, tokens, experts, top_k, skew=1.0):
    """Different experts for each token, some more often than others."""
    rng = np.random.default_rng(seed)
    score = rng.standard_normal((tokens, experts)) + skew * rng.standard_normal(experts)
    ids = np.argsort(-score, axis=1)[:, :top_k].astype(np.int32)
    return torch.from_numpy(np.ascontiguousarray(ids)).to(dev), torch.from_numpy(rng.random((tokens, top_k)).astype(np.float32)).to(dev)


FORMATS = [("fp4_e2m1", "e8m0", 32), ("fp4_e2m1", None, 32), ("fp6_e2m3", "e8m0", 32), ("fp6_e3m2", "e8m0", 32), ("fp6_e2m3", None, 32),
           ("int4", F16, 128), ("int4", BF16, 64), ("int4", F32, 32), ("uint4", F16, 32), ("uint4", F32, 128), ("uint4", F32, 64), ("int4", None, 32)]


@pytest.mark.parametrize("fmt,scales,block", FORMATS)
def test_experts_of_every_format(dev, fmt, scales, block):
    print(f"experts {fmt} {scales} {block}", flush=True)
    layer = Layer(dev, fmt, 5, 256, 384, scales, block)
    size = 0.02 if scales is None else 0.5
    for tokens, top_k in ((1, 2), (7, 3), (70, 2), (150, 3), (333, 4)):
        ids, weights = choice(dev, tokens, tokens, 5, top_k)
        x = randn(dev, tokens, tokens, 256, dtype=layer.e.dtype, scale=size)
        layer.check(layer.e.apply(x, ids, weights), x, ids, weights)


@pytest.mark.parametrize("fmt,scales,block", [("fp4_e2m1", "e8m0", 32), ("int4", F16, 128)])
@pytest.mark.parametrize("experts,hidden,ffn", [(1, 128, 128), (3, 640, 128), (8, 128, 1152), (64, 256, 256), (130, 128, 128)])
def test_experts_of_every_size(dev, fmt, scales, block, experts, hidden, ffn):
    print(f"experts {fmt} {experts} {hidden} {ffn}", flush=True)
    layer = Layer(dev, fmt, experts, hidden, ffn, scales, block)
    for tokens in (1, 2, 3, 8, 16, 17, 31, 65, 200):
        top_k = min(experts, 1 + tokens % 8)
        ids, weights = choice(dev, tokens, tokens, experts, top_k)
        x = randn(dev, tokens, tokens, hidden, dtype=layer.e.dtype, scale=0.5)
        layer.check(layer.e.apply(x, ids, weights), x, ids, weights)


def named(rows):
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("fmt,scales,block", [("fp4_e2m1", "e8m0", 32), ("uint4", BF16, 64)])
@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_experts_that_tokens_may_name(dev, fmt, scales, block, tokens):
    """None at all, ids of other machines' experts, one expert for all, the same one twice; weights that are NaN where no
    expert is named; weights of zero and below."""
    layer = Layer(dev, fmt, 6, 256, 256, scales, block)
    x = randn(dev, 1, tokens, 256, dtype=layer.e.dtype, scale=0.5)
    w = randn(dev, 2, tokens, 3)
    none = torch.full((tokens, 3), -1, dtype=torch.int32, device=dev)
    assert torch.equal(layer.e.apply(x, none, w * float("nan")), torch.zeros_like(x))
    for row in ([2, 2, 2], [5, -1, 5], [-7, 0, 6], [2 ** 31 - 1, -2 ** 31, 3], [0, 1, 2]):
        ids = named([row] * tokens).to(dev)
        ids[tokens // 2:, 0] = 4
        ids[::3] = -1
        clean = torch.where((ids < 0) | (ids >= 6), torch.full_like(w, float("nan")), w)
        got = layer.e.apply(x, ids, clean)
        layer.check(got, x, ids, torch.where(clean != clean, torch.zeros_like(w), clean))
        assert not got[::3].any()


def test_experts_of_views(dev):
    layer = Layer(dev, "fp4_e2m1", 8, 256, 256)
    ids, weights = choice(dev, 1, 50, 8, 2)
    rows = randn(dev, 1, 50, 3, 256, dtype=BF16)
    for x in (rows[:, 1], rows[:, 2], rows.view(150, 256)[:50], rows[0:1, 0]):
        i, w = ids[:x.shape[0]], weights[:x.shape[0]]
        want = layer.e.apply(x.contiguous(), i, w)
        layer.check(want, x, i, w)
        assert torch.equal(layer.e.apply(x, i, w), want)
        wide = torch.zeros((x.shape[0], 2, 256 + 1), device=dev)
        got = layer.e.apply(x, i, w, out=wide[:, 1, 1:])  # rows apart, not aligned to vectors
        layer.check(got, x, i, w)
        assert torch.equal(got.to(BF16), want) and not wide[:, 0].any() and not wide[:, 1, 0].any()
        same = x.clone()
        assert layer.e.apply(same, i, w, out=same) is same and torch.equal(same, want)
    empty = rows.view(150, 256)[:0]
    assert layer.e.apply(empty, ids[:0], weights[:0]).shape == (0, 256)


@pytest.mark.parametrize("tokens", [2, 300])
def test_experts_again_and_on_other_streams(dev, tokens):
    """Bit for bit alike whenever and wherever they run, replays among eager work included."""
    layer = Layer(dev, "fp4_e2m1", 8, 256, 384)
    ids, weights = choice(dev, 1, tokens, 8, 2)
    x = randn(dev, 1, tokens, 256, dtype=BF16)
    want = layer.e.apply(x, ids, weights)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(layer.e.apply(x, ids, weights))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.e.apply(x, ids, weights)
    for seed in (5, 6, 7):
        x.copy_(randn(dev, seed, tokens, 256, dtype=BF16))
        new = choice(dev, seed, tokens, 8, 2)
        ids.copy_(new[0])
        weights.copy_(new[1])
        want = layer.e.apply(x, ids, weights)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        layer.check(out, x, ids, weights)


def test_routed_experts(dev):
    """The two as a layer uses them: a router's logits, the choice, the products."""
    layer = Layer(dev, "fp4_e2m1", 16, 256, 256)
    for tokens in (1, 6, 100):
        x = randn(dev, tokens, tokens, 256, dtype=BF16)
        logits = x.float() @ randn(dev, 9, 256, 16, scale=0.1)
        r = route(logits, 4, score="sigmoid", bias=randn(dev, 3, 16, scale=0.1), groups=4, top_groups=2)
        ids, weights = X.route(np64(logits), 4, "sigmoid", np64(randn(dev, 3, 16, scale=0.1)), 4, 2)
        routes(r, (ids, weights))
        layer.check(layer.e.apply(x, r.ids, r.weights), x, r.ids, r.weights)


@pytest.mark.parametrize("fmt,scales,block", [("fp4_e2m1", "e8m0", 32), ("fp6_e2m3", "e8m0", 32), ("int4", F16, 32)])
@pytest.mark.parametrize("experts,hidden,ffn,tokens,top_k", [(64, 128, 1152, 600, 4), (64, 512, 1152, 300, 4), (24, 256, 2176, 700, 5),
                                                             (64, 640, 384, 60, 8)])
def test_more_tiles_than_workgroups(dev, fmt, scales, block, experts, hidden, ffn, tokens, top_k):
    """Workgroups that go through several tiles, of one K step up to more than are loaded ahead."""
    print(f"tiles {fmt} {experts} {hidden} {ffn} {tokens}", flush=True)
    layer = Layer(dev, fmt, experts, hidden, ffn, scales, block)
    ids, weights = choice(dev, tokens, tokens, experts, top_k)
    x = randn(dev, tokens, tokens, hidden, dtype=layer.e.dtype, scale=0.5)
    got = layer.e.apply(x, ids, weights)
    layer.check(got, x, ids, weights)
    for _ in range(3):
        assert torch.equal(layer.e.apply(x, ids, weights), got)


@pytest.mark.parametrize("tokens", [3, 40, 200])
def test_gates_of_every_size(dev, tokens):
    """Gates from 0 to a few hundred, of both signs: silu is the gate, or nothing."""
    layer = Layer(dev, "fp4_e2m1", 4, 256, 256)
    ids, weights = choice(dev, 1, tokens, 4, 2)
    x = randn(dev, 2, tokens, 256, dtype=BF16) * torch.logspace(-3, 2.5, tokens, device=dev)[:, None].to(BF16)
    gates = np64(x) @ layer.gate_up[0][::2].T
    assert gates.max() > 90 and gates.min() < -90
    layer.check(layer.e.apply(x, ids, weights, out=torch.empty((tokens, 256), device=dev)), x, ids, weights)


@pytest.mark.parametrize("fmt,scales,block", [("fp4_e2m1", "e8m0", 32), ("fp6_e3m2", "e8m0", 32), ("int4", F16, 64)])
def test_experts_at_the_border_of_few_tokens(dev, fmt, scales, block):
    """Calls of 1 to 17 tokens and up to 129 pairs, more than four tokens an expert among them."""
    layer = Layer(dev, fmt, 40, 256, 128, scales, block)
    for tokens, top_k in ((16, 8), (16, 9), (15, 8), (17, 7), (17, 1), (1, 40), (4, 32), (4, 33), (3, 40), (14, 9), (16, 2)):
        ids, weights = choice(dev, tokens, tokens, 40, top_k, skew=3.0)
        x = randn(dev, top_k, tokens, 256, dtype=layer.e.dtype, scale=0.5)
        layer.check(layer.e.apply(x, ids, weights), x, ids, weights)
    for tokens in (5, 16):  # all of them at the same experts
        ids = torch.tensor([[39, 2, 17]], dtype=torch.int32, device=dev).repeat(tokens, 1)
        weights = randn(dev, 3, tokens, 3)
        x = randn(dev, 4, tokens, 256, dtype=layer.e.dtype, scale=0.5)
        layer.check(layer.e.apply(x, ids, weights), x, ids, weights)


@pytest.mark.parametrize("tokens", [2, 40])
def test_experts_past_four_gib(dev, tokens):
    """The first and the last of experts whose codes pass 2^32 bytes give what they give alone."""
    experts, hidden, ffn = 80, 4096, 14336
    gen = torch.Generator(dev).manual_seed(1)

    def weight(rows, k):
        codes = torch.randint(0, 256, (experts * rows * k // 2,), dtype=torch.uint8, device=dev, generator=gen)
        sc = torch.randint(112, 120, (experts, rows, k // 32), dtype=torch.uint8, device=dev, generator=gen).view(torch.float8_e8m0fnu)
        return codes, sc

    def pack(w, shape):
        return PackedTensor(w[0], "fp4_e2m1", shape, w[1], 32)

    def ends(w, rows, k):
        n = rows * k // 2
        return torch.cat((w[0][:n], w[0][-n:])), torch.cat((w[1][:1].view(torch.uint8), w[1][-1:].view(torch.uint8))).view(w[1].dtype)

    up, down = weight(2 * ffn, hidden), weight(hidden, ffn)
    assert up[0].numel() > 2 ** 32
    every = PackedExperts(pack(up, (experts, 2 * ffn, hidden)), pack(down, (experts, hidden, ffn)))
    two = PackedExperts(pack(ends(up, 2 * ffn, hidden), (2, 2 * ffn, hidden)), pack(ends(down, hidden, ffn), (2, hidden, ffn)))
    ids = torch.randint(0, 2, (tokens, 2), dtype=torch.int32, device=dev, generator=gen)
    weights, x = randn(dev, 1, tokens, 2), randn(dev, 2, tokens, hidden, dtype=BF16)
    got, want = every.apply(x, ids * (experts - 1), weights), two.apply(x, ids, weights)
    # sums in another order: 14336 products, of a hidden value that may have rounded the other way (2^-8); what reads
    # another expert is off by the size of the rows
    assert (got.double() - want.double()).norm() <= 2.0 ** -6 * want.double().norm() and torch.isfinite(want).all()


@pytest.mark.parametrize("tokens,top_k", [(4096, 4), (4097, 4), (2500, 13)])
def test_more_pairs_than_registers_hold(dev, tokens, top_k):
    """16384 pairs and more, some of them of no expert: a row is what it is in a call of few tokens."""
    layer = Layer(dev, "fp4_e2m1", 16, 128, 128)
    ids, weights = choice(dev, tokens, tokens, 16, top_k)
    ids[torch.rand(ids.shape, generator=torch.Generator().manual_seed(1)).to(dev) < 0.1] = -1
    x = randn(dev, 1, tokens, 128, dtype=BF16, scale=0.5)
    got = layer.e.apply(x, ids, weights)
    layer.check(got, x, ids, weights)
    assert torch.equal(layer.e.apply(x, ids, weights), got)


def test_calls_of_several_threads(dev):
    """Threads that share two streams, of one layer and with other sizes in between."""
    from concurrent.futures import ThreadPoolExecutor

    from tinygrad_mi355x.sampling import log_probs

    layer = Layer(dev, "fp4_e2m1", 8, 256, 384)
    work = []
    for tokens in (1, 9, 40, 300):
        ids, weights = choice(dev, tokens, tokens, 8, 2)
        x = randn(dev, tokens, tokens, 256, dtype=BF16)
        logits, drawn = randn(dev, tokens, tokens, 40000), torch.arange(tokens, dtype=torch.int32, device=dev)
        work.append(lambda a=(x, ids, weights), b=(logits, drawn): (layer.e.apply(*a), *log_probs(*b, top=6), *route(b[0][:, :96], 8)))
    want = [w() for w in work]
    torch.cuda.synchronize()

    streams = torch.cuda.current_stream(), torch.cuda.Stream()

    def one(i):
        stream = streams[i % 2]
        with torch.cuda.stream(stream):
            got = [work[(i + j) % 4]() for j in range(12)]
        stream.synchronize()
        return all(torch.equal(a, b) for j, g in enumerate(got) for a, b in zip(g, want[(i + j) % 4]))

    with ThreadPoolExecutor(6) as pool:
        assert all(pool.map(one, range(12)))
