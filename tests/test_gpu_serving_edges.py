"""The serving operators where their arguments end: filters that keep one token, infinite temperatures, queries and scores
that are not finite, positions that nobody wrote, tensors that overlap (tolerances: test_gpu_serving.py)."""

import math

import pytest
import torch

from tinygrad_mi355x.rotary import Rotary
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.sampling import sample
from test_gpu_serving import BF16, F16, F32, check_sample, i32, make_cache, make_table, randn

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("head_dim,rotary_dim,layout", [(64, None, "half"), (128, None, "half"), (128, None, "interleaved"),
                                                        (128, 64, "half"), (64, 32, "interleaved"), (96, None, "half"),
                                                        (80, 48, "interleaved")])
def test_rotate_rounds_to_32_bits_and_then_to_its_type(dev, dtype, head_dim, rotary_dim, layout):
    """16-bit results are the 32-bit ones rounded, also where that is a tie which the exact value is not; the cache write's
    queries are those of ``rotate``."""
    print(f"roundings {dtype} {head_dim} {rotary_dim} {layout}", flush=True)
    rot, start = Rotary(head_dim, rotary_dim, layout=layout, device=dev), i32(dev, [5, 1000, 77777])
    x = randn(dev, 80, 3, 400, 16, head_dim, dtype=dtype)
    got = rot.rotate(x, start)
    assert torch.equal(got, rot.rotate(x.float(), start).to(dtype))
    if head_dim in (64, 128):
        c, none = make_cache(dev, 1, 1, head_dim, 64, "fp8_e4m3", "fp8_e4m3"), torch.full((3, 1), -1, dtype=torch.int32, device=dev)
        k = randn(dev, 81, 3, 400, 1, head_dim, dtype=dtype)
        assert torch.equal(c.append(k, k, none, start, rotary=rot, q=x).q, got)


# ----------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [400, 513, 1000, 2048, 5000])
@pytest.mark.parametrize("top_p", [0.0, -1.0, -math.inf])
def test_sample_keeps_the_largest_of_flat_rows(dev, dtype, n, top_p):
    """A top_p of 0 and less keeps the first maximum alone, also among tokens of nearly one weight."""
    print(f"flat rows {dtype} {n} {top_p}", flush=True)
    g = torch.Generator().manual_seed(n)
    flat, spread = torch.rand(2, n, generator=g) * 0.001, torch.randn(2, n, generator=g)
    for x, temperature in ((flat, 1.0), (spread, 500.0), (torch.ones(2, n), 0.7)):
        x = x.to(dtype)
        for u, min_p in ((torch.rand(2, generator=g), 0.0), (torch.zeros(2), 0.0), (torch.rand(2, generator=g), 0.5)):
            got = check_sample(dev, x, u, temperature, 0, top_p, min_p)
            assert torch.equal(got.cpu().long(), x.float().argmax(1))


@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1e30])
@pytest.mark.parametrize("n", [300, 1000, 2048, 5000])
def test_sample_at_huge_temperatures(dev, n, temperature):
    """An infinite temperature weighs all finite logits alike; a huge one still tells logits of 3e38 apart."""
    print(f"huge temperature {n} {temperature}", flush=True)
    g = torch.Generator().manual_seed(n)
    for scale in (1.0, 3.3e38):
        x = (torch.rand(3, n, generator=g) * 2 - 1) * scale
        for top_k, top_p, min_p in ((0, 0.9, 0.0), (0, 1.0, 0.5), (n // 2, 0.8, 0.0), (0, 1.0, 0.0)):
            for u in (torch.rand(3, generator=g), torch.zeros(3)):
                check_sample(dev, x, u, temperature, top_k, top_p, min_p)


# ----------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,n,shared", [(1, 40, 0), (1, 2000, 0), (3, 2000, 0), (40, 50, 0), (40, 2000, 0), (40, 2000, 1024),
                                             (1, 1100, 1024), (3, 1100, 1024)])
def test_attend_shows_what_is_not_finite(dev, dtype, tokens, n, shared):
    """A query row with a NaN or an infinity, and one whose score at one position is beyond 32 bits, are NaN, in one split
    and in several; a score of -infinity weighs nothing; the other rows are what they were, and a token that sees nothing
    still gives zeros.

    The other rows may be rescaled at other blocks than before: both results hold the tolerance of test_gpu_serving.py, with
    |v| and |k| up to 448 2^-7."""
    print(f"not finite {dtype} tokens {tokens} positions {n} shared {shared}", flush=True)
    batch, heads, hd = (104 if tokens < 40 and shared else 3), 12, 128
    own = -(-n // 64) - shared // 64
    c = make_cache(dev, shared // 64 + batch * own, 4, hd, 64, "fp8_e4m3", "fp8_e4m3", seed=50)
    table = make_table(dev, batch, shared // 64 + own, shared // 64 + batch * own, 51, shared // 64)
    lengths = i32(dev, [n, 0] + [n] * (batch - 2))
    p = (n - tokens) // 2  # the first block of a key that sequence 0 sees: 448 2^118 in dim 7, zeros beside it
    page = int(table[0, p // 64])
    c.k_data[page, :, p % 64, :32] = 0
    c.k_data[page, :, p % 64, 7], c.k_scales[page, :, 0, p % 64] = 0x7E, 245
    q = randn(dev, 52, batch, tokens, heads, hd, dtype=dtype)
    q[..., 7] = 0
    want = c.attend(q, table, lengths, shared=shared)
    assert torch.isfinite(want).all() and not want[1].any()
    q[0, -1, 0, 5], q[0, -1, 1], q[0, -1, 2, 7], q[0, -1, 3, 7] = math.nan, math.inf, 1000.0, -1000.0
    q[1, :, 4] = math.nan  # sees nothing
    got = c.attend(q, table, lengths, shared=shared)
    assert torch.isnan(got[0, -1, :3]).all()
    assert torch.isfinite(got[0, -1, 3:]).all() and torch.isfinite(got[0, :-1]).all() and not got[1].any()
    size = 3.5 * float(q[2:].abs().float().sum(-1).max()) / math.sqrt(hd)
    tol = 2 * 3.5 * (2 * ((hd + 6) * 2.0 ** -24 * size + 2.0 ** -22) + 2.0 ** -17 + 2.0 ** -18) + want.double().abs() * torch.finfo(dtype).eps
    off = (got.double() - want.double()).abs() - tol
    assert float(off[0, -1, 4:].max()) <= 0 and float(off[2:].max()) <= 0
    assert tokens == 1 or float(off[0, :-1].max()) <= 0


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_attend_ignores_what_is_masked_of_a_prefix(dev, tokens):
    """NaN codes and scales in positions of a prefix read in common that lie behind every sequence's end."""
    batch, shared = 104, 1024
    c = make_cache(dev, 16 + batch, 4, 128, 64, "fp8_e4m3", "fp8_e4m3", seed=60)
    table = make_table(dev, batch, 17, 16 + batch, 61, 16)
    q = randn(dev, 62, batch, tokens, 8, 128, dtype=BF16)
    for most in (777, 100, 1):
        lengths = i32(dev, [max(most - 3 * b, 0) for b in range(batch)])
        want = c.attend(q, table, lengths, shared=shared)
        assert torch.isfinite(want).all()
        for p in range(most, shared):
            page = int(table[0, p // 64])
            c.k_data[page, :, p % 64], c.v_data[page, :, p % 64] = 127, 255
            c.k_scales[page, :, :, p % 64] = c.v_scales[page, :, :, p % 64] = 255
        assert torch.equal(c.attend(q, table, lengths, shared=shared), want)


@pytest.mark.parametrize("tokens,n,shared", [(1, 60, 0), (1, 1500, 0), (40, 60, 0), (40, 1500, 0), (1, 1100, 1024), (3, 1100, 1024)])
def test_attend_in_place(dev, tokens, n, shared):
    """out may be q itself: what every workgroup reads of it, it alone writes."""
    batch = 104 if shared else 3
    own = -(-n // 64) - shared // 64
    c = make_cache(dev, shared // 64 + batch * own, 4, 128, 64, "fp8_e4m3", "fp4_e2m1", seed=65)
    table, lengths = make_table(dev, batch, shared // 64 + own, shared // 64 + batch * own, 66, shared // 64), i32(dev, [n] * batch)
    q = randn(dev, 67, batch, tokens, 8, 128, dtype=BF16)
    want = c.attend(q, table, lengths, shared=shared)
    assert c.attend(q, table, lengths, shared=shared, out=q) is q and torch.equal(q, want)


# ----------------------------------------------------------------------------- workspaces
def test_workspaces_are_held_until_the_launch(dev, monkeypatch):
    """Memory that another thread takes on the same stream between a call's allocations and its launch is not the call's
    workspace."""
    c = make_cache(dev, 64, 2, 128, 64, "fp8_e4m3", "fp8_e4m3", seed=70)
    q, table, lengths = randn(dev, 71, 1, 1, 8, 128), make_table(dev, 1, 64, 64, 72), i32(dev, [4000])
    logits, u = randn(dev, 73, 2, 5000), torch.rand(2, device=dev)
    seen = []

    def call(name, *args):
        at, need = args[11], args[12]
        other = torch.empty(need, dtype=torch.uint8, device=dev)
        seen.append((name, need > 0 and (other.data_ptr() >= at + need or other.data_ptr() + need <= at)))

    monkeypatch.setattr(K, "call", call)
    for _ in range(2):
        c.attend(q, table, lengths)
        sample(logits, u)
    assert seen == [("tgm_kv_attend", True), ("tgm_sample", True)] * 2
