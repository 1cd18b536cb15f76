"""The serving operators on gfx950 against their plain 64-bit forms (oracle/serving_oracle.py).

Tolerances.  A rounding to type t is off by at most half a step, eps(t) / 2 of the value (below the normal range: half
the smallest subnormal).  Everything that is computed in 64 bits or exactly is compared with that alone, or bit for bit.
"""

import math

import numpy as np
import pytest
import torch

import serving_oracle as S
from tinygrad_mi355x.kv_cache import PackedKVCache
from tinygrad_mi355x.rotary import Rotary
from tinygrad_mi355x.sampling import sample

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half the smallest subnormal


def half_step(dt: torch.dtype, want: np.ndarray) -> np.ndarray:
    return torch.finfo(dt).eps / 2 * np.abs(want) + TINY[dt]


def np64(t: torch.Tensor) -> np.ndarray:
    return t.double().cpu().numpy()


def i32(dev, values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=dev)


def randn(dev, seed, *shape, dtype=F32, scale=1.0) -> torch.Tensor:
    x = np.random.default_rng(seed).standard_normal(shape) * scale
    return torch.from_numpy(x).to(dtype).to(dev)


def near(got: torch.Tensor, want: np.ndarray, tol: np.ndarray) -> None:
    off = np.abs(np64(got) - want) - tol
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.size} off, by up to {off.max():.3g} over the tolerance"


# ----------------------------------------------------------------------------- rotary positions
def rotation_tolerance(dt, want, x, gain):
    """64-bit sums (their own errors: below 2^-44 of the pair's length up to positions of 2^20), rounded to 32 bits, then
    to dt."""
    size = np.abs(x).max() * abs(gain) * 2
    return half_step(dt, want) + half_step(F32, want) * (1 + torch.finfo(dt).eps) + size * 2.0 ** -44


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_dim,rotary_dim,layout,scaling", [
    (128, None, "half", None), (128, 64, "half", dict(kind="ntk", factor=4.0)), (64, None, "interleaved", None),
    (128, 32, "interleaved", dict(kind="yarn", factor=16.0, trained=8192)), (64, 22, "half", None), (64, 0, "half", None),
    (80, None, "half", dict(kind="linear", factor=4.0)), (96, 34, "interleaved", None), (2, None, "half", None)])
def test_rotate(dev, dtype, head_dim, rotary_dim, layout, scaling):
    print(f"rotate {dtype} {head_dim} {rotary_dim} {layout} {scaling}", flush=True)
    rot = Rotary(head_dim, rotary_dim, layout=layout, scaling=scaling, device=dev)
    for batch, tokens, h, start in ((1, 1, 1, [0]), (3, 5, 7, [0, 131071, 999983]), (2, 33, 40, [4096, 17])):
        x = randn(dev, 1, batch, tokens, h, head_dim, dtype=dtype)
        got = rot.rotate(x, i32(dev, start))
        want = S.rotate(np64(x), start, rot.freq.cpu().numpy(), rot.gain, layout)
        near(got, want, rotation_tolerance(dtype, want, np64(x), rot.gain))
        assert torch.equal(got[..., rot.rotary_dim:], x[..., rot.rotary_dim:])
        assert torch.equal(rot.rotate(x, i32(dev, start), out=x), got)  # in place


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout,rotary_dim", [("half", 128), ("interleaved", 128), ("half", 64)])
def test_rotate_of_views(dev, dtype, layout, rotary_dim):
    """Heads inside stacked q|k|v rows, transposed tokens and heads, and rows that are not 16-byte aligned."""
    rot = Rotary(128, rotary_dim, layout=layout, device=dev)
    start = i32(dev, [3, 700])
    flat = randn(dev, 2, 2 * 9 * 12 * 128 + 1, dtype=dtype)
    stacked = flat[:-1].view(2, 9, 12, 128)
    odd = flat[1:].view(2, 9, 12, 128)
    for x in (stacked[:, :, 2:7], stacked.transpose(1, 2), odd, stacked.flip(0)[:1].expand(2, 9, 12, 128)):
        got = rot.rotate(x, start)
        want = rot.rotate(x.contiguous(), start)
        assert got.is_contiguous() and torch.equal(got, want)


def test_rotate_keeps_what_does_not_rotate(dev):
    """Infinities and NaN beyond rotary_dim do not reach the rotated values, nor the other way round."""
    for layout in ("half", "interleaved"):
        rot = Rotary(64, 32, layout=layout, device=dev)
        x = torch.ones((1, 1, 1, 64), device=dev)
        x[..., 32:] = math.nan
        got = rot.rotate(x, i32(dev, [5]))
        assert torch.isfinite(got[..., :32]).all() and torch.isnan(got[..., 32:]).all()
        got = rot.rotate(x.flip(3).contiguous(), i32(dev, [5]))
        assert torch.isnan(got[..., :32]).all() and (got[..., 32:] == 1).all()


# ----------------------------------------------------------------------------- cache write and read
def make_cache(dev, pages, hk, hd, page, kf, vf, seed=None):
    """A cache; with a seed, filled with random codes and scales (no NaN codes)."""
    c = PackedKVCache(pages, hk, hd, page_size=page, k_format=kf, v_format=vf, device=dev)
    if seed is not None:
        g = np.random.default_rng(seed)
        for data, scales, fmt in ((c.k_data, c.k_scales, kf), (c.v_data, c.v_scales, vf)):
            codes = g.integers(0, 256, tuple(data.shape), dtype=np.uint8)
            if fmt == "fp8_e4m3":
                codes = np.where(codes & 127 == 127, codes & 0x80, codes)
                scale = g.integers(117, 121, tuple(scales.shape))  # values up to 448 * 2^-7
            else:
                scale = g.integers(124, 127, tuple(scales.shape))
            data.copy_(torch.from_numpy(codes))
            scales.copy_(torch.from_numpy(scale.astype(np.uint8)))
    return c


def make_table(dev, batch, cols, pages, seed, shared=0):
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    assert shared + batch * (cols - shared) <= pages
    rows = order[shared:shared + batch * (cols - shared)].reshape(batch, -1)
    return torch.from_numpy(np.concatenate((np.tile(order[:shared], (batch, 1)), rows), 1)).to(dev).contiguous()


def values_of(c):
    return (S.store_values(c.k_data.cpu().numpy(), c.k_scales.cpu().numpy(), c.k_format),
            S.store_values(c.v_data.cpu().numpy(), c.v_scales.cpu().numpy(), c.v_format))


def rows_of(store, table, page):
    """[positions, heads, D] of one table row; positions without a page are None's zeros and marked."""
    ok = (table >= 0) & (table < store.shape[0])
    rows = np.where(ok[:, None, None, None], store[np.where(ok, table, 0)], 0.0)
    return rows.transpose(0, 2, 1, 3).reshape(-1, store.shape[1], store.shape[3]), np.repeat(ok, page)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kf,vf,hd,page", [("fp8_e4m3", "fp8_e4m3", 128, 64), ("fp8_e4m3", "fp4_e2m1", 64, 16),
                                           ("fp4_e2m1", "fp8_e4m3", 128, 128), ("fp4_e2m1", "fp4_e2m1", 64, 32)])
@pytest.mark.parametrize("turn", [None, ("half", None), ("interleaved", 32), ("half", 48)])
def test_append(dev, dtype, kf, vf, hd, page, turn):
    """What is stored is the oracle's code and scale of the (rotated, 32-bit) values, at the token's position and nowhere
    else; what comes back is its value rounded once."""
    print(f"append {dtype} {kf} {vf} {hd} {page} {turn}", flush=True)
    hk, h = 3, 6
    rot = turn and Rotary(hd, turn[1], layout=turn[0], device=dev)
    for batch, tokens, start in ((1, 1, [0]), (2, 37, [page - 1, 5]), (3, 1, [7, page, 2 * page + 1])):
        cols = (max(start) + tokens + page - 1) // page
        c = make_cache(dev, batch * cols + 2, hk, hd, page, kf, vf)
        table = make_table(dev, batch, cols, batch * cols + 2, 3)
        qkv = randn(dev, 4, batch, tokens, h + 2 * hk, hd, dtype=dtype, scale=3.0)
        qkv[0, 0, h, :32] = 0  # a block of zeros
        qkv[0, 0, h + hk, :32] *= 2.0 ** -14
        q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
        for seen in (None, F32, BF16):
            got = c.append(k, v, table, i32(dev, start), rotary=rot, q=q, seen=seen)
        want_k, want_q = np64(k), np64(q)
        if rot:
            freq = rot.freq.cpu().numpy()
            want_k = S.rotate(want_k, start, freq, rot.gain, rot.layout)
            want_q = S.rotate(want_q, start, freq, rot.gain, rot.layout)
            near(got.q, want_q, rotation_tolerance(dtype, want_q, np64(q), rot.gain))
        else:
            assert torch.equal(got.q, q)
        stores = values_of(c)
        table_np = table.cpu().numpy()
        for i, (x, fmt, out) in enumerate(((want_k, kf, got.k), (np64(v), vf, got.v))):
            idx, e = S.quantise(x.astype(np.float32), fmt)
            want = S.value(idx, e, fmt)
            assert torch.equal(out.cpu(), torch.from_numpy(want).to(F32).to(BF16)), "kv"[i]
            scales = (c.k_scales, c.v_scales)[i].cpu().numpy()
            written = np.zeros(stores[i].shape[0::2][:2] + (), bool)
            for b in range(batch):
                for t in range(tokens):
                    p = start[b] + t
                    pg, slot = table_np[b, p // page], p % page
                    assert np.array_equal(stores[i][pg, :, slot], want[b, t])
                    assert np.array_equal(scales[pg, :, :, slot], e[b, t])
                    written[pg, slot] = True
            assert not stores[i].transpose(0, 2, 1, 3)[~written].any()
            assert not scales.transpose(0, 3, 1, 2)[~written].any()


@pytest.mark.parametrize("fmt", ["fp8_e4m3", "fp4_e2m1"])
def test_quantiser_over_the_whole_range(dev, fmt):
    """Ties, saturation, subnormal and huge blocks, NaN and infinities."""
    g = np.random.default_rng(5)
    rows = [np.ldexp(g.standard_normal(32).astype(np.float32), e) for e in range(-160, 120, 7)]
    levels = np.concatenate([S.LEVELS[fmt], (S.LEVELS[fmt][1:] + S.LEVELS[fmt][:-1]) / 2, [S.LEVELS[fmt][-1] * 1.1]])
    for s in (-130, -60, -3, 0, 5, 100):
        v = np.ldexp(levels, s).astype(np.float32)
        v = v[:len(v) // 31 * 31].reshape(-1, 31) if len(v) >= 31 else np.pad(v, (0, 31 - len(v)))[None]
        top = np.full((len(v), 1), np.ldexp(S.LEVELS[fmt][-1], s), np.float32)
        rows += list(np.concatenate((v * (-1) ** np.arange(31), top), 1).astype(np.float32))
    odd = np.ones((4, 32), np.float32)
    odd[0, 3], odd[1, 4], odd[2, 5], odd[3] = np.nan, np.inf, -np.inf, np.nan
    x = np.concatenate((np.array(rows), odd)).astype(np.float32)
    x = np.concatenate((x, np.zeros((-len(x) % 2, 32), np.float32))).reshape(-1, 64)
    n = len(x)
    c = make_cache(dev, -(-n // 64), 1, 64, 64, fmt, fmt)
    table = torch.arange(-(-n // 64), dtype=torch.int32, device=dev)[None]
    k = torch.from_numpy(x).to(dev).view(1, n, 1, 64)
    got = c.append(k, k, table, i32(dev, [0]), seen=F32)
    idx, e = S.quantise(x, fmt)
    want = S.value(idx, e, fmt)
    for out in (got.k, got.v, *c.read(table, i32(dev, [0]), n, F32)):
        assert np.array_equal(np64(out).reshape(n, 64), want.astype(np.float32))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kf,vf,hd,page", [("fp8_e4m3", "fp4_e2m1", 128, 64), ("fp4_e2m1", "fp8_e4m3", 64, 16)])
def test_read(dev, dtype, kf, vf, hd, page):
    hk, batch = 3, 2
    c = make_cache(dev, 20, hk, hd, page, kf, vf, seed=6)
    table = make_table(dev, batch, 9, 20, 7)
    table[1, 4], table[1, 5] = -1, 20  # name no page
    stores = values_of(c)
    for first, count in (([0, 0], 1), ([page - 1, 3 * page + 5], 2 * page + 3), ([8 * page, 8 * page + 7], page + 40),
                         ([-3, 0], 9 * page + 5), ([5, 5], 0)):
        print(f"read {first} {count}", flush=True)
        got = c.read(table, i32(dev, first), count, dtype)
        for out, store in zip(got, stores):
            assert out.shape == (batch, count, hk, hd)
            for b in range(batch):
                rows, _ = rows_of(store, table[b].cpu().numpy(), page)
                want = np.zeros((count, hk, hd))
                for i in range(count):
                    if 0 <= first[b] + i < len(rows):
                        want[i] = rows[first[b] + i]
                assert torch.equal(out[b].cpu(), torch.from_numpy(want).to(dtype))


def test_append_drops_positions_without_a_page(dev):
    c = make_cache(dev, 4, 2, 64, 16, "fp8_e4m3", "fp8_e4m3")
    table = i32(dev, [[-1, 2, 4]])
    k = randn(dev, 8, 1, 60, 2, 64)
    for start in (0, -7, 40):
        got = c.append(k, k, table, i32(dev, [start]), seen=F32)
        idx, e = S.quantise(np64(k).astype(np.float32), "fp8_e4m3")
        assert np.array_equal(np64(got.k), S.value(idx, e, "fp8_e4m3"))  # given back all the same
        assert not c.k_scales[[0, 1, 3]].any() and not c.v_data[[0, 1, 3]].any()
    back = c.read(table, i32(dev, [0]), 48, F32)[0]
    assert not back[:, :16].any() and not back[:, 32:].any() and back[:, 16:32].any()


# ----------------------------------------------------------------------------- attention
def attention_tolerance(dt, hd, want, size, vmax):
    """Scores: products are exact (f32 queries: what three bf16 terms leave of q, 2^-26 of it), their fp32 sums off by
    hd 2^-24 of the sum of magnitudes `size`, the exponent's argument by two more roundings of it and of the maximum (at
    most size each), so a weight by d = (hd + 6) 2^-24 size and one unit of exp2; weights enter the sums in terms that
    leave 2^-17 of them (f32: 2^-25); sums over blocks of 64 rescale and add in fp32, under 2^-18 of the weights' sum
    for the lengths here.  Numerator and denominator each."""
    d = (hd + 6) * 2.0 ** -24 * size + 2.0 ** -22
    term = 2.0 ** -25 if dt is F32 else 2.0 ** -17
    return vmax * (2 * d + term + 2.0 ** -18)[..., None] + half_step(dt, want)


def check_attend(dev, c, q, table, lengths, shared=0, scale=None, out=None):
    got = c.attend(q, table, lengths, shared=shared, scale=scale, out=out)
    assert got.shape == q.shape and got.dtype is q.dtype
    ks, vs = values_of(c)
    batch, tokens, _, hd = q.shape
    k, v, seen = [], [], []
    for b in range(batch):
        row = table[b].cpu().numpy().copy()
        row[:shared // c.page_size] = table[0, :shared // c.page_size].cpu().numpy()
        kb, ok = rows_of(ks, row, c.page_size)
        vb, _ = rows_of(vs, row, c.page_size)
        last = int(lengths[b]) - tokens + np.arange(tokens)
        k.append(kb), v.append(vb)
        seen.append(ok[None] & (np.arange(len(kb))[None] <= last[:, None]))
    want, size = S.attend(np64(q), k, v, seen, 1 / math.sqrt(hd) if scale is None else scale)
    vmax = max((np.abs(x[s.any(0)]).max(initial=0.0) for x, s in zip(v, seen)), default=0.0)
    near(got, want, attention_tolerance(q.dtype, hd, want, size, vmax))
    none = np.array([~s.any(1) for s in seen])
    assert not np64(got)[none].any()
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,hd,page,kf,vf", [
    (2, 4, 128, 64, "fp8_e4m3", "fp8_e4m3"), (1, 8, 64, 16, "fp8_e4m3", "fp4_e2m1"), (2, 7, 128, 16, "fp4_e2m1", "fp8_e4m3"),
    (3, 1, 64, 128, "fp4_e2m1", "fp4_e2m1"), (1, 2, 128, 32, "fp8_e4m3", "fp4_e2m1"), (1, 5, 128, 128, "fp4_e2m1", "fp4_e2m1")])
@pytest.mark.parametrize("tokens", [1, 2, 5, 33])
def test_attend(dev, dtype, hk, group, hd, page, kf, vf, tokens):
    """Decode and chunks: lengths of none and one, fewer than the tokens, ends inside tiles and pages, one split and
    several."""
    print(f"attend {dtype} {hk}x{group} {hd} page {page} {kf} {vf} tokens {tokens}", flush=True)
    lengths = [0, 1, tokens, 63, 64, 65 + tokens, 700]
    batch = len(lengths)
    cols = -(-704 // page)
    c = make_cache(dev, batch * cols + 3, hk, hd, page, kf, vf, seed=9)
    table = make_table(dev, batch, cols, batch * cols + 3, 10)
    q = randn(dev, 11, batch, tokens, hk * group, hd, dtype=dtype, scale=1.5)
    check_attend(dev, c, q, table, i32(dev, lengths))
    short = -(-64 // page)  # a table of one chunk: no join
    check_attend(dev, c, q, table[:, :short].contiguous(), i32(dev, [min(n, 64) for n in lengths]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 40])
def test_attend_over_many_splits(dev, dtype, tokens):
    c = make_cache(dev, 160, 1, 128, 64, "fp8_e4m3", "fp8_e4m3", seed=12)
    table = make_table(dev, 1, 150, 160, 13)
    q = randn(dev, 14, 1, tokens, 4, 128, dtype=dtype, scale=1.5)
    for n in (9000, 9600, 4097):
        check_attend(dev, c, q, table, i32(dev, [n]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,tokens,shared,hk,group", [(3, 1, 64, 2, 4), (5, 2, 640, 1, 7), (40, 1, 320, 1, 4), (2, 9, 192, 2, 2),
                                                             (52, 2, 1024, 4, 4), (100, 1, 1024, 4, 2),
                                                             (100, 3, 1024, 4, 2)])
def test_attend_shared_prefix(dev, dtype, batch, tokens, shared, hk, group):
    """The prefix once for all gives what each sequence's own attention gives; some sequences end inside it.  The last
    three are large enough to be read in common by few rows each (the last two for f32 too), in one launch with the
    sequences' own positions (up to 8 rows, f32 5) and in one of its own."""
    print(f"shared {dtype} {batch} {tokens} {shared} {hk}x{group}", flush=True)
    page, hd = 64, 128
    cols = shared // page + 3
    c = make_cache(dev, shared // page + batch * 3 + 1, hk, hd, page, "fp8_e4m3", "fp4_e2m1", seed=15)
    table = make_table(dev, batch, cols, shared // page + batch * 3 + 1, 16, shared // page)
    lengths = [shared + 1 + (37 * b) % (3 * page) for b in range(batch)]
    lengths[0], lengths[1] = shared - 5, shared
    q = randn(dev, 17, batch, tokens, hk * group, hd, dtype=dtype, scale=1.5)
    n = i32(dev, lengths)
    got = check_attend(dev, c, q, table, n, shared=shared)
    rows = table.clone()
    rows[1:, :shared // page] = -1  # only row 0's are read
    assert torch.equal(c.attend(q, rows, n, shared=shared), got)
    all_of_it = table[:, :shared // page].contiguous()
    check_attend(dev, c, q, all_of_it, n.clamp(max=shared), shared=shared)


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_attend_ignores_what_is_masked(dev, tokens):
    """NaN codes and scales in positions behind the last, in pages that no table names, and page numbers that name none;
    lengths beyond the table."""
    c = make_cache(dev, 24, 2, 64, 16, "fp8_e4m3", "fp8_e4m3", seed=18)
    table = make_table(dev, 2, 10, 24, 19)
    q = randn(dev, 20, 2, tokens, 8, 64, dtype=BF16)
    lengths = i32(dev, [73, 150])
    want = check_attend(dev, c, q, table, lengths)
    named = table[0, :5].tolist() + table[1].tolist()
    for p in set(range(24)) - set(named):
        c.k_data[p], c.v_data[p], c.k_scales[p], c.v_scales[p] = 127, 127, 255, 255
    for b, n in ((0, 73), (1, 150)):
        p = int(table[b, n // 16])
        for t, fill in ((c.k_data, 127), (c.v_data, 255)):
            t[p, :, n % 16:] = fill
        c.k_scales[p, :, :, n % 16:] = c.v_scales[p, :, :, n % 16:] = 255
    assert torch.equal(c.attend(q, table, lengths), want)
    table[0, 5:] = torch.tensor([-1, 24, 2 ** 31 - 1, -2 ** 31, 10 ** 6], device=dev)
    assert torch.equal(c.attend(q, table, lengths), want)
    c2 = make_cache(dev, 24, 2, 64, 16, "fp8_e4m3", "fp8_e4m3", seed=18)
    table[1, 2], table[1, 6] = -1, 99  # holes among the positions that are seen
    check_attend(dev, c2, q, table, i32(dev, [73, 150]))
    check_attend(dev, c2, q, table, i32(dev, [-4, 2 ** 31 - 1]).clamp(max=160 + tokens))
    got = c2.attend(q, table, i32(dev, [2 ** 31 - 1, -2 ** 31]))
    assert torch.isfinite(got).all() and not got[1].any()


def test_attend_views_scale_and_out(dev):
    c = make_cache(dev, 12, 2, 128, 64, "fp8_e4m3", "fp8_e4m3", seed=21)
    table, lengths = make_table(dev, 2, 5, 12, 22), i32(dev, [300, 129])
    wide = make_table(dev, 2, 6, 12, 22)
    flat = randn(dev, 23, 2 * 3 * 12 * 128 + 1, dtype=BF16)
    for tokens in (1, 3):
        for x in (flat[:-1].view(2, 3, 12, 128)[:, :tokens, :8], flat[1:].view(2, 3, 12, 128)[:, :tokens, 4:]):
            out = torch.empty((2, tokens, 8, 128), dtype=BF16, device=dev)
            got = check_attend(dev, c, x, table, lengths, scale=0.2, out=out)
            assert got is out and torch.equal(got, c.attend(x.contiguous(), table, lengths, scale=0.2))
    q = flat[:2 * 8 * 128].view(2, 1, 8, 128)
    assert torch.equal(c.attend(q, wide[:, :5], lengths), c.attend(q, wide[:, :5].contiguous(), lengths))


def test_empty_calls(dev):
    c, rot = make_cache(dev, 4, 2, 64, 64, "fp8_e4m3", "fp8_e4m3", seed=1), Rotary(64, device=dev)
    none, table = i32(dev, []), torch.zeros((0, 2), dtype=torch.int32, device=dev)
    x, y = torch.zeros((0, 3, 2, 64), device=dev), torch.zeros((2, 0, 2, 64), device=dev)
    start, rows = i32(dev, [0, 0]), i32(dev, [[0, 1], [2, 3]])
    assert rot.rotate(x, none).shape == x.shape and rot.rotate(y, start).shape == y.shape
    assert c.append(x, x, table, none, rotary=rot, q=x, seen=F32).k.shape == x.shape
    assert c.append(y, y, rows, start, rotary=rot, q=y, seen=F32).q.shape == y.shape
    assert c.attend(x, table, none).shape == x.shape and c.attend(y, rows, start).shape == y.shape
    assert c.read(table, none, 5)[0].shape == (0, 5, 2, 64)
    assert sample(torch.zeros((0, 9), device=dev), torch.zeros(0, device=dev)).shape == (0,)


def test_large_scores_and_flat_ones(dev):
    """One position takes all the weight; and all weigh the same."""
    for factor in (60.0, 0.0):
        c = make_cache(dev, 6, 1, 64, 64, "fp8_e4m3", "fp8_e4m3", seed=24)
        table = make_table(dev, 1, 6, 6, 25)
        for tokens in (1, 20):
            q = randn(dev, 26, 1, tokens, 4, 64) * factor
            check_attend(dev, c, q, table, i32(dev, [350]))


def test_offsets_past_32_bits(dev):
    """Pages whose codes and scales lie beyond 2^31 and 2^32 bytes."""
    pages = 70000  # of 64 positions, 8 heads, 128 bytes: 4.6e9 bytes of keys
    c = PackedKVCache(pages, 8, 128, page_size=64, k_format="fp8_e4m3", v_format="fp4_e2m1", device=dev)
    table = i32(dev, [[pages - 1, 33000, 1], [pages - 2, 65600, 2]])
    k, v = randn(dev, 27, 2, 150, 8, 128), randn(dev, 28, 2, 150, 8, 128)
    got = c.append(k, v, table, i32(dev, [0, 0]), seen=F32)
    back = c.read(table, i32(dev, [0, 0]), 150, F32)
    assert torch.equal(back[0], got.k) and torch.equal(back[1], got.v)
    small = PackedKVCache(6, 8, 128, page_size=64, k_format="fp8_e4m3", v_format="fp4_e2m1", device=dev)
    near_table = i32(dev, [[0, 1, 2], [3, 4, 5]])
    small.append(k, v, near_table, i32(dev, [0, 0]))
    for tokens in (1, 30):
        q = randn(dev, 29, 2, tokens, 16, 128, dtype=BF16)
        n = i32(dev, [150, 97])
        assert torch.equal(c.attend(q, table, n), small.attend(q, near_table, n))


# ----------------------------------------------------------------------------- sampling
def check_sample(dev, logits, u, temperature, top_k, top_p, min_p):
    rows = logits.shape[0]
    full = lambda v, dt: torch.full((rows,), v, dtype=dt) if not isinstance(v, torch.Tensor) else v  # noqa: E731
    t, k, p, m = full(temperature, F32), full(top_k, torch.int32), full(top_p, F32), full(min_p, F32)
    got = sample(logits.to(dev), u.to(dev), temperature=t.to(dev), top_k=k.to(dev), top_p=p.to(dev), min_p=m.to(dev))
    want = S.sample(np64(logits), u.numpy(), t.numpy(), k.numpy(), p.double().numpy(), m.double().numpy())
    assert got.dtype is torch.int32 and got.cpu().numpy().tolist() == want.tolist()
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(5, 1), (7, 2), (4, 63), (3, 1000), (2, 32000), (2, 50257), (1, 131072)])
def test_sample(dev, dtype, rows, n):
    g = torch.Generator().manual_seed(n)
    logits = (torch.randn(rows, n, generator=g) * 3).to(dtype)
    for temperature, top_k, top_p, min_p in ((1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (0.7, 50, 0.9, 0.02), (1.5, 0, 0.95, 0.0),
                                             (0.3, 400, 1.0, 0.0), (1.0, 1, 0.9, 0.0), (1.0, 0, 1.0, 0.1), (1.3, 7, 0.0, 0.0),
                                             (2.0, n, 0.5, 1.0)):
        print(f"sample {dtype} {rows}x{n} {temperature} {top_k} {top_p} {min_p}", flush=True)
        check_sample(dev, logits, torch.rand(rows, generator=g), temperature, top_k, top_p, min_p)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_ties_and_edges(dev, dtype):
    """Cuts that fall among equal logits; -inf, NaN, zeros of both signs; the ends of u."""
    g = torch.Generator().manual_seed(1)
    n = 3001
    x = torch.randint(-3, 4, (6, n), generator=g).to(dtype)
    x[1] = 2.5
    x[2, ::2] = -math.inf
    x[3, 5:] = -math.inf
    x[4] = torch.where(torch.rand(n, generator=g) < 0.5, 0.0, -0.0)
    x[5, 7:900] = math.nan
    for u in (torch.zeros(6), torch.full((6,), 1 - 2.0 ** -24), torch.rand(6, generator=g), torch.rand(6, generator=g)):
        for temperature, top_k, top_p, min_p in ((1.0, 0, 1.0, 0.0), (1.0, 700, 1.0, 0.0), (0.5, 0, 0.37, 0.0),
                                                 (1.0, 431, 0.61, 0.0), (1.0, 431, 0.61, 0.2), (0.0, 0, 1.0, 0.0)):
            check_sample(dev, x, u, temperature, top_k, top_p, min_p)


def test_sample_rows_of_their_own(dev):
    """Every row its own parameters, rows inside wider ones, no token at all, an infinite logit, sharp distributions."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(8, 5003, generator=g) * 4
    logits = wide[:, 1:4999]
    logits[6] = -math.inf
    logits[7, 1234] = math.inf
    u = torch.rand(8, generator=g)
    t = torch.tensor([1.0, 0.0, 0.01, 100.0, 1e-6, 1.0, 1.0, 1.0])
    k = torch.tensor([0, 3, 9, 100, 0, 2, 1, 5], dtype=torch.int32)
    p = torch.tensor([0.3, 1.0, 0.9, 0.8, 0.99, 1.0, 0.5, 1.0])
    m = torch.tensor([0.0, 0.1, 0.0, 0.9, 0.0, 0.5, 0.0, 0.0])
    check_sample(dev, logits, u, t, k, p, m)
    on = wide.to(dev)[:, 1:4999]
    want = sample(on.contiguous(), u.to(dev), temperature=t.to(dev), top_k=k.to(dev), top_p=p.to(dev), min_p=m.to(dev))
    got = sample(on, u.to(dev), temperature=t.to(dev), top_k=k.to(dev), top_p=p.to(dev), min_p=m.to(dev))
    assert torch.equal(got, want)
    plain = sample(on, u.to(dev), temperature=0.5)
    assert torch.equal(plain, sample(on, u.to(dev), temperature=torch.full((8,), 0.5, device=dev), top_p=1.0, top_k=0, min_p=0.0))


def test_sample_draws_with_the_right_frequencies(dev):
    n, draws = 50, 20000
    row = torch.randn(n, generator=torch.Generator().manual_seed(3))
    u = (torch.arange(draws) + 0.5) / draws
    got = sample(row.expand(draws, n).contiguous().to(dev), u.to(dev))
    freq = np.bincount(got.cpu().numpy(), minlength=n) / draws
    want = torch.softmax(row.double(), 0).numpy()
    assert np.abs(freq - want).max() <= 1.0 / draws + 1e-6  # evenly spaced u: each interval holds its share to one draw


def test_sample_long_lists_and_many_rows(dev):
    """Lists of every length class, cuts among more equal logits than a list holds, u = 0, and more rows than a slab."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 40000, generator=g)
    x[1] = torch.randint(0, 5, (40000,), generator=g).float()
    x[2] = 1.0
    for k, p in ((300, 1.0), (600, 0.9), (1500, 0.99), (2048, 1.0), (5000, 0.97), (0, 0.02), (0, 0.1), (0, 0.6), (39999, 0.5)):
        print(f"sample lists {k} {p}", flush=True)
        for u in (torch.rand(3, generator=g), torch.zeros(3)):
            check_sample(dev, x, u, 1.0, k, p, 0.0)
    rows = 2048 * 2 + 77
    logits = torch.randn(rows, 130, generator=g)
    check_sample(dev, logits, torch.rand(rows, generator=g), 0.8, 20, 0.9, 0.01)


def test_a_whole_vocabulary_of_2_to_the_20(dev):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 1 << 20, generator=g) * 2
    for dtype in (F32, BF16):
        for k, p, t in ((0, 0.9, 1.0), (50, 0.95, 0.7), (0, 1.0, 1.0), (4000, 1.0, 1.0)):
            check_sample(dev, x.to(dtype), torch.rand(2, generator=g), t, k, p, 0.0)


# ----------------------------------------------------------------------------- streams and graphs
def test_operators_on_a_side_stream_and_in_a_graph(dev):
    c = make_cache(dev, 12, 2, 128, 64, "fp8_e4m3", "fp8_e4m3", seed=30)
    rot, table = Rotary(128, device=dev), make_table(dev, 2, 6, 12, 31)
    qkv = randn(dev, 32, 2, 1, 12, 128, dtype=BF16)
    start, lengths = i32(dev, [300, 120]), i32(dev, [301, 121])
    logits, u = randn(dev, 33, 2, 5000), torch.rand(2, device=dev)

    def step():
        a = c.append(qkv[:, :, 8:10], qkv[:, :, 10:], table, start, rotary=rot, q=qkv[:, :, :8], seen=BF16)
        o = c.attend(a.q, table, lengths)
        s = c.attend(a.q, table, lengths, shared=64)
        return a.q, a.k, a.v, o, s, *c.read(table, start, 1), sample(logits, u, temperature=0.9, top_p=0.9)

    want = [x.clone() for x in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        qkv.copy_(randn(dev, 40 + i, 2, 1, 12, 128, dtype=BF16))
        start.add_(1)
        lengths.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(step(), replayed)), f"replay {i}"
        torch.cuda.synchronize()
