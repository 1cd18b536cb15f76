"""Refusals of the serving operators, and the host's own arithmetic: no GPU needed."""

import ctypes
import math
import struct

import numpy as np
import pytest
import torch

import serving_oracle as S
from tinygrad_mi355x.kv_cache import PackedKVCache
from tinygrad_mi355x.rotary import Rotary, frequencies
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.sampling import sample

I32 = torch.int32


def cache(**kw):
    return PackedKVCache(kw.pop("pages", 4), kw.pop("kv_heads", 2), kw.pop("head_dim", 64), device="cpu", **kw)


# ----------------------------------------------------------------------------- construction
@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(page_size=2048),
                                dict(pages=0), dict(kv_heads=0), dict(k_format="fp8_e5m2"), dict(v_format="int4")])
def test_cache_refuses(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_cache_stores_have_the_stated_shapes():
    c = cache(page_size=16, k_format="fp8_e4m3", v_format="fp4_e2m1")
    assert c.k_data.shape == (4, 2, 16, 64) and c.v_data.shape == (4, 2, 16, 32)
    assert c.k_scales.shape == c.v_scales.shape == (4, 2, 2, 16)
    assert c.nbytes() == 4 * 2 * 16 * (64 + 32 + 4)


@pytest.mark.parametrize("args,kw", [((64, 66), {}), ((64, 7), {}), ((0,), {}), ((64,), dict(layout="pairs")),
                                     ((64,), dict(base=1.0)), ((64,), dict(scaling=dict(kind="dynamic", factor=2.0))),
                                     ((64,), dict(scaling=dict(kind="linear", factor=0.5))),
                                     ((64,), dict(scaling=dict(kind="yarn", factor=2.0))),
                                     ((64, 2), dict(scaling=dict(kind="ntk", factor=2.0))),
                                     ((64,), dict(scaling=dict(kind="linear", factor=2.0, ramp=3)))])
def test_rotary_refuses(args, kw):
    with pytest.raises(ValueError):
        Rotary(*args, device="cpu", **kw)


def test_frequencies_of_each_scaling():
    n, base = 64, 10000.0
    plain, gain = frequencies(n, base)
    assert gain == 1.0 and np.allclose(plain, base ** (-np.arange(32) / 32), rtol=1e-15)
    assert torch.equal(frequencies(n, base, dict(kind="linear", factor=4.0))[0], plain / 4)
    ntk = frequencies(n, base, dict(kind="ntk", factor=4.0))[0]
    assert ntk[0] == plain[0] and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    yarn, gain = frequencies(n, base, dict(kind="yarn", factor=16.0, trained=8192))
    turns = plain * 8192 / (2 * math.pi)
    assert math.isclose(gain, 0.1 * math.log(16) + 1)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    assert np.allclose(yarn[turns < 0.7], plain[turns < 0.7] / 16, rtol=1e-15)
    assert bool(((yarn <= plain) & (yarn >= plain / 16 * (1 - 1e-15))).all())


# ----------------------------------------------------------------------------- refusals of calls
def heads(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_operators_have_no_cpu_implementation():
    c, r = cache(), Rotary(64, device="cpu")
    x, start, table = heads(1, 1, 2, 64), torch.zeros(1, dtype=I32), torch.zeros((1, 2), dtype=I32)
    for call in (lambda: r.rotate(x, start), lambda: c.append(x, x, table, start), lambda: c.read(table, start, 1),
                 lambda: c.attend(x, table, start), lambda: sample(torch.zeros(1, 8), torch.zeros(1))):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


@pytest.mark.parametrize("x,start", [
    (heads(1, 2, 64), torch.zeros(1, dtype=I32)), (heads(1, 1, 2, 64, dtype=torch.float64), torch.zeros(1, dtype=I32)),
    (heads(1, 1, 2, 128), torch.zeros(1, dtype=I32)), (heads(1, 1, 2, 64), torch.zeros(2, dtype=I32)),
    (heads(1, 1, 2, 64), torch.zeros(1, dtype=torch.int64)), (heads(1, 1, 64, 2).transpose(2, 3), torch.zeros(1, dtype=I32))])
def test_rotate_refuses(x, start):
    with pytest.raises(ValueError):
        Rotary(64, device="cpu").rotate(x, start)


def test_append_refuses():
    c, x, start, table = cache(), heads(1, 3, 2, 64), torch.zeros(1, dtype=I32), torch.zeros((1, 2), dtype=I32)
    for args, kw in [((x, heads(1, 2, 2, 64), table, start), {}), ((heads(1, 3, 4, 64), heads(1, 3, 4, 64), table, start), {}),
                     ((x, x.half(), table, start), {}), ((x, x, table.long(), start), {}),
                     ((x, x, torch.zeros((2, 2), dtype=I32), start), {}), ((x, x, table, torch.zeros(2, dtype=I32)), {}),
                     ((x, x, table, start), dict(q=heads(1, 2, 2, 64))), ((x, x, table, start), dict(q=x.half())),
                     ((x, x, table, start), dict(seen=torch.float64)),
                     ((x, x, table, start), dict(rotary=Rotary(128, device="cpu")))]:
        with pytest.raises(ValueError):
            c.append(*args, **kw)


def test_read_and_attend_refuse():
    c, q, n, table = cache(), heads(1, 1, 4, 64), torch.zeros(1, dtype=I32), torch.zeros((1, 2), dtype=I32)
    for args in [(table[0], n, 1), (table, n.long(), 1), (table, n, -1), (table, n, 1, torch.float64)]:
        with pytest.raises(ValueError):
            c.read(*args)
    for args, kw in [((heads(1, 1, 3, 64), table, n), {}), ((heads(1, 1, 4, 128), table, n), {}), ((q, table.long(), n), {}),
                     ((q, table, torch.zeros(2, dtype=I32)), {}), ((q, table, n), dict(shared=32)),
                     ((q, table, n), dict(shared=192)), ((q, table, n), dict(shared=-64)), ((q, table, n), dict(scale=0.0)),
                     ((q, table, n), dict(scale=math.nan)), ((q, table, n), dict(out=q.half()))]:
        with pytest.raises(ValueError):
            c.attend(*args, **kw)


def test_sample_refuses():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for args, kw in [((x[0], u), {}), ((x.double(), u), {}), ((x, u[:1]), {}), ((x, u.double()), {}),
                     ((x.T.contiguous().T, u), {}), ((torch.zeros(2, 0), u), {}), ((x, u), dict(temperature=torch.zeros(3))),
                     ((x, u), dict(top_k=torch.zeros(2))), ((x, u), dict(top_p=torch.zeros(2, 1))),
                     ((x, u), dict(min_p=torch.zeros(2, dtype=torch.float64))), ((x, u), dict(out=torch.zeros(2)))]:
        with pytest.raises(ValueError):
            sample(*args, **kw)


# ----------------------------------------------------------------------------- the C entries
class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("kd", "ks", "vd", "vs")] + [
        (n, ctypes.c_int64) for n in ("pages", "kv_heads", "head_dim", "page_size", "k_format", "v_format")]


def c_cache(**kw):
    f = dict(kd=256, ks=512, vd=768, vs=1024, pages=4, kv_heads=2, head_dim=64, page_size=64, k_format=0, v_format=1)
    f.update(kw)
    return bytes(Cache(**f))


def c_heads(h=2, dtype=13):
    return struct.pack("qqqqq", h * 64, h * 64, 64, h, dtype)


@pytest.mark.parametrize("kw", [dict(kd=None), dict(kd=8), dict(pages=0), dict(kv_heads=0), dict(head_dim=80),
                                dict(page_size=63), dict(page_size=8), dict(k_format=2), dict(v_format=-1)])
def test_c_entries_refuse_a_bad_cache(kw):
    """Every refusal comes before a launch: the addresses are never read."""
    x = c_heads()
    with pytest.raises(ValueError):
        K.call("tgm_kv_append", c_cache(**kw), None, None, None, None, None, x, 4096, x, 4096, None, None, None, 4096, 2, 2,
               4096, 1, 1, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_read", c_cache(**kw), 4096, 2, 2, 4096, 1, 1, 4096, 4096, 13, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_attend", c_cache(**kw), x, 4096, 4096, 2, 2, 4096, 1, 1, 0, 1.0, 4096, 1 << 30, 4096, None)


def test_c_entries_refuse_bad_calls():
    c, x = c_cache(), c_heads()
    attend = dict(q=x, data=4096, table=4096, ld=2, cols=2, lengths=4096, batch=1, tokens=1, shared=0, scale=1.0, ws=4096, wsb=1 << 30,
                  out=4096)
    for bad in (dict(q=None), dict(data=None), dict(q=c_heads(3)), dict(q=c_heads(dtype=14)), dict(table=None), dict(ld=1), dict(cols=1 << 40),
                dict(lengths=None), dict(batch=-1), dict(tokens=-1), dict(shared=32), dict(shared=192), dict(scale=0.0),
                dict(scale=math.nan), dict(out=None), dict(out=8), dict(cols=8, ld=8, wsb=16), dict(cols=8, ld=8, ws=None)):
        with pytest.raises(ValueError):
            K.call("tgm_kv_attend", c, *{**attend, **bad}.values(), None)
    rot = struct.pack("Pdqq", 4096, 1.0, 64, 0)
    for r, a, b, start, batch in [(None, x, x, 4096, 1), (struct.pack("Pdqq", 4096, 1.0, 66, 0), x, x, 4096, 1),
                                  (struct.pack("Pdqq", 4096, 1.0, 63, 0), x, x, 4096, 1),
                                  (struct.pack("Pdqq", 0, 1.0, 64, 0), x, x, 4096, 1),
                                  (struct.pack("Pdqq", 4096, 1.0, 64, 2), x, x, 4096, 1), (rot, x, c_heads(3), 4096, 1),
                                  (rot, x, c_heads(dtype=12), 4096, 1), (rot, x, x, None, 1), (rot, x, x, 4096, -1)]:
        with pytest.raises(ValueError):
            K.call("tgm_rotate", r, a, 4096, b, 4096, start, batch, 1, 64, None)
    with pytest.raises(ValueError):
        K.call("tgm_rotate", rot, x, None, x, 4096, 4096, 1, 1, 64, None)
    for args in [(4096, 14, 1, 8, 8), (4096, 13, -1, 8, 8), (4096, 13, 1, 0, 8), (4096, 13, 1, (1 << 20) + 1, 1 << 21),
                 (4096, 13, 2, 8, 7), (None, 13, 1, 8, 8)]:
        with pytest.raises(ValueError):
            K.call("tgm_sample", *args, 4096, 4096, None, None, None, 4096, 4096, 1 << 30, None)


def test_nothing_to_do_is_no_error():
    K.call("tgm_kv_attend", c_cache(), c_heads(), None, 4096, 2, 2, None, 0, 1, 0, 1.0, None, 0, None, None)
    K.call("tgm_kv_read", c_cache(), 4096, 2, 2, None, 1, 0, None, None, 13, None)
    K.call("tgm_sample", None, 13, 0, 8, 8, None, None, None, None, None, None, None, 0, None)


# ----------------------------------------------------------------------------- the oracle itself
def test_oracle_quantiser_follows_the_formats():
    x = np.array([0.0, 448.0, 17.0, -18.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9] + [0.0] * 25, np.float32)[None]
    idx, e = S.quantise(x, "fp8_e4m3")
    assert e[0, 0] == 127
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(S.value(idx, e, "fp8_e4m3"), want)
    x4 = np.array([6.0, 5.0, 2.5, 0.25, 0.75, -3.5, 7.9] + [0.0] * 25, np.float32)[None]
    idx, e = S.quantise(x4, "fp4_e2m1")
    assert S.value(idx, e, "fp4_e2m1")[0, :7].tolist() == [6.0, 4.0, 2.0, 0.0, 1.0, -4.0, 6.0]
