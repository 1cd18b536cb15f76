"""Refusals of the serving operators at the ends of their arguments: no GPU needed."""

import itertools
import random

import pytest
import torch

from test_serving_host import c_cache, c_heads
from tinygrad_mi355x.kv_cache import PackedKVCache
from tinygrad_mi355x.rotary import Rotary
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.runtime.overlap import overlap, overlaps_itself


@pytest.mark.parametrize("batch,tokens,cols", [(1 << 32, 1 << 32, 2), (4, 1 << 62, 2), (1 << 62, 4, 2), (1, 1, 1 << 58)])
def test_sizes_whose_products_pass_64_bits(batch, tokens, cols):
    """They are refused before anything is computed from the products, which wrap to 0."""
    c, x = c_cache(), c_heads()
    with pytest.raises(ValueError):
        K.call("tgm_kv_append", c, None, None, None, None, None, x, 4096, x, 4096, None, None, None, 4096, cols, cols,
               4096, batch, tokens, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_attend", c, x, 4096, 4096, cols, cols, 4096, batch, tokens, 0, 1.0, 4096, 1 << 30, 4096, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_read", c, 4096, cols, cols, 4096, batch, tokens, 4096, 4096, 13, None)
    assert K.load_library().tgm_kv_attend_workspace(c, 13, 2, batch, tokens, cols, 0) == 0


# ----------------------------------------------------------------------------- memory that tensors share
def elements(t):
    """First byte of every element."""
    size = t.element_size()
    return [t.data_ptr() + size * sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))]


def test_overlap_of_strided_tensors():
    """Against the set of all bytes, over random shapes, strides and offsets."""
    rng = random.Random(0)
    store = torch.empty(1200)
    both = [[0, 0], [0, 0]]
    for _ in range(4000):
        two = []
        for _ in range(2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 4))]
            strides = [rng.choice([0, 1, 1, 2, 3, 4, 5, 8, 12, 16, 17, 24, 48]) for _ in shape]
            two.append(torch.as_strided(store, shape, strides, rng.randint(0, 200)))
        at = [elements(t) for t in two]
        want = [len(set(at[0])) < len(at[0]), bool(set(at[0]) & set(at[1]))]
        got = [overlaps_itself(two[0]), overlap(*two)]
        assert got == want, [(t.shape, t.stride(), t.storage_offset()) for t in two]
        for i in range(2):
            both[i][want[i]] += 1
    assert min(map(min, both)) > 200


def test_overlap_of_heads_in_stacked_rows():
    rows = torch.empty((2, 8192, 48, 128), dtype=torch.bfloat16)
    q, k, v = rows.split((32, 8, 8), 2)
    assert not overlaps_itself(q) and not overlap(q, k) and not overlap(k, v)
    assert overlap(q, rows) and overlap(rows[:, 1:], rows[:, :-1])
    assert not overlap(rows[:, 0::2], rows[:, 1::2]) and overlap(rows[..., 1:], rows[..., :-1])
    assert not overlap(rows.transpose(1, 2)[:, 32:], q) and overlap(rows.transpose(1, 2)[:, 31:], q)
    assert overlaps_itself(q[:, :, :1].expand_as(q)) and not overlap(q[:, :0], q)


def test_rotate_refuses_an_output_that_overlaps(monkeypatch):
    """Checked before the launch, which is replaced here: the elements are written in no order."""
    calls = []
    monkeypatch.setattr(K, "require_device", lambda t: None)
    monkeypatch.setattr(K, "stream_on", lambda i: 0)
    monkeypatch.setattr(K, "call", lambda name, *args: calls.append(name))
    r, start = Rotary(64, device="cpu"), torch.zeros(2, dtype=torch.int32)
    flat = torch.zeros(2 * 6 * 8 * 64 + 32)
    rows = flat[:-32].view(2, 6, 8, 64)
    x = rows[:, 2:4, 1:3]
    for out in (x, rows[:, 2:4, 3:5], rows[:, 4:, 1:3], torch.zeros_like(x), x.clone().transpose(1, 2).contiguous().transpose(1, 2)):
        assert r.rotate(x, start, out=out) is out
    assert len(calls) == 5
    for out in (rows[:, 2:3, 1:3].expand_as(x), rows[:, :2, :1].expand(2, 2, 2, 64), rows[:, 3:5, 1:3], rows[:, 2:4, 2:4],
                flat[32:].view(2, 6, 8, 64)[:, 2:4, 1:3], x.transpose(1, 2)):
        with pytest.raises(ValueError):
            r.rotate(x, start, out=out)
    with pytest.raises(ValueError):
        r.rotate(x[:, :, :1].expand_as(x), start, out=x[:, :, :1].expand_as(x))
    assert len(calls) == 5


def test_attend_refuses_an_output_that_overlaps(monkeypatch):
    calls = []
    monkeypatch.setattr(K, "require_device", lambda t: None)
    monkeypatch.setattr(K, "stream_on", lambda i: 0)
    monkeypatch.setattr(K, "call", lambda name, *args: calls.append(name))
    c, table, n = PackedKVCache(4, 2, 64, device="cpu"), torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    flat = torch.zeros(3 * 3 * 4 * 64)
    q, wide = flat[:2 * 3 * 4 * 64].view(2, 3, 4, 64), torch.zeros(2, 3, 8, 64)
    for x, out in ((q, q), (q, torch.zeros_like(q)), (flat[256:512].view(1, 1, 4, 64), flat[:256].view(1, 1, 4, 64)),
                   (wide[:, :, :4], torch.zeros_like(q))):
        assert c.attend(x, table[:len(x)], n[:len(x)], out=out) is out
    assert len(calls) == 4
    for x, out in ((q, flat[64:][:q.numel()].view(2, 3, 4, 64)), (q, flat[768:].view(2, 3, 4, 64)),
                   (wide[:, :, :4], wide.view(-1)[:q.numel()].view(2, 3, 4, 64))):
        with pytest.raises(ValueError):
            c.attend(x, table, n, out=out)
    assert len(calls) == 4
