"""Refusals of the mixture-of-experts operators and of log probabilities: no GPU needed."""

import struct

import pytest
import torch

from tinygrad_mi355x.codegen.decomp.mi355x import PackedTensor
from tinygrad_mi355x.experts import PackedExperts, route
from tinygrad_mi355x.runtime import kernels as K
from tinygrad_mi355x.sampling import log_probs


# ----------------------------------------------------------------------------- routing
@pytest.mark.parametrize("logits,kw", [
    (torch.zeros(8), {}), (torch.zeros(4, 8, 2), {}), (torch.zeros(4, 8, dtype=torch.float64), {}), (torch.zeros(4, 0), {}),
    (torch.zeros(2, 1025), {}), (torch.zeros(8, 4).t(), {}), (torch.zeros(1, 8).expand(4, 8), {}),
    (torch.zeros(4, 8), dict(top_k=0)), (torch.zeros(4, 8), dict(top_k=9)), (torch.zeros(4, 8), dict(top_k=2.0)),
    (torch.zeros(4, 8), dict(score="relu")), (torch.zeros(4, 8), dict(groups=3)), (torch.zeros(4, 8), dict(groups=0)),
    (torch.zeros(4, 130), dict(groups=65)), (torch.zeros(4, 8), dict(groups=4, top_groups=5)),
    (torch.zeros(4, 8), dict(groups=4, top_groups=0)), (torch.zeros(4, 8), dict(groups=4, top_groups=1, top_k=3)),
    (torch.zeros(4, 8), dict(scale=float("inf"))), (torch.zeros(4, 8), dict(bias=torch.zeros(7))),
    (torch.zeros(4, 8), dict(bias=torch.zeros(8, dtype=torch.bfloat16))), (torch.zeros(4, 8), dict(bias=torch.zeros(16)[::2])),
    (torch.zeros(4, 8), dict(bias=torch.zeros(8, device="meta")))])
def test_route_refuses(logits, kw):
    with pytest.raises(ValueError):
        route(logits, kw.pop("top_k", 2), **kw)


def test_route_needs_the_device():
    with pytest.raises(RuntimeError):
        route(torch.zeros(4, 8), 2)


@pytest.mark.parametrize("args", [
    (9, 4, 8, 8, None, 0, 1, 1, 2, 1, 1.0), (13, -1, 8, 8, None, 0, 1, 1, 2, 1, 1.0), (13, 4, 1025, 1025, None, 0, 1, 1, 2, 1, 1.0),
    (13, 4, 8, 7, None, 0, 1, 1, 2, 1, 1.0), (13, 4, 8, 8, None, 2, 1, 1, 2, 1, 1.0), (13, 4, 8, 8, None, 0, 3, 1, 2, 1, 1.0),
    (13, 4, 8, 8, None, 0, 2, 3, 2, 1, 1.0), (13, 4, 8, 8, None, 0, 2, 1, 5, 1, 1.0), (13, 4, 8, 8, None, 0, 1, 1, 0, 1, 1.0),
    (13, 4, 8, 8, None, 0, 1, 1, 2, 1, float("nan")), (13, 4, 8, 8, None, 0, 1, 1, 2, 1, 1.0)])
def test_route_entry_point_refuses(args):
    """What the C entry point is given is checked before any launch; the last one has no operands."""
    with pytest.raises(ValueError):
        K.call("tgm_route", None, *args, None, None, None)


# ----------------------------------------------------------------------------- the experts' products
def weight(fmt, shape, scales=torch.float8_e8m0fnu, block=32, device="cpu"):
    bits = 4 if fmt in ("fp4_e2m1", "int4", "uint4") else 6
    n = 1
    for s in shape:
        n *= s
    sc = None if scales is None else torch.zeros(shape[:-1] + (-(-shape[-1] // block),), dtype=scales, device=device)
    return PackedTensor(torch.zeros((n * bits + 7) // 8, dtype=torch.uint8, device=device), fmt, shape, sc, block)


def layer(fmt="fp4_e2m1", experts=2, hidden=128, ffn=128, scales=torch.float8_e8m0fnu, block=32):
    return PackedExperts(weight(fmt, (experts, 2 * ffn, hidden), scales, block), weight(fmt, (experts, hidden, ffn), scales, block))


@pytest.mark.parametrize("gate_up,down", [
    (weight("fp4_e2m1", (512, 128)), weight("fp4_e2m1", (2, 128, 128))),
    (weight("fp4_e2m1", (2, 256, 128)), torch.zeros(2, 128, 128)),
    (weight("fp4_e2m1", (2, 256, 128)), weight("fp4_e2m1", (3, 128, 128))),
    (weight("fp4_e2m1", (2, 256, 128)), weight("fp4_e2m1", (2, 128, 256))),
    (weight("fp4_e2m1", (2, 257, 128)), weight("fp4_e2m1", (2, 128, 128))),
    (weight("fp4_e2m1", (2, 256, 96)), weight("fp4_e2m1", (2, 96, 128))),
    (weight("fp4_e2m1", (2, 192, 128)), weight("fp4_e2m1", (2, 128, 96))),
    (weight("fp4_e2m1", (2, 256, 128)), weight("fp6_e2m3", (2, 128, 128))),
    (weight("fp4_e2m1", (2, 256, 128)), weight("fp4_e2m1", (2, 128, 128), None)),
    (weight("fp4_e2m1", (2, 256, 128), torch.float32), weight("fp4_e2m1", (2, 128, 128), torch.float32)),
    (weight("fp4_e2m1", (2, 256, 128), block=64), weight("fp4_e2m1", (2, 128, 128), block=64)),
    (weight("int4", (2, 256, 128)), weight("int4", (2, 128, 128))),
    (weight("int4", (2, 256, 128), torch.float16, 16), weight("int4", (2, 128, 128), torch.float16, 16)),
    (weight("fp4_e2m1", (0, 256, 128)), weight("fp4_e2m1", (0, 128, 128))),
    (weight("fp4_e2m1", (1025, 256, 128)), weight("fp4_e2m1", (1025, 128, 128)))])
def test_experts_refuse_weights(gate_up, down):
    with pytest.raises(ValueError):
        PackedExperts(gate_up, down)


BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("x,ids,weights,out", [
    (torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(4, 2, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(4, 128), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(4, 128, dtype=torch.float16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(128, 4, dtype=BF16).t(), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(1, 128, dtype=BF16).expand(4, 128), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(4, 132, dtype=BF16)[:, :128], torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(3, 2, dtype=I32), torch.zeros(3, 2), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 0, dtype=I32), torch.zeros(4, 0), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(2, 4, dtype=I32).t(), torch.zeros(4, 2), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 3), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2, dtype=BF16), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32, device="meta"), torch.zeros(4, 2), None),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), torch.zeros(4, 128, dtype=torch.float16)),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), torch.zeros(5, 128, dtype=BF16)),
    (torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2), torch.zeros(1, 128, dtype=BF16).expand(4, 128))])
def test_experts_refuse_operands(x, ids, weights, out):
    with pytest.raises(ValueError):
        layer().apply(x, ids, weights, out=out)


def test_experts_need_the_device():
    with pytest.raises(RuntimeError):
        layer().apply(torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2))


def experts_arg(**kw):
    v = dict(experts=4, hidden=256, ffn=384, format=2, scale_dtype=15, block=32) | kw
    return struct.pack("PPPPqqqqqq", 4096, 4096, 4096, 4096, *v.values())


@pytest.mark.parametrize("kw", [dict(format=5), dict(experts=0), dict(experts=1025), dict(hidden=192), dict(ffn=0), dict(hidden=1 << 18),
                                dict(scale_dtype=11), dict(block=64), dict(format=0), dict(format=0, scale_dtype=11, block=16),
                                dict(hidden=1 << 17, ffn=1 << 17)])
def test_experts_entry_points_refuse_layers(kw):
    lib = K.load_library()
    assert lib.tgm_experts_workspace(experts_arg(**kw), 4, 2) == 0
    with pytest.raises(ValueError):
        K.call("tgm_experts_apply", experts_arg(**kw), 4096, 12, 4, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40, None)


@pytest.mark.parametrize("args", [
    (4096, 11, 4, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40), (4096, 12, 4, 256, 4096, 4096, 2, 4096, 11, 256, 4096, 1 << 40),
    (4096, 12, 4, 255, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40), (4096, 12, 4, 260, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40),
    (4096, 12, 4, 256, 4096, 4096, 2, 4096, 12, 255, 4096, 1 << 40), (4096, 12, -1, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40),
    (4096, 12, 1 << 23, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 50), (4096, 12, 1 << 22, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 50),
    (4096, 12, 4, 256, 4096, 4096, 0, 4096, 12, 256, 4096, 1 << 40), (4104, 12, 4, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 1 << 40),
    (4096, 12, 4, 256, None, 4096, 2, 4096, 12, 256, 4096, 1 << 40), (4096, 12, 4, 256, 4096, 4096, 2, None, 12, 256, 4096, 1 << 40),
    (4096, 12, 4, 256, 4096, 4096, 2, 4096, 12, 256, 4096, 100), (4096, 12, 4, 256, 4096, 4096, 2, 4096, 12, 256, 4097, 1 << 40)])
def test_experts_entry_point_refuses_operands(args):
    with pytest.raises(ValueError):
        K.call("tgm_experts_apply", experts_arg(), *args, None)


def test_experts_workspace_of_no_tokens_and_of_more():
    lib = K.load_library()
    assert lib.tgm_experts_workspace(experts_arg(), 0, 2) == 0
    few, more = (lib.tgm_experts_workspace(experts_arg(), t, 2) for t in (4, 4000))
    assert few >= 8 * (384 * 2 + 256 * 4) and more >= 8000 * (384 * 2 + 256 * 4)


# ----------------------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("logits,tokens,top", [
    (torch.zeros(8), torch.zeros(8, dtype=I32), 0), (torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, dtype=I32), 0),
    (torch.zeros(4, 0), torch.zeros(4, dtype=I32), 0), (torch.zeros(1, (1 << 20) + 1), torch.zeros(1, dtype=I32), 0),
    (torch.zeros(8, 4).t(), torch.zeros(4, dtype=I32), 0), (torch.zeros(1, 8).expand(4, 8), torch.zeros(4, dtype=I32), 0),
    (torch.zeros(4, 8), torch.zeros(3, dtype=I32), 0), (torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), 0),
    (torch.zeros(4, 8), torch.zeros(8, dtype=I32)[::2], 0), (torch.zeros(4, 8), 3, 0), (torch.zeros(4, 8), torch.zeros(4, 1, dtype=I32), 0),
    (torch.zeros(4, 8), torch.zeros(4, dtype=I32, device="meta"), 0), (torch.zeros(4, 8), torch.zeros(4, dtype=I32), 9),
    (torch.zeros(4, 100), torch.zeros(4, dtype=I32), 65), (torch.zeros(4, 8), torch.zeros(4, dtype=I32), -1),
    (torch.zeros(4, 8), torch.zeros(4, dtype=I32), 2.0)])
def test_log_probs_refuses(logits, tokens, top):
    with pytest.raises(ValueError):
        log_probs(logits, tokens, top=top)


def test_log_probs_needs_the_device():
    with pytest.raises(RuntimeError):
        log_probs(torch.zeros(4, 8), torch.zeros(4, dtype=I32), top=2)


@pytest.mark.parametrize("args", [
    (4096, 9, 4, 8, 8, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0), (4096, 13, -1, 8, 8, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0),
    (4096, 13, 4, 0, 8, 4096, 0, 4096, 4096, 4096, 4096, 4096, None, 0), (4096, 13, 4, 8, 7, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0),
    (4096, 13, 4, 8, 8, 4096, 9, 4096, 4096, 4096, 4096, 4096, None, 0), (4096, 13, 4, 100, 100, 4096, 65, 4096, 4096, 4096, 4096, 4096, None, 0),
    (None, 13, 4, 8, 8, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0), (4096, 13, 4, 8, 8, 4096, 2, 4096, 4096, 4096, None, 4096, None, 0),
    (4098, 13, 4, 8, 8, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0),
    (4096, 13, 4, 200000, 200000, 4096, 2, 4096, 4096, 4096, 4096, 4096, None, 0)])
def test_log_probs_entry_point_refuses(args):
    with pytest.raises(ValueError):
        K.call("tgm_log_probs", *args, None)
