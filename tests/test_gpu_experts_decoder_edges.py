"""Layers of experts that a decoder is given: what it refuses."""

from dataclasses import replace

import pytest
import torch

from test_gpu_experts_decoder import MIXED
from tinygrad_mi355x.codegen.decomp.mi355x import PackedTensor
from tinygrad_mi355x.decoder import Decoder, random_weights

pytestmark = pytest.mark.gpu


def test_routers_and_experts_that_the_kernels_cannot_read(dev):
    """A router's rows lie one after another, on the decoder's device as the experts do."""
    w = random_weights(MIXED, dev, seed=8)
    L = w.layers[1]

    def host(t):
        return PackedTensor(t.data.cpu(), t.format, t.shape, t.scales.cpu(), t.block_size)

    transposed = L.router.t().contiguous().t()
    apart = torch.zeros((MIXED.experts, MIXED.hidden + 64), dtype=torch.bfloat16, device=dev)[:, :MIXED.hidden]
    for bad in (replace(L, router=transposed), replace(L, router=apart), replace(L, router=L.router[:1].expand(MIXED.experts, -1)),
                replace(L, router=L.router.cpu()), replace(L, w_gate_up=host(L.w_gate_up), w_down=host(L.w_down))):
        with pytest.raises(ValueError):
            Decoder(replace(w, layers=[w.layers[0], bad]), MIXED, 1, 32, 16)
    Decoder(replace(w, layers=[w.layers[0], replace(L, router=transposed.contiguous())]), MIXED, 1, 32, 16)
