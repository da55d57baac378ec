"""Weights loaded between a 4-bit decoder's making and a capture that no eager
step precedes."""

from __future__ import annotations

import pytest
import torch

from src.models.inference import Mamba3Decoder
from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import MambaBlock, MambaConfig, MambaLMHeadModel
from src.models.stack import Mamba3StackDecoder

pytestmark = pytest.mark.gpu
FUSED = dict(use_triton_full_fused=True, w4_group_size=64)
LAYER = dict(d_state=32, headdim=16, is_mimo=True, mimo_rank=4)


def _new(kind):
    """(module, its decoder with or without a graph, an input)"""
    torch.manual_seed(0)
    if kind == "lm":
        m = MambaLMHeadModel(MambaConfig(d_model=64, n_layer=2, vocab_size=50, d_intermediate=64, ssm_cfg=LAYER),
                             device="cuda").eval()
        return m, lambda graph: Mamba3LMDecoder(m, use_cuda_graph=graph, **FUSED), torch.tensor([3, 9], device="cuda")
    blocks = torch.nn.ModuleList([MambaBlock(64, LAYER, device="cuda") for _ in range(2)])
    u = torch.randn(2, 64, device="cuda")
    if kind == "stack":
        return blocks, lambda graph: Mamba3StackDecoder(blocks, use_cuda_graph=graph, **FUSED), u
    return blocks, lambda graph: Mamba3Decoder(blocks[0].mixer, use_cuda_graph=graph, **FUSED), u


@pytest.mark.parametrize("kind", ["lm", "stack", "layer"])
def test_capture_without_eager_steps(kind):
    module, decoder, u = _new(kind)
    with torch.no_grad():
        eager = decoder(False)
        eager.step(u, eager.init_state(2, device="cuda"))  # kernel attributes are set
        dec = decoder(True)
        for p in module.parameters():
            if p.dim() == 2:
                p.mul_(1.5)
        states = dec.init_state(2, device="cuda")
        dec.warmup_cuda_graph(states, n_warmup=0)
        got, _ = dec.step(u, states)
        fresh = decoder(False)
        want, _ = fresh.step(u, fresh.init_state(2, device="cuda"))
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)
