"""Captured 4-bit decoders and weights that change behind the capture."""

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


def _change(module):
    for p in module.parameters():
        if p.dim() == 2:
            p.mul_(-1.25)


def _zero(states):
    for st in states:
        for v in st.values():
            v.zero_()


@pytest.mark.parametrize("w4", [None, 64])
def test_language_model(w4):
    """As the unquantised captured decoder, whose graph reads the weights."""
    torch.manual_seed(0)
    m = MambaLMHeadModel(MambaConfig(d_model=64, n_layer=2, vocab_size=50, d_intermediate=64, ssm_cfg=LAYER),
                         device="cuda").eval()
    kw = dict(use_triton_full_fused=True, w4_group_size=w4)
    ids = torch.randint(0, 50, (3, 5), device="cuda")
    with torch.no_grad():
        dec = Mamba3LMDecoder(m, use_cuda_graph=True, **kw)
        states = dec.init_state(3, device="cuda")
        dec.warmup_cuda_graph(states)
        first = dec.generate(ids, 8)
        _change(m)
        toks, lps, _ = dec.generate(ids, 8)
        want, want_lps, _ = Mamba3LMDecoder(m, **kw).generate(ids, 8)
        assert torch.equal(toks, want) and not torch.equal(lps, first[1])
        torch.testing.assert_close(lps, want_lps, rtol=1e-4, atol=1e-4)
        _change(m)
        _zero(states)
        got, _ = dec.decode_sequence(ids, states)
        want, _ = Mamba3LMDecoder(m, **kw).decode_sequence(ids)
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
        _change(m)
        _zero(states)
        dec.update_w4()
        fresh = Mamba3LMDecoder(m, **kw)
        want, _ = fresh.step(ids[:, 0], fresh.init_state(3, device="cuda"))
        torch.testing.assert_close(dec.step(ids[:, 0], states)[0], want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("kind", ["layer", "stack"])
def test_layers(kind):
    torch.manual_seed(1)
    blocks = torch.nn.ModuleList([MambaBlock(64, LAYER, device="cuda") for _ in range(2)])
    new = (lambda graph: Mamba3StackDecoder(blocks, use_cuda_graph=graph, **FUSED)) if kind == "stack" else \
        (lambda graph: Mamba3Decoder(blocks[0].mixer, use_cuda_graph=graph, **FUSED))
    u = torch.randn(2, 4, 64, device="cuda")
    with torch.no_grad():
        dec = new(True)
        state = dec.init_state(2, device="cuda")
        dec.warmup_cuda_graph(state)
        for ways in ("step", "sequence"):
            if kind == "stack" and ways == "sequence":
                continue
            _change(blocks)
            _zero(state if kind == "stack" else [state])
            fresh = new(False)
            if ways == "step":
                dec.update_w4()
                got = dec.step(u[:, 0], state)[0]
                want = fresh.step(u[:, 0].contiguous(), fresh.init_state(2, device="cuda"))[0]
            else:
                got, want = dec.decode_sequence(u, state)[0], fresh.decode_sequence(u)[0]
            torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)


def test_changes_that_are_not_counted():
    torch.manual_seed(2)
    m = MambaLMHeadModel(MambaConfig(d_model=64, n_layer=1, vocab_size=50, d_intermediate=64, ssm_cfg=LAYER),
                         device="cuda").eval()
    ids = torch.randint(0, 50, (2, 3), device="cuda")
    dec = Mamba3LMDecoder(m, **FUSED)
    for p in m.parameters():
        if p.dim() == 2:
            p.data.mul_(-1.25)
    dec.update_w4(force=True)
    assert torch.equal(dec.decode_sequence(ids)[0], Mamba3LMDecoder(m, **FUSED).decode_sequence(ids)[0])
