"""What ``generate`` refuses, it refuses before it touches a state."""

from __future__ import annotations

import pytest
import torch

from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import MambaConfig, MambaLMHeadModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_rows_of_the_states(graph):
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=50, ssm_cfg=dict(d_state=32, headdim=16))
    model = MambaLMHeadModel(cfg, device="cuda").eval()
    dec = Mamba3LMDecoder(model, use_triton_full_fused=True, use_cuda_graph=graph)
    states = dec.init_state(4, device="cuda")
    ids = torch.randint(0, 50, (4, 3), device="cuda")
    with torch.no_grad():
        if graph:
            dec.warmup_cuda_graph(states)
        toks, _, _ = dec.generate(ids, 3, states=None if graph else states)
    before = [{k: v.clone() for k, v in st.items()} for st in states]
    assert any(bool(v.any()) for st in before for v in st.values())
    passed = [states] + ([None] if graph else [])
    for rows in (1, 2, 5):  # one row would be repeated by the copy into a captured step's input
        for st in passed:
            with pytest.raises(ValueError, match="rows"):
                dec.generate(ids[:1].expand(rows, 3), 2, states=st)
    for st in passed:
        with pytest.raises(AssertionError, match="seeds"):
            dec.generate(ids, 2, states=st, temperature=0.5)
    assert all(torch.equal(v, b[k]) for st, b in zip(states, before) for k, v in st.items())
    if graph:
        assert torch.equal(dec.generate(ids, 3)[0], toks)
