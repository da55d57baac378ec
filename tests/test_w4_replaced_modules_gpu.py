"""4-bit decoders follow a model whose projections are replaced, weight and
module alike, as the unquantised decoders do."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import MambaConfig, MambaLMHeadModel

pytestmark = pytest.mark.gpu


def _model(dtype=torch.float32):
    torch.manual_seed(0)
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=50, d_intermediate=64,
                      ssm_cfg=dict(d_state=32, headdim=16, is_mimo=True, mimo_rank=4))
    return MambaLMHeadModel(cfg, device="cuda", dtype=dtype).eval()


PLACES = [lambda m: (m, "lm_head"), lambda m: (m.layers[1].mixer, "in_proj"), lambda m: (m.layers[0].mixer, "out_proj"),
          lambda m: (m.mlp_layers[0], "fc1"), lambda m: (m.mlp_layers[1], "fc2")]


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("place", range(len(PLACES)))
@pytest.mark.parametrize("w4", [None, 64])
def test_replaced(w4, place, whole):
    model = _model()
    ids = torch.tensor([3, 9], device="cuda")
    kw = dict(use_triton_full_fused=True, w4_group_size=w4)
    step = lambda dec: dec.step(ids, dec.init_state(2, device="cuda"))[0]  # noqa: E731
    with torch.no_grad():
        dec = Mamba3LMDecoder(model, **kw)
        before = step(dec)
        owner, name = PLACES[place](model)
        old = getattr(owner, name)
        if whole:
            setattr(owner, name, nn.Linear(old.in_features, old.out_features, bias=False, device="cuda"))
        else:
            old.weight = nn.Parameter(torch.randn_like(old.weight) * 0.1)
        got = step(dec)
        assert torch.equal(got, step(Mamba3LMDecoder(model, **kw)))
        assert not torch.equal(got, before)
