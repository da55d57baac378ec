"""Who reads the library's device error word, and when."""

from __future__ import annotations

import pytest
import torch

from src import _native as nat

pytestmark = pytest.mark.gpu


def test_reading_waits_for_streams_of_their_own():
    """PyTorch's streams do not block the legacy stream: a wait that runs out
    on one of them is still seen by the next read."""
    assert nat.device_error(reset=True) == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        assert nat.load().m3_selftest_wait_timeout(side.cuda_stream) == nat.M3_OK
    assert nat.device_error(reset=True) == nat.M3_DEVERR_TIMEOUT
    assert nat.device_error() == 0


def test_generate_raises(monkeypatch):
    """The word is stood in for: no kernel gives up here."""
    from src.models.lm import Mamba3LMDecoder
    from src.models.mamba3 import MambaConfig, MambaLMHeadModel
    cfg = MambaConfig(d_model=64, n_layer=1, vocab_size=50, ssm_cfg=dict(d_state=32, headdim=16))
    model = MambaLMHeadModel(cfg, device="cuda").eval()
    dec = Mamba3LMDecoder(model, use_triton_full_fused=True, w4_group_size=64)
    ids = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    words = [nat.M3_DEVERR_TIMEOUT]
    monkeypatch.setattr(nat, "device_error", lambda reset=False: words.pop() if words else 0)
    with pytest.raises(RuntimeError, match="bounded wait"):
        dec.generate(ids, 2)
    toks, _, _ = dec.generate(ids, 2)
    assert toks.shape == (2, 5) and not words
    # a captured decode_sequence does not read the word
    words.append(nat.M3_DEVERR_TIMEOUT)
    states = dec.init_state(2, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        dec.decode_sequence(ids, states)
    assert words
