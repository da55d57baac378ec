"""The decoders of token sequences report a kernel that gave up a bounded
wait.  No GPU and no such kernel: the library's error word and the layers'
steps are stood in for."""

from __future__ import annotations

import pytest
import torch

from src import _native as nat
from src.models.inference import check_device_error
from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import Mamba3, MambaBlock, MambaConfig, MambaLMHeadModel
from src.models.stack import Mamba3StackDecoder


@pytest.fixture
def word(monkeypatch):
    """What the library's word holds; a read clears it."""
    held = [nat.M3_DEVERR_TIMEOUT]

    def read(reset=False):
        v = held[0]
        if reset:
            held[0] = 0
        return v
    monkeypatch.setattr(nat, "device_error", read)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    return held


def _lm():
    model = MambaLMHeadModel(MambaConfig(d_model=32, n_layer=2, vocab_size=16, ssm_cfg=dict(d_state=16, headdim=16)))
    dec = Mamba3LMDecoder(model, use_triton=False)
    dec.cuda = True
    return dec


def test_decode_sequence_raises(word):
    dec = _lm()
    dec.step = lambda ids, states: (torch.zeros(len(ids), 16), states)
    ids = torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="bounded wait"):
        dec.decode_sequence(ids)
    assert word == [0] and dec.decode_sequence(ids)[0].shape == (2, 3, 16)


def test_warm_up_raises_before_the_capture(word):
    for dec in (_lm(), Mamba3StackDecoder([MambaBlock(32, dict(d_state=16, headdim=16))], use_triton=False)):
        dec.use_cuda_graph = True
        dec._step_eager = lambda x, states: (x, states)
        word[0] = nat.M3_DEVERR_TIMEOUT
        with pytest.raises(RuntimeError, match="bounded wait"):
            dec.warmup_cuda_graph(dec.init_state(2))
        assert dec._graph is None


def test_every_layers_workspace_is_zeroed(word):
    class Launch:
        def __init__(self):
            self.workspace = torch.ones(8)

    class Layer:
        def __init__(self, launch):
            self.model, self._step_cache = Mamba3(32, d_state=16, headdim=16), launch
    launches = [Launch(), Launch()]
    layers = [Layer(None), Layer((0, launches[0])), Layer((0, None)), Layer((0, launches[1]))]
    with pytest.raises(RuntimeError, match="bounded wait"):
        check_device_error(layers)
    assert not any(x.workspace.any() for x in launches)
    check_device_error(layers)
    word[0] = -1
    with pytest.raises(RuntimeError, match="could not be read"):
        check_device_error(layers)
