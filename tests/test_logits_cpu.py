"""Refusals of the logit operators that need no GPU: the C entry points'
checks and the Python checks on CPU tensors."""

from __future__ import annotations

import pytest
import torch

from src import _native as nat
from src.kernels.logits import next_tokens, process_logits
from src.models.lm import Mamba3LMDecoder
from src.models.mamba3 import Mamba3, MambaConfig, MambaLMHeadModel
from src.models.inference import Mamba3Decoder

FAKE = 0x7000_0000_0000


def _args(**change):
    v = dict(B=2, V=100, T=5, dtype=0, logits=FAKE, ld=100, tokens=FAKE, ts=5, lengths=FAKE, prompt=FAKE, ti=1, li=1,
             pi=1, sample=1, rep=0, pres=0, freq=0, rv=1.0, pv=0.0, fv=0.0, tv=1.0, bias=FAKE, bs=0, allowed=FAKE,
             als=0, out=FAKE, old=100, od=0, reserved=0, temp=0, seeds=FAKE, pos=0, ids=FAKE, lp=FAKE)
    v.update(change)
    return nat.LOGITS_ARGS.pack(*v.values())


@pytest.mark.parametrize("entry", ["m3_process_logits", "m3_next_tokens"])
@pytest.mark.parametrize("change,status", [
    (dict(logits=0), "NULL"), (dict(dtype=2), "DTYPE"), (dict(B=-1), "SHAPE"), (dict(V=0), "SHAPE"),
    (dict(V=(1 << 30) + 1, old=1 << 31), "SHAPE"), (dict(T=-1), "SHAPE"), (dict(ld=-1), "SHAPE"),
    (dict(ts=-1), "SHAPE"), (dict(bs=-1), "SHAPE"), (dict(als=-1), "SHAPE"), (dict(logits=FAKE + 2), "ALIGN"),
    (dict(tokens=FAKE + 4), "ALIGN"), (dict(lengths=FAKE + 4), "ALIGN"), (dict(prompt=FAKE + 4), "ALIGN"),
    (dict(bias=FAKE + 2), "ALIGN"), (dict(allowed=FAKE + 1), "ALIGN"), (dict(rep=FAKE + 1), "ALIGN"),
    (dict(B=0), "OK")])
def test_abi_validation(entry, change, status):
    want = nat.M3_OK if status == "OK" else getattr(nat, "M3_ERR_" + status)
    assert getattr(nat.load(), entry)(_args(**change), None) == want


@pytest.mark.parametrize("entry,change,status", [
    ("m3_process_logits", dict(out=0), "NULL"), ("m3_process_logits", dict(od=3), "DTYPE"),
    ("m3_process_logits", dict(old=99), "SHAPE"), ("m3_process_logits", dict(out=FAKE + 2), "ALIGN"),
    ("m3_next_tokens", dict(ids=0), "NULL"), ("m3_next_tokens", dict(lp=0), "NULL"),
    ("m3_next_tokens", dict(seeds=0), "NULL"), ("m3_next_tokens", dict(ids=FAKE + 4), "ALIGN"),
    ("m3_next_tokens", dict(pos=FAKE + 4), "ALIGN"), ("m3_next_tokens", dict(temp=FAKE + 2), "ALIGN")])
def test_abi_validation_of_one(entry, change, status):
    assert getattr(nat.load(), entry)(_args(**change), None) == getattr(nat, "M3_ERR_" + status)


def test_cpu_tensors_are_refused():
    for f in (process_logits, next_tokens):
        with pytest.raises(AssertionError):
            f(torch.zeros(2, 10))


def test_decoders_refuse_what_they_cannot_do(monkeypatch):
    model = MambaLMHeadModel(MambaConfig(d_model=32, n_layer=1, vocab_size=13, ssm_cfg=dict(d_state=16, headdim=16)))
    with pytest.raises(RuntimeError):
        Mamba3LMDecoder(model, use_triton=False).generate(torch.zeros(1, 2, dtype=torch.long), 3)
    with pytest.raises(ValueError):
        Mamba3LMDecoder(model, use_triton=False, w4_group_size=64)
    with pytest.raises(ValueError):
        Mamba3Decoder(Mamba3(32, d_state=16, headdim=16), use_triton=False, w4_group_size=64)
