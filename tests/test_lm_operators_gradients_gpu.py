"""The language-model operators have no gradient: whatever asks for one, in
reverse or forward mode, is refused and never dropped."""

from __future__ import annotations

import importlib

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from src import _native as nat
from src.kernels.linear_w4 import linear_w4, quantize_w4
from src.kernels.logits import next_tokens, process_logits

pytestmark = pytest.mark.gpu


def _calls():
    """(inputs that may ask for a gradient, call of them)"""
    g = torch.Generator(device="cuda").manual_seed(0)
    w = quantize_w4(torch.randn(40, 200, generator=g, device="cuda"), 64)
    x = torch.randn(3, 200, generator=g, device="cuda")
    z = torch.randn(2, 100, generator=g, device="cuda")
    bias, ones = torch.randn(100, generator=g, device="cuda"), torch.ones(2, device="cuda")
    hist = torch.zeros(2, 5, dtype=torch.long, device="cuda")
    seeds = torch.arange(2, device="cuda")
    names = ("repetition_penalty", "presence_penalty", "frequency_penalty")
    yield "w4", [x, w.scales], lambda x, s: linear_w4(x, w.codes, s, group_size=64)
    yield "process", [z, bias, ones, ones, ones], lambda z, b, *p: process_logits(z, hist, bias=b,
                                                                                   **dict(zip(names, p)))
    yield "next", [z, bias, ones, ones, ones, ones], lambda z, b, *p: next_tokens(
        z, hist, bias=b, **dict(zip(names, p)), temperature=p[3], seeds=seeds)[1]


CALLS = {"w4": 2, "process": 5, "next": 6}


@pytest.mark.parametrize("python_path", [False, True])
@pytest.mark.parametrize("name,i", [(n, i) for n, k in CALLS.items() for i in range(k)])
def test_refused(name, i, python_path, monkeypatch):
    if python_path:
        monkeypatch.setattr(importlib.import_module("src.kernels.linear_w4"), "_host", nat._no_host)
        monkeypatch.setattr(importlib.import_module("src.kernels.logits"), "_host_process", nat._no_host)
        monkeypatch.setattr(importlib.import_module("src.kernels.logits"), "_host_next", nat._no_host)
    inputs, call = next((a, f) for n, a, f in _calls() if n == name)
    assert len(inputs) == CALLS[name]
    want = call(*inputs)
    put = lambda t: [t if j == i else v for j, v in enumerate(inputs)]  # noqa: E731
    leaf = inputs[i].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        call(*put(leaf))
    with torch.no_grad():
        assert torch.equal(call(*put(leaf)), want)
    with fwAD.dual_level():
        dual = fwAD.make_dual(inputs[i], torch.ones_like(inputs[i]))
        for grad in (True, False):  # tangents go on under no_grad
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no gradient"):
                call(*put(dual))
        assert torch.equal(call(*inputs), want)
    assert torch.equal(call(*inputs), want)


def test_out_is_refused():
    z = torch.randn(2, 100, device="cuda")
    out = torch.full((2, 100), 7.0, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        process_logits(z, out=out)
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        process_logits(z, out=fwAD.make_dual(out.detach(), torch.ones_like(z)))
    assert bool((out == 7).all())
    with torch.no_grad():
        assert process_logits(z, out=out) is out and torch.equal(out, z)
