"""``W4Projection`` and the tensors that a captured graph may hold."""

from __future__ import annotations

import torch

from src.kernels.linear_w4 import W4Projection, dequantize_w4, quantize_w4


def test_tensors_of_another_form_outlive_it():
    """The graph knows addresses only: what it reads must not be freed, or
    written by anything else."""
    lin = torch.nn.Linear(256, 48, bias=False)
    p = W4Projection(lambda: lin.weight, 64)
    first = p.get()
    held, codes, scales = first.codes.data_ptr(), first.codes.clone(), first.scales.clone()
    del first
    lin.weight = torch.nn.Parameter(lin.weight.detach().bfloat16())  # another type
    second = p.get()
    assert second.codes.data_ptr() != held and second.scales.dtype == torch.bfloat16
    assert torch.equal(dequantize_w4(second), dequantize_w4(quantize_w4(lin.weight, 64)))
    lin.weight = torch.nn.Parameter(torch.randn(16, 128))            # another shape
    p.get()
    kept = [w for w in p.kept if w.codes.data_ptr() == held]
    assert len(p.kept) == 2 and len(kept) == 1
    assert torch.equal(kept[0].codes, codes) and torch.equal(kept[0].scales, scales)
    n = len(p.kept)
    with torch.no_grad():
        lin.weight.mul_(2.0)                                         # the same form: in place
    p.get()
    assert len(p.kept) == n
