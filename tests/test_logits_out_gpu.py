"""``process_logits`` into other columns of the buffer that holds its logits."""

from __future__ import annotations

import pytest
import torch

from src.kernels.logits import process_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                             (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("B,V,first", [(3, 1000, 0), (300, 501, 3), (2, 20001, 5)])
def test_parts_of_one_buffer(B, V, first, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    width = 2 * V + 16  # of fp32
    ref = torch.randn(B, width, generator=g, device="cuda")
    hist = torch.randint(0, V, (B, 90), generator=g, device="cuda")
    kw = dict(repetition_penalty=1.5, frequency_penalty=0.25, presence_penalty=0.5)
    for swap in (False, True):
        buf = ref.clone()
        at, to = (V + 8, first) if swap else (first, V + 8)  # places of fp32
        # bf16 views put the same bytes at twice the place
        cut = lambda t, place: buf.view(t)[:, place * (4 // t.itemsize):][:, :V]  # noqa: E731
        logits, out = cut(dtype, at), cut(out_dtype, to)
        logits.copy_(torch.randn(B, V, generator=g, device="cuda") * 3)
        want = process_logits(logits.clone(), hist, **kw, out=torch.empty(B, V, device="cuda", dtype=out_dtype))
        before = buf.clone()
        got = process_logits(logits, hist, **kw, out=out)
        assert got is out and torch.equal(out, want)
        out.copy_(before.view(out_dtype)[:, to * (4 // out_dtype.itemsize):][:, :V])
        assert torch.equal(buf.view(torch.int32), before.view(torch.int32))  # nothing else was written
    with pytest.raises(AssertionError, match="overlap"):
        process_logits(ref[:, :V], hist, **kw, out=ref[:, V - 1:2 * V - 1])
