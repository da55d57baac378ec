"""``linear_w4`` of the smallest inputs."""

from __future__ import annotations

import pytest
import torch

from src.kernels.linear_w4 import linear_w4, pack_w4

pytestmark = pytest.mark.gpu


def _columns(K):
    """A weight of 1 in column 5 and 0 elsewhere, scaled by 2^60, so that no
    output is subnormal."""
    q = torch.full((16, K), 8, device="cuda")
    q[:, 5] = 9
    return pack_w4(q, torch.full((16, -(-K // 128)), 2.0 ** 60, device="cuda"))


@pytest.mark.parametrize("K", [6, 300, 13000])  # x in shared memory, and where it lies
@pytest.mark.parametrize("low,high", [(-110, -90), (-126, -110), (-149, -126)])
def test_fp32_terms(K, low, high):
    """Exact from 2^-110 on; below, each of the three terms is cut at bf16's
    smallest subnormal number, which loses less than 2^-133 of x.  The product
    with 1, the sum with zeros and the scale, a power of two, round nothing."""
    g = torch.Generator(device="cuda").manual_seed(-low)
    w = _columns(K)
    x = torch.zeros(64, K, device="cuda")
    e = torch.randint(low, high, (64,), generator=g, device="cuda").double()
    x[:, 5] = ((torch.rand(64, generator=g, device="cuda", dtype=torch.float64) + 1) * 2.0 ** e).float()
    x[1::2] = -x[1::2]
    x[0, 5] = 2.0 ** low
    y = linear_w4(x, w.codes, w.scales).double() / 2.0 ** 60
    assert bool((y == y[:, :1]).all())
    want = x[:, 5].double()
    if low >= -110:
        assert torch.equal(y[:, 0], want)
    else:
        assert bool(((y[:, 0] - want).abs() < 2.0 ** -133).all())


def test_bf16_subnormals():
    w = _columns(300)
    x = torch.zeros(8, 300, device="cuda").bfloat16()
    x[:, 5] = torch.tensor([2.0 ** -133, -(2.0 ** -133), 3 * 2.0 ** -133, 2.0 ** -127, 2.0 ** -126, -(2.0 ** -130), 0.0,
                            1.5 * 2.0 ** -126], device="cuda").bfloat16()
    y = linear_w4(x, w.codes, w.scales, out_dtype=torch.float32).double() / 2.0 ** 60
    assert torch.equal(y, x[:, 5:6].double().expand(8, 16))
