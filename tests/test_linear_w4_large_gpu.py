"""``linear_w4`` where offsets pass 31 and 32 bits."""

from __future__ import annotations

import pytest
import torch

from src.kernels.linear_w4 import W4Weight, linear_w4
from test_linear_w4_gpu import check, make

pytestmark = pytest.mark.gpu


def _part(w: W4Weight, block: int, n: int) -> W4Weight:
    rows = slice(block * 16, (block + n) * 16)
    return W4Weight(w.codes[block:block + n], w.scales[rows], None if w.zeros is None else w.zeros[rows],
                    w.group_size, w.in_features)


@pytest.fixture(scope="module")
def weight():
    """3.4 GB of codes and 0.8 GB of scales: past 2^31 bytes, below 2^32."""
    N, K, G = 414_720, 16384, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(-2 ** 31, 2 ** 31, (N // 16, K // 128, 16, 16), generator=g, device="cuda",
                          dtype=torch.int64).int()
    scales = torch.rand(N, K // G, generator=g, device="cuda") + 0.5
    zeros = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8)
    assert 2 ** 31 < codes.numel() * 4 < 2 ** 32
    return W4Weight(codes, scales, zeros, G, K)


@pytest.mark.parametrize("M,dtype", [(1, torch.bfloat16), (16, torch.bfloat16), (40, torch.bfloat16),
                                     (1, torch.float32), (20, torch.float32)])
def test_large_weights(weight, M, dtype):
    w = weight
    x = torch.randn(M, w.in_features, device="cuda").to(dtype)
    y = linear_w4(x, w.codes, w.scales, w.zeros, group_size=w.group_size)
    half = 2 ** 31 // (w.codes.shape[1] * 1024)  # the block at 2^31 bytes
    for block in (0, half - 2, w.codes.shape[0] - 4):
        p = _part(w, block, 4)
        check(y[:, block * 16:(block + 4) * 16], x, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_outputs_and_inputs(dtype):
    """2.2e9 outputs; rows of x 2^20 elements apart."""
    w = make(50280, 128, 128, True, seed=1)
    x = torch.randn(44000, 128, device="cuda").to(dtype)
    y = linear_w4(x, w.codes, w.scales, w.zeros, out_dtype=torch.bfloat16)
    assert y.numel() > 2 ** 31
    for r in (0, 42700, 43990):
        check(y[r:r + 10], x[r:r + 10], w)
    del y
    wide = torch.zeros(2100, 1 << 20, device="cuda", dtype=dtype)
    wide[:, :128] = x[:2100]
    y = linear_w4(wide[:, :128], w.codes[:64], w.scales[:1024], w.zeros[:1024])
    check(y[2040:], x[2040:2100], _part(w, 0, 64))


def test_a_weight_past_the_offsets_is_refused():
    """4 GB of codes and more, on a GPU that holds them; nothing is launched."""
    codes = torch.empty(16385, 256, 16, 16, dtype=torch.int32, device="cuda")
    scales = torch.empty(16385 * 16, 256, device="cuda")
    x = torch.empty(1, 32768, device="cuda").bfloat16()
    with pytest.raises(AssertionError, match="m3_linear_w4"):
        linear_w4(x, codes, scales)
