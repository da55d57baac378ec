"""Every kernel of ``linear_w4`` at sizes that take it.

Which kernel a call takes is not visible from outside; the tests state the
launcher's conditions (csrc/m3_w4.cu) for the device's number of SMs, so that
a changed rule shows here."""

from __future__ import annotations

import pytest
import torch

from src import _native as nat
from src.kernels.linear_w4 import GROUP_SIZES, linear_w4
from test_linear_w4_gpu import MANY, check, make

pytestmark = pytest.mark.gpu


def sms() -> int:
    return torch.cuda.get_device_properties(0).multi_processor_count


def blocks(N: int) -> int:
    return -(-N // 16)


def tiles(K: int) -> int:
    return -(-K // 128)


def tensor_memory(M: int, N: int, K: int, G: int) -> bool:
    """A bf16 x with rows on 16 bytes goes to w4_tc_kernel."""
    work = blocks(N) * tiles(K) * -(-M // 64)
    return K >= 128 and ((M > 32 and work >= 30 * sms()) or (M > 16 and G == 128 and work >= 150 * sms()))


def run(M, N, K, G, dtype):
    for zeros, s_dtype in ((False, torch.float32), (True, torch.bfloat16)):
        w = make(N, K, G, zeros, s_dtype, seed=M + N + K)
        g = torch.Generator(device="cuda").manual_seed(K)
        x = torch.randn(M, K, device="cuda", generator=g).to(dtype)
        for out_dtype in (torch.float32, torch.bfloat16):
            check(linear_w4(x, w.codes, w.scales, w.zeros, group_size=G, out_dtype=out_dtype), x, w)
    assert nat.device_error() == 0


def test_the_many_rows_cases_reach_tensor_memory():
    assert all(tensor_memory(M, N, K, G) for M, N, K in MANY for G in GROUP_SIZES)


@pytest.mark.parametrize("M,N,K", [(17, 50280, 1032), (32, 50280, 1160), (24, 50277, 1160)])
def test_tensor_memory_with_few_rows(M, N, K):
    """More than half of a copy's box and of an accumulator lie behind x."""
    assert tensor_memory(M, N, K, 128)
    run(M, N, K, 128, torch.bfloat16)


@pytest.mark.parametrize("M", [9, 16])
@pytest.mark.parametrize("K", [640, 1111])
@pytest.mark.parametrize("G", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_row_blocks_a_warp(dtype, G, K, M):
    """9 to 16 rows of a weight with two row blocks an SM or more; the last
    pair of an odd number has one, and that one is not whole."""
    n = 2 * sms() + 1
    assert n % 2 == 1
    for N in (16 * n - 5, 16 * (n + 1)):
        run(M, N, K, G, dtype)


@pytest.mark.parametrize("M", [1, 8, 9, 16, 40])
@pytest.mark.parametrize("K", [5120, 5111])
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_fp32_rows_that_shared_memory_does_not_hold(G, K, M):
    """Three terms of 8 rows are 6 KB a tile of columns: past 32 tiles x is
    read where it lies."""
    assert tiles(K) * 6 * 1024 > 227 * 1024 - 16 * 8 * 17 * 4
    run(M, 5003, K, G, torch.float32)


@pytest.mark.parametrize("M", [1, 9, 40])
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_bf16_rows_that_shared_memory_does_not_hold(G, M):
    """2 KB a tile; rows off 16 bytes, which TMA does not read."""
    K = 14501
    assert tiles(K) * 2 * 1024 > 227 * 1024 - 16 * 8 * 17 * 4
    run(M, 1003, K, G, torch.bfloat16)
