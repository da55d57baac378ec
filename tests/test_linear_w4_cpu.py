"""4-bit weights without a GPU: the storage form, the quantiser, the C
argument block and the refusals of ``linear_w4``."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from src import _native as nat
from src.kernels.linear_w4 import (GROUP_SIZES, W4Weight, dequantize_w4, linear_w4, pack_w4, quantize_w4, unpack_w4)

SHAPES = [(1, 1), (16, 128), (17, 130), (33, 1111), (100, 257)]


@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_codes_survive_packing(N, K, G):
    g = torch.Generator().manual_seed(N * K + G)
    q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    s = torch.rand(N, -(-K // G), generator=g)
    z = torch.randint(0, 16, s.shape, generator=g)
    w = pack_w4(q, s, z, G)
    assert w.shape == (N, K) and w.codes.shape == (-(-N // 16), -(-K // 128), 16, 16)
    assert torch.equal(unpack_w4(w), q)
    at = torch.arange(K) // G
    assert torch.equal(dequantize_w4(w), (q.float() - z.float()[:, at]) * s[:, at])


def test_storage_places():
    """Word 4 t + j of a block's row holds columns 32 j + 8 t .. + 7, the even
    ones in the low half."""
    for k, place in [(0, (0, 0)), (1, (0, 16)), (2, (0, 4)), (7, (0, 28)), (8, (4, 0)), (32, (1, 0)), (127, (15, 28))]:
        q = torch.zeros(16, 128, dtype=torch.uint8)
        q[3, k] = 9
        words = pack_w4(q, torch.ones(16, 1)).codes[0, 0]
        word, bit = place
        assert (int(words[3, word]) >> bit) & 15 == 9
        words[3, word] = 0
        assert not words[3].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_quantise_is_nearest(G, zero_points, dtype):
    g = torch.Generator().manual_seed(G)
    w = torch.randn(20, 300, generator=g).to(dtype)
    w[3] = 0
    w[4, :G] = 2.0    # one-sided groups
    w[5, :G] = -3.0
    q = quantize_w4(w, G, zero_points)
    assert q.scales.dtype == dtype and (q.zeros is None) == (not zero_points)
    d = dequantize_w4(q)
    assert not d[3].any()
    scale = q.scales.float()[:, torch.arange(300) // G]
    # half a step; the zero point and the ends of the range are rounded too:
    # the stored scale may be short of range / 15 (or / 7) by half a place of
    # its type, 7 or 15 times, and a rounded zero point shifts the range by
    # up to half a step
    eps = torch.finfo(dtype).eps / 2
    room = 0.5 + 15 * eps + (0.5 if zero_points else 0.0) + 1e-5
    assert bool(((d - w.float()).abs() <= room * scale).all())


def test_quantise_refusals():
    with pytest.raises(ValueError):
        quantize_w4(torch.tensor([[1.0, float("nan")]]))
    with pytest.raises(ValueError):
        quantize_w4(torch.ones(2, 2), group_size=16)
    with pytest.raises(AssertionError):
        quantize_w4(torch.ones(4))
    with pytest.raises(AssertionError):
        pack_w4(torch.full((2, 2), 16), torch.ones(2, 1))
    with pytest.raises(AssertionError):
        pack_w4(torch.zeros(2, 2, dtype=torch.int64), torch.ones(2, 2))


def test_linear_refuses_without_a_gpu_tensor():
    w = quantize_w4(torch.randn(16, 128))
    with pytest.raises(AssertionError):
        linear_w4(torch.randn(2, 128), w.codes, w.scales)
    with pytest.raises(ValueError):
        linear_w4(torch.randn(2, 128), w.codes, w.scales, group_size=100)


_LAYOUT_C = r"""
#include <stdio.h>
#include <stddef.h>
#include "mamba3_b200_lm.h"
int main(void) {
  printf("%zu %zu %zu %zu\n", sizeof(m3_w4_args), offsetof(m3_w4_args, x_dtype), offsetof(m3_w4_args, zeros),
         offsetof(m3_w4_args, y_dtype));
  printf("%zu %zu %zu %zu %zu\n", sizeof(m3_logits_args), offsetof(m3_logits_args, tokens_i64),
         offsetof(m3_logits_args, repetition_value), offsetof(m3_logits_args, out_dtype),
         offsetof(m3_logits_args, logprobs));
  return 0;
}
"""


def test_packed_blocks_match_the_c_structs(tmp_path):
    import struct
    src, exe = str(tmp_path / "l.c"), str(tmp_path / "l")
    open(src, "w").write(_LAYOUT_C)
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
    w4, lg = [[int(v) for v in line.split()]
              for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines()]
    at = lambda prefix, code: struct.calcsize(prefix + code) - struct.calcsize("@" + code)  # noqa: E731
    f = nat.W4_ARGS.format
    assert f.startswith("@iiiiPqiPPqiPqPqi")
    assert w4 == [nat.W4_ARGS.size, at("@iiiiPq", "i"), at("@iiiiPqiPPqi", "P"), at("@iiiiPqiPPqiPqPq", "i")]
    assert lg == [nat.LOGITS_ARGS.size, at("@iiiiPqPqPP", "i"), at("@iiiiPqPqPPiiiiPPP", "f"),
                  at("@iiiiPqPqPPiiiiPPPffffPqPqPq", "i"), at("@iiiiPqPqPPiiiiPPPffffPqPqPqiiPPPP", "P")]


def _w4(**change):
    fake = 0x7000_0000_0000
    v = dict(M=2, N=16, K=200, group=64, x=fake, ldx=200, xd=0, codes=fake, scales=fake, ss=4, sd=0, zeros=fake, zs=4,
             y=fake, ldy=16, yd=1)
    v.update(change)
    return nat.W4_ARGS.pack(*v.values())


@pytest.mark.parametrize("change,status", [
    (dict(x=0), "NULL"), (dict(codes=0), "NULL"), (dict(scales=0), "NULL"), (dict(y=0), "NULL"),
    (dict(xd=2), "DTYPE"), (dict(sd=5), "DTYPE"), (dict(yd=-1), "DTYPE"),
    (dict(group=16), "SHAPE"), (dict(group=0), "SHAPE"), (dict(M=-1), "SHAPE"), (dict(N=0), "SHAPE"),
    (dict(K=0), "SHAPE"), (dict(ldx=-1), "SHAPE"), (dict(ldy=15), "SHAPE"), (dict(ss=3), "SHAPE"),
    (dict(zs=3), "SHAPE"), (dict(codes=0x7000_0000_0008), "ALIGN"), (dict(x=0x7000_0000_0002), "ALIGN"),
    (dict(M=0), "OK")])
def test_abi_validation(change, status):
    want = nat.M3_OK if status == "OK" else getattr(nat, "M3_ERR_" + status)
    assert nat.load().m3_linear_w4(_w4(**change), None) == want


def test_abi_null_block():
    assert nat.load().m3_linear_w4(None, None) == nat.M3_ERR_NULL
    assert isinstance(ctypes.c_char_p(_w4()).value, bytes)
    assert W4Weight._fields == ("codes", "scales", "zeros", "group_size", "in_features")


def test_projection_follows_its_weight():
    """A change in place, another parameter on the same memory, another shape,
    and one that is not counted."""
    from src.kernels.linear_w4 import W4Projection
    lin = torch.nn.Linear(256, 48, bias=False)
    p = W4Projection(lambda: lin.weight, 64)
    first = p.get()
    assert p.get() is first
    want = lambda: dequantize_w4(quantize_w4(lin.weight, 64))  # noqa: E731
    codes = first.codes.data_ptr()
    with torch.no_grad():
        lin.weight.mul_(-2.0)
    assert torch.equal(dequantize_w4(p.get()), want()) and p.get().codes.data_ptr() == codes
    other = torch.nn.Parameter(lin.weight.data)
    other.data.mul_(3.0)
    lin.weight = other
    assert torch.equal(dequantize_w4(p.get()), want())
    lin.weight.data.mul_(0.5)
    p.refresh()
    assert torch.equal(dequantize_w4(p.get()), want())
    lin.weight = torch.nn.Parameter(torch.randn(16, 128))
    assert p.get().shape == (16, 128) and torch.equal(dequantize_w4(p.get()), want())
    lin.weight = torch.nn.Parameter(torch.randn(16, 128).half())
    with pytest.raises(ValueError):
        p.get()
