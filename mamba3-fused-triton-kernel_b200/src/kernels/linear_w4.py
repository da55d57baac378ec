"""Projections with 4-bit weights (``m3_linear_w4``).

A decode step of a few sequences is a stream of its projections' weights, so
a weight held in half a byte takes about a quarter of bf16's time.  A weight
(N, K) becomes codes 0..15 with one scale, and optionally one zero point, for
every row and group of 32, 64 or 128 columns:

    W[n, k] ~ (code[n, k] - zero[n, k // G]) * scale[n, k // G]

``quantize_w4`` makes that form from a weight and ``pack_w4`` from codes that
another tool has chosen; ``dequantize_w4`` is the weight it stands for.  They
are set-up work in plain PyTorch and run on any device.  ``linear_w4`` is the
product, ``x @ W.T``, on the GPU: fp32 or bf16 x, fp32 sums, the scale applied
to a group's sum and not to the weight, the output rounded once.  A weight
``W4Weight`` also goes through ``src.kernels.linear.linear``.

No counterpart in the reference, whose projections are ``nn.Linear``
(src/models/mamba3.py:115,158).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from src import _native as nat

GROUP_SIZES = (32, 64, 128)
ROWS, TILE = 16, 128  # rows and columns of a storage block
# bits of a word at which the eight columns it holds start
_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


class W4Weight(NamedTuple):
    """A quantised (out_features, in_features) weight.

    codes  (ceil(N / 16), ceil(K / 128), 16, 16) int32: blocks of 16 rows by
           128 columns; word 4 t + j of a block's row holds its columns
           32 j + 8 t .. + 7 (include/mamba3_b200_lm.h gives the bits)
    scales (N, ceil(K / G)) float32 or bfloat16
    zeros  (N, ceil(K / G)) uint8 in 0..15, or None for 8 throughout
    """

    codes: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    group_size: int
    in_features: int

    @property
    def shape(self) -> tuple:
        return (self.scales.shape[0], self.in_features)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)


def _check_group(group_size: int) -> None:
    if group_size not in GROUP_SIZES:
        raise ValueError(f"Unsupported group_size={group_size}. Supported values: {list(GROUP_SIZES)}")


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
            group_size: int = 128) -> W4Weight:
    """``W4Weight`` from codes (N, K) of any integer type with values 0..15,
    scales and zeros (N, ceil(K / group_size))."""
    _check_group(group_size)
    assert codes.dim() == 2 and codes.shape[0] > 0 and codes.shape[1] > 0, "codes must be (N, K)"
    N, K = codes.shape
    groups = -(-K // group_size)
    assert tuple(scales.shape) == (N, groups), f"scales must be {(N, groups)}, got {tuple(scales.shape)}"
    assert not codes.is_floating_point() and int(codes.min()) >= 0 and int(codes.max()) <= 15, "codes must be 0..15"
    if zeros is not None:
        assert tuple(zeros.shape) == (N, groups), f"zeros must be {(N, groups)}, got {tuple(zeros.shape)}"
        assert not zeros.is_floating_point() and int(zeros.min()) >= 0 and int(zeros.max()) <= 15, \
            "zeros must be 0..15"
        zeros = zeros.to(device=codes.device, dtype=torch.uint8).contiguous()
    scales = (scales if scales.dtype in (torch.float32, torch.bfloat16) else scales.float()).detach()
    blocks, tiles = -(-N // ROWS), -(-K // TILE)
    q = torch.full((blocks * ROWS, tiles * TILE), 8, dtype=torch.uint8, device=codes.device)
    q[:N, :K] = codes
    q = q.view(blocks, ROWS, tiles, 4, 4, 8).permute(0, 2, 1, 4, 3, 5)  # [..][row][t][j][8 columns]
    words = torch.zeros(q.shape[:-1], dtype=torch.int32, device=codes.device)
    for i, shift in enumerate(_SHIFTS):
        words |= q[..., i].int() << shift
    words = words.reshape(blocks, tiles, ROWS, 16).contiguous()
    return W4Weight(words, scales.to(codes.device).contiguous(), zeros, group_size, K)


def unpack_w4(weight: W4Weight) -> torch.Tensor:
    """The codes (N, K) of a ``W4Weight`` as uint8."""
    N, K = weight.shape
    shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=weight.codes.device)
    words = weight.codes.unflatten(3, (4, 4)).permute(0, 2, 1, 4, 3)  # [..][row][tile][j][t]
    q = (words.unsqueeze(-1) >> shifts) & 15
    return q.flatten(0, 1).flatten(1)[:N, :K].to(torch.uint8)


def quantize_w4(weight: torch.Tensor, group_size: int = 128, zero_points: bool = False) -> W4Weight:
    """4-bit form of a float weight (N, K), rounded to nearest per group.

    Without zero points a group's scale is its largest magnitude / 7 and the
    codes are 8 + round(w / scale), 1..15; with them the codes 0..15 span the
    group's range, widened to hold 0, which keeps a zero weight exactly zero.
    The scale is stored in the weight's type (fp32 unless that is bf16), and
    the codes are chosen for the stored scale.  A group of zeros gets scale
    0; a weight that is not finite is refused."""
    _check_group(group_size)
    assert weight.dim() == 2 and weight.shape[0] > 0 and weight.shape[1] > 0, "weight must be (N, K)"
    w = weight.detach().float()
    if not bool(torch.isfinite(w).all()):
        raise ValueError("quantize_w4: the weight has values that are not finite")
    N, K = w.shape
    groups = -(-K // group_size)
    pad = groups * group_size - K
    wg = torch.nn.functional.pad(w, (0, pad)).view(N, groups, group_size)
    s_dtype = torch.bfloat16 if weight.dtype == torch.bfloat16 else torch.float32
    if zero_points:
        lo, hi = wg.amin(-1).clamp(max=0.0), wg.amax(-1).clamp(min=0.0)
        scale = (hi / 15 - lo / 15).to(s_dtype)
        zeros = torch.where(scale > 0, (-lo / scale.float()).round(), 0.0).clamp(0, 15)
    else:
        scale = (wg.abs().amax(-1) / 7).to(s_dtype)
        zeros = torch.full((N, groups), 8.0, device=w.device)
    q = torch.where((scale > 0)[..., None], (wg / scale.float()[..., None]).round(), 0.0) + zeros[..., None]
    lowest = 0 if zero_points else 1
    q = q.clamp(lowest, 15).to(torch.uint8).reshape(N, -1)[:, :K]
    return pack_w4(q, scale, zeros.to(torch.uint8) if zero_points else None, group_size)


def dequantize_w4(weight: W4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The (N, K) weight that ``weight`` stands for."""
    K, G = weight.in_features, weight.group_size
    at = torch.arange(K, device=weight.codes.device) // G
    zeros = 8.0 if weight.zeros is None else weight.zeros.float()[:, at]
    return ((unpack_w4(weight).float() - zeros) * weight.scales.float()[:, at]).to(dtype)


class W4Projection:
    """The 4-bit form of one projection of a model, for a decoder.

    ``get()`` quantises the weight when first called, and again, into the
    same tensors, once the weight has been replaced or modified in place.  A
    change that PyTorch does not count (through ``.data``) needs
    ``refresh()``.  A captured graph replays what the tensors hold: it sees a
    change after the next ``get()``.  A weight of another shape, type or
    device gets new tensors; the old ones are kept, since a captured graph
    may still read them, and such a graph does not see the change.  Quantising
    waits for the GPU: it belongs before a capture."""

    __slots__ = ("weight", "group_size", "source", "key", "w4", "kept")

    def __init__(self, weight, group_size: int):
        _check_group(group_size)
        self.weight, self.group_size = weight, group_size  # weight: a callable, the current parameter
        self.source = self.key = self.w4 = None
        self.kept = []
        self.get()

    def get(self) -> W4Weight:
        w = self.weight()
        # the parameter itself is held, so that no other can be taken for it
        if w is not self.source or self.key != (w._version, w.data_ptr(), w.dtype):
            self.refresh()
        return self.w4

    def refresh(self) -> None:
        w = self.weight()
        if w.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"4-bit projections need a float32 or bfloat16 model (got {w.dtype})")
        new = quantize_w4(w, self.group_size)
        old = self.w4
        if old is not None and old.shape == new.shape and old.codes.device == new.codes.device and \
                old.scales.dtype == new.scales.dtype:
            old.codes.copy_(new.codes)
            old.scales.copy_(new.scales)
        else:
            if old is not None:
                self.kept.append(old)
            self.w4 = new
        self.source, self.key = w, (w._version, w.data_ptr(), w.dtype)


_host = None  # the host module's linear_w4, once looked up

_CODE = {torch.float32: nat.M3_F32, torch.bfloat16: nat.M3_BF16}


def linear_w4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
              group_size: int = 128, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ W.T`` for x (M, K) and the 4-bit weight (N, K) given by ``codes``,
    ``scales`` and ``zeros`` as ``W4Weight`` holds them.

    x is fp32 or bf16 with any row stride; the output has ``out_dtype`` (x's
    type by default).  Written for the batches of a decode step, right for
    any M.  Of a bf16 x, up to 16 rows are faster than with an unquantised
    weight, 32 about as fast or faster; beyond that the library's product
    with a bf16 weight is faster, except for the largest weights (50,280 x
    2,560: from 256 rows on).  The codes' products with x must stay within
    fp32's range before the scale; codes, scales and zeros take less than 4 GB
    each.  Inference only: x or scales that ask for a gradient, also a
    forward-mode one, are refused."""
    global _host
    if out_dtype is None:
        if _host is None:
            _host = nat.host_entry("linear_w4")
        y = _host(x, codes, scales, zeros, group_size)
        if y is not None:
            return y
    if group_size not in GROUP_SIZES:
        _check_group(group_size)
    dev = x.get_device() if x.is_cuda else -1
    assert dev >= 0 and x.dim() == 2, "x must be a (M, K) CUDA tensor"
    if nat.wants_gradient(x, scales):
        raise RuntimeError("linear_w4 has no gradient: call it under torch.no_grad() or on detached tensors")
    M, K = x.shape
    N, groups = scales.shape
    dtype = x.dtype
    if out_dtype is None:
        out_dtype = dtype
    x_code, s_code, y_code = _CODE.get(dtype), _CODE.get(scales.dtype), _CODE.get(out_dtype)
    assert x_code is not None and s_code is not None and y_code is not None, \
        f"x, scales and out_dtype must be float32 or bfloat16 (got {dtype}, {scales.dtype}, {out_dtype})"
    assert K > 0 and N > 0, "linear_w4 needs at least one row and one column of weight"
    blocks = ((N + ROWS - 1) // ROWS, (K + TILE - 1) // TILE, ROWS, 16)
    assert codes.shape == blocks and codes.dtype == torch.int32 and codes.is_contiguous(), \
        f"codes must be contiguous int32 {blocks}, got {codes.dtype} {tuple(codes.shape)}"
    assert groups == (K + group_size - 1) // group_size, \
        f"scales must be {(N, -(-K // group_size))}, got {tuple(scales.shape)}"
    assert codes.get_device() == dev and scales.get_device() == dev, f"all tensors must be on {x.device}"
    if scales.is_contiguous():
        s_pitch = groups
    else:
        scales = _rows(scales)
        s_pitch = _pitch(scales)
    z_ptr = z_pitch = 0
    if zeros is not None:
        assert zeros.dtype == torch.uint8 and zeros.shape == (N, groups) and zeros.get_device() == dev, \
            f"zeros must be uint8 {(N, groups)} on {x.device}, got {zeros.dtype} {tuple(zeros.shape)} on {zeros.device}"
        zeros = _rows(zeros)
        z_ptr, z_pitch = zeros.data_ptr(), _pitch(zeros)
    if x.is_contiguous():
        ldx = K
    else:
        if x.stride(1) != 1 and K > 1:
            x = x.contiguous()
        ldx = x.stride(0)
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    if M > 0:
        nat.call("m3_linear_w4", nat.W4_ARGS.pack(
            M, N, K, group_size, x.data_ptr(), ldx, x_code, codes.data_ptr(), scales.data_ptr(), s_pitch, s_code,
            z_ptr, z_pitch, y.data_ptr(), N, y_code), dev)
    return y


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with unit column stride and rows that do not overlap."""
    return t if t.is_contiguous() or (t.stride(1) == 1 and _pitch(t) >= t.shape[1]) else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    """Row stride; of a single row, its length (its stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]
