"""Which outputs ``process_logits`` takes for apart from its logits."""

from __future__ import annotations

import random

import torch

from src.kernels.logits import _overlap


def _bytes(t: torch.Tensor) -> set:
    rows, cols = ([i * s for i in range(n)] for n, s in zip(t.shape, t.stride()))
    return {t.data_ptr() + (r + c) * t.element_size() + b for r in rows for c in cols for b in range(t.element_size())}


def test_columns_of_one_buffer():
    buf = torch.zeros(4, 64)
    half = buf.view(torch.bfloat16)
    assert not _overlap(buf[:, :32], buf[:, 32:]) and not _overlap(buf[:, 32:], buf[:, :32])
    assert not _overlap(buf[:, 8:40], half[:, 80:112]) and not _overlap(half[:, :16], buf[:, 8:24])
    assert not _overlap(buf[0::2, :], buf[1::2, :])
    assert _overlap(buf[:, :33], buf[:, 31:]) and _overlap(buf, buf) and _overlap(buf[:, 40:], buf[:, 30:54])
    assert _overlap(half[:, :18], buf[:, 8:26]) and _overlap(buf[:1, :9], buf[:1, 8:17])
    assert not _overlap(buf[:1, :8], buf[:1, 8:16])
    assert not _overlap(buf, torch.zeros(4, 64)) and not _overlap(buf[:0], buf[:0])


def test_never_misses_shared_memory():
    """Against the sets of bytes, for all kinds of strides; exact for equal
    distances of rows."""
    rng = random.Random(5)
    buf = torch.zeros(4000, dtype=torch.uint8)
    apart = 0
    for _ in range(4000):
        B, V = rng.randint(1, 5), rng.randint(1, 12)
        pitch = rng.choice([0, V, V + rng.randint(0, 20)])
        ts = []
        for _ in range(2):
            typed = buf.view(rng.choice([torch.float32, torch.bfloat16]))
            p = pitch * (4 // typed.element_size()) if rng.random() < 0.8 else rng.randint(0, 30)
            ts.append(typed.as_strided((B, V), (p, 1 if rng.random() < 0.9 else 2), rng.randint(0, 150)))
        a, b = ts
        shared = bool(_bytes(a) & _bytes(b))
        assert _overlap(a, b) or not shared, (a.shape, a.stride(), b.stride(), a.dtype, b.dtype)
        apart += not _overlap(a, b) and min(b.data_ptr(), a.data_ptr()) + (B - 1) * pitch * 4 >= max(
            a.data_ptr(), b.data_ptr()) > 0
    assert apart > 50  # interleaved rows among them
