"""``linear_w4`` against the product in 64 bits of the values that the codes
stand for."""

from __future__ import annotations

import importlib

import pytest
import torch

from src.kernels.linear import linear
from src.kernels.linear_w4 import GROUP_SIZES, W4Weight, dequantize_w4, linear_w4, pack_w4, quantize_w4

pytestmark = pytest.mark.gpu


def make(N, K, G, zeros, s_dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (N, K), generator=g, device="cuda")
    s = (torch.rand(N, -(-K // G), generator=g, device="cuda") + 0.5).to(s_dtype)
    z = torch.randint(0, 16, s.shape, generator=g, device="cuda") if zeros else None
    return pack_w4(q, s, z, G)


def check(y, x, w: W4Weight):
    """|error| <= sums in fp32 + the output's rounding.

    Products are exact.  A group's sum of at most 128 products (three terms
    each for fp32 x) goes through at most 24 tensor-core instructions, each
    an addition of aligned products that may truncate: 2 places of 2^-23
    each.  One fused multiply-add scales and adds it; at most K / 32 groups
    and 16 warps' partial sums follow, half a place each.  All relative to
    the sum of the products' magnitudes."""
    wd = dequantize_w4(w).double()
    ref = x.double() @ wd.t()
    mag = x.double().abs() @ wd.abs().t()
    places = 24 * 2 + (x.shape[1] / 32 + 1 + 16) / 2
    tol = mag * places * 2.0 ** -23 + ref.abs() * torch.finfo(y.dtype).eps / 2 + 1e-30
    assert y.shape == ref.shape
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {(y.double() - ref).abs().max()}"


# one row to beyond the largest tile; every tile count around the 16-row
# blocks, the 128-column tiles and the groups
SHAPES = [(1, 1, 1), (2, 5, 7), (1, 16, 128), (1, 1600, 256), (3, 17, 130), (7, 33, 1111), (8, 100, 257),
          (9, 100, 257), (16, 250, 4096), (17, 500, 640), (32, 129, 300), (33, 129, 300), (64, 1000, 2560),
          (65, 77, 128), (130, 50, 500), (5, 20, 13000), (20, 40, 9000), (64, 33, 5120)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_product(M, N, K, G, dtype):
    for zeros, s_dtype in ((False, torch.float32), (True, torch.bfloat16)):
        w = make(N, K, G, zeros, s_dtype, seed=M + N + K)
        x = torch.randn(M, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K)).to(dtype)
        for out_dtype in (torch.float32, torch.bfloat16):
            y = linear_w4(x, w.codes, w.scales, w.zeros, group_size=G, out_dtype=out_dtype)
            assert y.dtype == out_dtype
            check(y, x, w)


def test_default_output_type_and_linear_dispatch():
    w = quantize_w4(torch.randn(48, 256, device="cuda"))
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(4, 256, device="cuda").to(dtype)
        y = linear_w4(x, w.codes, w.scales)
        assert y.dtype == dtype
        assert torch.equal(linear(x, w), y)


def test_fp32_input_keeps_all_its_bits():
    """One column: y is x times a power of two, exactly."""
    q = torch.full((16, 1), 9, device="cuda")
    w = pack_w4(q, torch.full((16, 1), 0.5, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(200, 1, device="cuda", generator=g) * 10.0 ** torch.randint(-20, 20, (200, 1), device="cuda")
    y = linear_w4(x, w.codes, w.scales)
    assert torch.equal(y, (x * 0.5).expand(200, 16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(dtype):
    w = make(40, 200, 64, True)
    wide = torch.randn(9, 256, device="cuda").to(dtype)
    for x in (wide[:, 8:208], wide[:, 3:203], wide[::2, 1:201], torch.randn(200, 9, device="cuda").to(dtype).t(),
              wide[:1, :200].expand(9, 200), wide[4:5, 7:207]):
        check(linear_w4(x, w.codes, w.scales, w.zeros, group_size=64), x, w)


def test_strided_scales_and_zeros():
    w = make(40, 200, 64, True)
    s, z = torch.zeros(40, 9, device="cuda"), torch.zeros(40, 7, dtype=torch.uint8, device="cuda")
    s[:, 2:6], z[:, 1:5] = w.scales, w.zeros
    x = torch.randn(3, 200, device="cuda")
    check(linear_w4(x, w.codes, s[:, 2:6], z[:, 1:5], group_size=64), x, w)
    check(linear_w4(x, w.codes, w.scales.t().contiguous().t(), w.zeros, group_size=64), x, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_are_not_finite(dtype):
    """As the formula: an infinity times a weight that is not 0 is an
    infinity, times 0 NaN; other rows are untouched."""
    q = torch.tensor([[10, 8], [6, 9]], device="cuda")
    w = pack_w4(q.repeat(8, 1), torch.ones(16, 1, device="cuda"))
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, 1.0], [nan, 1.0], [2.0, 1.0], [-inf, inf]], device="cuda").to(dtype)
    y = linear_w4(x, w.codes, w.scales)
    assert float(y[0, 0]) == inf and float(y[0, 1]) == -inf
    assert bool(y[1].isnan().all())
    assert float(y[2, 0]) == 4.0 and float(y[2, 1]) == -3.0
    assert bool(y[3, 0].isnan()) and float(y[3, 1]) == inf


def test_largest_group_sums():
    """Inputs up to a thousandth of fp32's range."""
    w = make(16, 128, 128, False)
    x = torch.full((2, 128), 1e35, device="cuda")
    x[1, ::2] = -1e35
    check(linear_w4(x, w.codes, w.scales), x, w)


def test_no_rows():
    w = make(16, 128, 128, False)
    y = linear_w4(torch.empty(0, 128, device="cuda"), w.codes, w.scales)
    assert y.shape == (0, 16)


def test_same_bits_on_every_run_and_stream():
    w = make(500, 1000, 32, True)
    x = torch.randn(5, 1000, device="cuda")
    y = linear_w4(x, w.codes, w.scales, w.zeros, group_size=32)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append([linear_w4(x, w.codes, w.scales, w.zeros, group_size=32) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, y) for run in got for a in run)


def test_weight_written_just_before():
    """The launch may start while the kernel before it runs: it must not read
    the weight early."""
    x = torch.randn(2, 2048, device="cuda")
    w = [make(4096, 2048, 128, True, seed=i) for i in range(2)]
    buf = W4Weight(*(t.clone() if isinstance(t, torch.Tensor) else t for t in w[0]))
    want = [linear_w4(x, v.codes, v.scales, v.zeros) for v in w]
    for i in (1, 0, 1, 0):
        buf.scales.copy_(w[i].scales), buf.zeros.copy_(w[i].zeros), buf.codes.copy_(w[i].codes)
        assert torch.equal(linear_w4(x, buf.codes, buf.scales, buf.zeros), want[i])


def test_captured():
    w = make(300, 640, 64, True)
    x = torch.randn(3, 640, device="cuda")
    linear_w4(x, w.codes, w.scales, w.zeros, group_size=64)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(linear_w4(x, w.codes, w.scales, w.zeros, group_size=64))
        graphs.append(g)
    x.copy_(torch.randn(3, 640, device="cuda"))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for y in outs:
        check(y, x, w)


def test_refusals():
    w = make(40, 200, 64, True)
    x = torch.randn(3, 200, device="cuda")
    ok = dict(group_size=64)
    with pytest.raises(AssertionError):
        linear_w4(x.half(), w.codes, w.scales, **ok)
    with pytest.raises(AssertionError):
        linear_w4(x[:, :100], w.codes, w.scales, **ok)
    with pytest.raises(AssertionError):
        linear_w4(x, w.codes, w.scales, w.zeros, group_size=128)
    with pytest.raises(AssertionError):
        linear_w4(x, w.codes.transpose(0, 1), w.scales, **ok)
    with pytest.raises(AssertionError):
        linear_w4(x, w.codes, w.scales, w.zeros.int(), **ok)
    with pytest.raises(AssertionError):
        linear_w4(x, w.codes.cpu(), w.scales, **ok)
    with pytest.raises(AssertionError):
        linear_w4(x[0], w.codes, w.scales, **ok)
    with pytest.raises(RuntimeError):
        linear_w4(x.requires_grad_(), w.codes, w.scales, **ok)
    with torch.no_grad():
        linear_w4(x, w.codes, w.scales, **ok)


def test_host_module_and_python_path_agree(monkeypatch):
    """The host module serves the ordinary call and leaves the others."""
    from src import _native as nat
    mod = importlib.import_module("src.kernels.linear_w4")
    host = nat.host_entry("linear_w4")
    assert host is not nat._no_host, "lib/m3_host.so is not built"
    w = make(100, 300, 64, True)
    x = torch.randn(5, 300, device="cuda")
    y = host(x, w.codes, w.scales, w.zeros, 64)
    assert y is not None and torch.equal(host(x, w.codes, w.scales, None, 64),
                                         linear_w4(x, w.codes, w.scales, group_size=64))
    for args in ((x.t().contiguous().t(), w.codes, w.scales, w.zeros, 64), (x, w.codes, w.scales, w.zeros, 128),
                 (x.half(), w.codes, w.scales, w.zeros, 64), (x.cpu(), w.codes, w.scales, w.zeros, 64),
                 (x, w.codes[:1], w.scales, w.zeros, 64), (x, w.codes, w.scales, w.zeros.int(), 64),
                 (x[:0], w.codes, w.scales, w.zeros, 64), (x.clone().requires_grad_(), w.codes, w.scales, w.zeros, 64),
                 (x, w.codes, None, w.zeros, 64), (x, w.codes, w.scales, w.zeros)):
        assert host(*args) is None
    monkeypatch.setattr(mod, "_host", nat._no_host)
    assert torch.equal(linear_w4(x, w.codes, w.scales, w.zeros, group_size=64), y)


# more than 32 batch rows of a weight large enough for the tensor memory path:
# ragged rows and columns, one and several items a CTA, split K
MANY = [(40, 9000, 1200), (64, 50000, 264), (33, 9440, 2048), (65, 4225, 1160), (130, 20001, 136), (300, 1000, 2560),
        (513, 2048, 520), (2200, 17, 8200), (128, 2048, 4096), (1000, 9440, 384)]


@pytest.mark.parametrize("M,N,K", MANY)
@pytest.mark.parametrize("G", GROUP_SIZES)
def test_many_rows(M, N, K, G):
    from src import _native as nat
    for zeros, s_dtype in ((False, torch.float32), (True, torch.bfloat16)):
        w = make(N, K, G, zeros, s_dtype, seed=M + N + K)
        g = torch.Generator(device="cuda").manual_seed(K)
        x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
        for out_dtype in (torch.float32, torch.bfloat16):
            check(linear_w4(x, w.codes, w.scales, w.zeros, group_size=G, out_dtype=out_dtype), x, w)
    assert nat.load().m3_device_error(0) == 0


def test_many_rows_of_other_layouts():
    """Strided rows behind whose end NaN stands; rows off 16 bytes, of an odd
    length or the same row (not read by TMA); fp32."""
    w = make(9440, 1160, 64, True)
    wide = torch.full((200, 1280), float("nan"), device="cuda").bfloat16()
    wide[:, 8:1168] = torch.randn(200, 1160, device="cuda")
    shifted = torch.full((200, 1280), float("nan"), device="cuda").bfloat16()
    shifted[:, 3:1163] = wide[:, 8:1168]
    for x in (wide[:, 8:1168], wide[::2, 8:1168], shifted[:, 3:1163], wide[:1, 8:1168].expand(100, 1160),
              wide[:100, 8:1168].float()):
        check(linear_w4(x, w.codes, w.scales, w.zeros, group_size=64), x, w)
    w = make(9440, 1111, 128, False)
    x = torch.randn(70, 1111, device="cuda").bfloat16()
    check(linear_w4(x, w.codes, w.scales), x, w)


def test_many_rows_not_finite():
    """A row of x or of the scales that is not finite stays in its row or
    column, also where the last rows and groups are not whole."""
    w = make(9001, 1032, 128, False)
    x = torch.randn(130, 1032, device="cuda").bfloat16()
    want = linear_w4(x, w.codes, w.scales)
    x[7], x[129, 0] = float("nan"), float("inf")
    scales = w.scales.clone()
    scales[5], scales[9000] = float("inf"), float("nan")
    y = linear_w4(x, w.codes, scales)
    rows, cols = torch.ones(130, dtype=torch.bool, device="cuda"), torch.ones(9001, dtype=torch.bool, device="cuda")
    rows[7] = rows[129] = False
    cols[5] = cols[9000] = False
    assert torch.equal(y[rows][:, cols], want[rows][:, cols])
    assert bool(y[7].isnan().all()) and not bool(y[129].isfinite().any())
    assert bool(y[:, 9000].isnan().all()) and not bool(y[:, 5].isfinite().any())


def test_many_rows_same_bits_streams_and_graphs():
    w = [make(9440, 1032, 32, True, seed=i) for i in range(2)]
    x = torch.randn(100, 1032, device="cuda").bfloat16()
    want = [linear_w4(x, v.codes, v.scales, v.zeros, group_size=32) for v in w]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got += [(i, linear_w4(x, w[i].codes, w[i].scales, w[i].zeros, group_size=32)) for i in (0, 1, 0, 1)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    graphs, outs = [], []
    for v in w:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(linear_w4(x, v.codes, v.scales, v.zeros, group_size=32))
        graphs.append(graph)
    x.copy_(torch.randn(100, 1032, device="cuda"))
    for graph, s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for y, v in zip(outs, w):
        check(y, x, v)


def test_many_rows_weight_written_just_before():
    x = torch.randn(64, 2048, device="cuda").bfloat16()
    w = [make(9440, 2048, 128, True, seed=i) for i in range(2)]
    buf = W4Weight(*(t.clone() if isinstance(t, torch.Tensor) else t for t in w[0]))
    want = [linear_w4(x, v.codes, v.scales, v.zeros) for v in w]
    for i in (1, 0, 1, 0):
        buf.scales.copy_(w[i].scales), buf.zeros.copy_(w[i].zeros), buf.codes.copy_(w[i].codes)
        assert torch.equal(linear_w4(x, buf.codes, buf.scales, buf.zeros), want[i])
