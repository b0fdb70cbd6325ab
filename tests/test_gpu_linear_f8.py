"""linear_f8 against its definition in 64 bits (hidden_reference.py): types, sizes from one
on, inner sizes that end inside a block, strides, every kind of tile and splits of the
reduction, extreme scales, infinities, other streams, graphs."""
import math

import hidden_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(t, pad=0, shift=0):
    """t on the device as rows of a wider buffer of NaN, from element `shift` on"""
    rows, q = t.shape
    size = rows * (q + pad) + shift + 1
    if t.dtype == F8:
        wide = torch.full((size,), 0x7F, dtype=torch.uint8, device="cuda").view(F8)
    else:
        wide = torch.full((size,), math.nan, dtype=t.dtype, device="cuda")
    view = wide[shift:shift + rows * (q + pad)].view(rows, q + pad)[:, :q]
    view.copy_(t)
    return view


def _inputs(rows, k, q, dtype, pad=0, shift=0, seed=0):
    g = _gen(seed + rows * 100 + k * 3 + q)
    x = torch.randn(rows, k, generator=g) * (1 + 20 * (torch.rand(k, generator=g) < 0.02))
    w = (torch.randn(q, k, generator=g) * 100).clamp(-448, 448).to(F8)
    ws = (0.5 + torch.rand(-(-q // 128), -(-k // 128), generator=g)) * (0.01 / math.sqrt(k))
    return _rows(x.to(dtype), pad, shift), _rows(w, pad, shift), ws.cuda(), torch.randn(q, generator=g).cuda()


def _check(device, x, w, ws, bias, out=None):
    got = th.linear_f8(device, x, w, ws, bias=bias, out_dtype=out)
    assert got.dtype == (out or x.dtype) and got.is_contiguous()
    ref.close(got.cpu(), *ref.linear_f8(x, w, ws, bias, got.dtype), "linear_f8")
    return got


SIZES = [
    # rows, k, q
    (1, 1, 1), (1, 128, 16), (2, 127, 17), (3, 129, 33), (1, 1000, 300), (17, 16, 129), (33, 272, 501), (70, 400, 640),
    (130, 640, 257), (1, 4096, 130), (257, 136, 260), (300, 2048, 1000),
]


@pytest.mark.parametrize("dtype,out", [(BF16, None), (F16, None), (F32, None), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("rows,k,q", SIZES)
def test_sizes(device, rows, k, q, dtype, out):
    log_case(f"linear_f8 {rows} {k} {q} {dtype} {out}")
    x, w, ws, bias = _inputs(rows, k, q, dtype)
    _check(device, x, w, ws, bias, out)
    _check(device, x, w, ws, None, out)


@pytest.mark.parametrize("pad,shift", [(16, 0), (1, 0), (0, 3), (5, 16)])
@pytest.mark.parametrize("rows,k,q", [(3, 144, 40), (70, 256, 130), (300, 320, 600)])
def test_rows_of_wider_buffers(device, rows, k, q, pad, shift):
    """(NaN between the rows and behind the last)"""
    log_case(f"linear_f8 {rows} {k} {q} pad {pad} shift {shift}")
    _check(device, *_inputs(rows, k, q, BF16, pad, shift))
    _check(device, *_inputs(rows, k, q, F32, pad, shift))


@pytest.mark.parametrize("rows,k,q", [(600, 1040, 1100), (1030, 512, 2300)])
def test_large_tiles(device, rows, k, q):
    log_case(f"linear_f8 {rows} {k} {q}")
    for dtype in (BF16, F32):
        _check(device, *_inputs(rows, k, q, dtype))


@pytest.mark.parametrize("size", [1e-38, 2e-41, 1e30, 0.0])
def test_extreme_scales(device, size):
    """rows of zeros, of values whose scale is at its least, and of large ones"""
    x, w, ws, _ = _inputs(5, 300, 40, F32)
    x = x * 0.01
    x[1] *= size
    x[3, 128:] *= size
    a, s = ref.quantised(x)
    assert s.min() >= 2.0**-126 and a.abs().max() <= 448
    got = _check(device, x, w, ws, None)
    if size == 0.0:
        assert not got[1].any()


def test_not_finite(device):
    x, w, ws, bias = _inputs(40, 300, 200, BF16)
    want = th.linear_f8(device, x, w, ws, bias=bias)
    bad = x.clone()
    bad[2, 5], bad[7, 299], bad[39, 128] = math.inf, math.nan, -math.inf
    got = th.linear_f8(device, bad, w, ws, bias=bias)
    rows = torch.tensor([2, 7, 39], device="cuda")
    assert got[rows].isnan().all()
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert torch.equal(got[rest], want[rest])


def test_other_strides(device):
    x, w, ws, bias = _inputs(9, 256, 200, BF16)
    want = th.linear_f8(device, x, w, ws, bias=bias)
    assert torch.equal(th.linear_f8(device, x, w.view(torch.uint8).t().contiguous().t().view(F8), ws, bias=bias), want)
    assert torch.equal(th.linear_f8(device, x, w, ws.t().contiguous().t(), bias=bias), want)
    wide = torch.full((2, 5), math.nan, device="cuda")
    wide[:, :2] = ws
    assert torch.equal(th.linear_f8(device, x, w, wide[:, :2], bias=bias), want)
    assert torch.equal(th.linear_f8(device, x.t().contiguous().t(), w, ws, bias=bias), want)
    assert torch.equal(th.linear_f8(device, x[:1].expand(9, 256), w, ws, bias=bias), want[:1].expand(9, 200))
    assert th.linear_f8(device, x[:0], w, ws).shape == (0, 200)
    assert torch.equal(th.linear_f8(device, x, w[:1], ws[:1], bias=bias[:1]), want[:, :1])


def test_streams_and_graphs(device):
    dev = th.Device(0)
    side = torch.cuda.Stream()
    dev.set_stream(side.cuda_stream)
    cases = [(3, 300, 200), (260, 256, 512)]
    ins = [_inputs(*c, BF16) for c in cases]
    torch.cuda.synchronize()
    for x, w, ws, b in ins:  # from torch's default stream: ordered with the device's
        y = th.linear_f8(dev, x * 1.0, w, ws, bias=b) * 1.0
        assert torch.equal(y, th.linear_f8(device, x, w, ws, bias=b))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, w, ws, b in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(th.linear_f8(dev, x, w, ws, bias=b))
        graphs.append(graph)
    for turn in range(3):
        for c, (x, w, _, _) in zip(cases, ins):
            new = _inputs(*c, BF16, seed=turn + 1)
            x.copy_(new[0])
            w.copy_(new[1])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for graph in graphs:
                graph.replay()
            eager = [th.linear_f8(dev, x, w, ws, bias=b) for x, w, ws, b in ins]
            for graph in reversed(graphs):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, eager))
    del graphs
    torch.cuda.synchronize()
    dev.close()


@pytest.mark.parametrize("stride", [(1 << 23) - 16, 1 << 23])
def test_rows_far_apart(device, stride):
    """weights whose offsets pass 32 bits, at the largest stride that tiles read as it lies and
    at the first that is copied"""
    rows, k, q = 100, 144, 600
    x, w, ws, bias = _inputs(rows, k, q, BF16)
    wide = torch.empty((q - 1) * stride + k, dtype=torch.uint8, device="cuda").view(F8)
    far = wide.as_strided((q, k), (stride, 1))
    far.view(torch.uint8).copy_(w.view(torch.uint8))
    want = th.linear_f8(device, x, w, ws, bias=bias)
    assert torch.equal(th.linear_f8(device, x, far, ws, bias=bias), want)
    ref.close(th.linear_f8(device, x[:5], far, ws, bias=bias).cpu(), *ref.linear_f8(x[:5], w, ws, bias, BF16), "few rows")


def test_few_rows_of_every_count(device):
    """rows quantised by the workgroups themselves, or read by the kernel for unaligned weights"""
    for k in (256, 257):
        x, w, ws, bias = _inputs(65, k, 200, F16)
        for rows in (1, 2, 15, 16, 17, 31, 32, 33, 48, 49, 64, 65):
            got = th.linear_f8(device, x[:rows], w, ws, bias=bias)
            ref.close(got.cpu(), *ref.linear_f8(x[:rows], w, ws, bias, F16), f"{rows} rows of {k}")
