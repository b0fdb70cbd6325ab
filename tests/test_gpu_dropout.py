"""dropout against the key's stream as the CPU oracle gives it: the words of
chacha_block(seed_from_u64(key)), halves compared with the border; types, residuals, rows
of wider buffers, parts of a batch, in place, the gradient's way back, keys on the device."""
import ctypes
import math

import numpy as np
import pyoracle as orc
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _bits(seed, first, count):
    """half words first .. first + count - 1 of the stream"""
    b0, b1 = first // 32, (first + count + 31) // 32
    words = np.concatenate([orc.chacha_block(orc.seed_from_u64(seed), b) for b in range(b0, b1)]).astype("<u4")
    return torch.from_numpy(words.view("<u2").astype(np.int32)[first - 32 * b0:][:count]).cuda()


def _want(x, seed, p, residual, first_row):
    """the same steps in f32, rounded once (exact up to nothing: compared bit for bit)"""
    rows, cols = x.shape
    border = round(65536 * p)
    kept = (_bits(seed, first_row * cols, rows * cols) >= border).view(rows, cols)
    scale = torch.tensor(65536.0 / (65536 - border) if border < 65536 else 0.0, dtype=torch.float32, device="cuda")
    y = torch.where(kept, x.float() * scale, torch.zeros((), device="cuda"))
    return ((residual.float() + y) if residual is not None else y).to(x.dtype)


def _rows(t, pad, shift):
    rows, q = t.shape
    wide = torch.full((rows * (q + pad) + shift + 1,), 7.0, dtype=t.dtype, device="cuda")
    view = wide[shift:shift + rows * (q + pad)].view(rows, q + pad)[:, :q]
    view.copy_(t)
    return view


def _randn(seed, rows, cols, dtype):
    return torch.randn(rows, cols, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


CASES = [
    # rows, cols, first_row, pad, shift
    (1, 1, 0, 0, 0), (1, 1, 31, 0, 0), (3, 5, 0, 0, 1), (2, 31, 7, 2, 0), (5, 33, 1000003, 0, 0), (9, 96, 0, 8, 0),
    (1, 2048, 0, 0, 0), (4, 2047, 3, 0, 0), (2, 2049, 5, 7, 3), (70, 130, 0, 1, 0), (1, 20000, 17, 0, 5),
]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols,first,pad,shift", CASES)
def test_bits(device, rows, cols, first, pad, shift, dtype, residual):
    log_case(f"dropout {rows} {cols} {first} {pad} {shift} {dtype} {residual}")
    x = _rows(_randn(rows + cols, rows, cols, dtype), pad, shift)
    res = _rows(_randn(rows * cols + 1, rows, cols, dtype), pad, shift) if residual else None
    for p in (0.0, 0.1, 0.5, 1 / 3, 1.0):
        seed = 0x9E3779B97F4A7C15 ^ rows * cols
        got = th.dropout(device, x, th.RngKey(seed), p, residual=res, first_row=first)
        assert got.dtype == dtype and torch.equal(got, _want(x, seed, p, res, first)), p


def test_share_of_kept_units(device):
    x = torch.ones(1000, 1000, device="cuda")
    for p in (0.1, 0.5, 0.9):
        y = th.dropout(device, x, th.RngKey(3), p)
        border = round(65536 * p)
        kept = float((y != 0).double().mean())
        q = 1 - border / 65536
        assert abs(kept - q) < 5 * math.sqrt(q * (1 - q) / 1e6)
        assert (y[y != 0] == torch.tensor(65536 / (65536 - border), dtype=F32, device="cuda")).all()
    other = th.dropout(device, x, th.RngKey(4), 0.5) != 0
    same = float((other == (th.dropout(device, x, th.RngKey(3), 0.5) != 0)).double().mean())
    assert abs(same - 0.5) < 5 * 0.5e-3


def test_parts_of_a_batch(device):
    x = _randn(1, 37, 77, BF16)
    whole = th.dropout(device, x, th.RngKey(8), 0.4)
    parts = [th.dropout(device, x[i:j], th.RngKey(8), 0.4, first_row=i) for i, j in ((0, 1), (1, 20), (20, 37))]
    assert torch.equal(torch.cat(parts), whole)


def test_dropped_units_count_as_zero(device):
    x = torch.full((4, 512), math.nan, device="cuda")
    x[1], x[2] = math.inf, -math.inf
    y = th.dropout(device, x, th.RngKey(5), 0.5)
    kept = th.dropout(device, torch.ones_like(x), th.RngKey(5), 0.5) != 0
    assert (y[~kept] == 0).all() and torch.equal(y[kept].nan_to_num(3.0), x[kept].nan_to_num(3.0))
    assert not th.dropout(device, x, th.RngKey(5), 1.0).any()


def test_in_place_and_out(device):
    for pad in (0, 3):
        x, res = _rows(_randn(2, 50, 130, F16), pad, 0), _rows(_randn(3, 50, 130, F16), pad, 0)
        want = th.dropout(device, x, th.RngKey(6), 0.3, residual=res)
        wide = torch.full((50, 140), 2.0, dtype=F16, device="cuda")
        assert torch.equal(th.dropout(device, x, th.RngKey(6), 0.3, residual=res, out=wide[:, :130]), want)
        assert (wide[:, 130:] == 2.0).all()
        a, b = x.clone(), res.clone()
        assert th.dropout(device, a, th.RngKey(6), 0.3, residual=b, out=a) is a and torch.equal(a, want)
        a = x.clone()
        assert th.dropout(device, a, th.RngKey(6), 0.3, residual=b, out=b) is b and torch.equal(b, want)
    assert th.dropout(device, x[:0], th.RngKey(6), 0.3).shape == (0, 130)
    assert th.dropout(device, x[:, :0], th.RngKey(6), 0.3).shape == (50, 0)
    t = _randn(4, 130, 50, F16).t()
    assert torch.equal(th.dropout(device, t, th.RngKey(6), 0.3), th.dropout(device, t.contiguous(), th.RngKey(6), 0.3))


def test_gradient(device):
    """of sum(g y) in x: g where kept, scaled; against differences, which are exact up to
    rounding for what is linear"""
    x, g = _randn(1, 30, 70, F32), _randn(2, 30, 70, F32)
    dx = th.dropout(device, g, th.RngKey(9), 0.25, first_row=4)
    way = _randn(3, 30, 70, F32)
    f = lambda t: (g.double() * th.dropout(device, x + t * way, th.RngKey(9), 0.25, first_row=4).double()).sum()  # noqa: E731
    got, want = float((dx.double() * way.double()).sum()), float(f(1.0) - f(-1.0)) / 2
    # each y is off by a rounding of x + way and one of the product: 2 half steps of |g (|x| + |way|) scale|
    assert abs(got - want) < 4 * 2.0**-24 * float((g.abs() * (x.abs() + way.abs())).double().sum() * 4 / 3)


def test_key_on_the_device(device):
    x = _randn(1, 20, 300, BF16)
    for seed in (0, 5, 2**63 - 1, -1, -2**63):
        key = torch.tensor([seed], dtype=torch.int64, device="cuda")
        assert torch.equal(th.dropout(device, x, key, 0.5), th.dropout(device, x, th.RngKey(seed % 2**64), 0.5))


def test_captured_with_a_key_that_changes(device):
    dev = th.Device(0)
    side = torch.cuda.Stream()
    dev.set_stream(side.cuda_stream)
    x, key = _randn(1, 40, 130, BF16), torch.zeros(1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        th.dropout(dev, x, key, 0.5)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = th.dropout(dev, x, key, 0.5)
        back = th.dropout(dev, y, key, 0.5)
    for seed in (3, 4, 3):
        key.fill_(seed)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = _want(x, seed, 0.5, None, 0)
        assert torch.equal(y, want) and torch.equal(back, _want(want, seed, 0.5, None, 0))
    del graph
    torch.cuda.synchronize()
    dev.close()


def test_far_blocks(device):
    """block counters near 2^32, where a row's first unit is the last of the stream's range"""
    cols = 4096
    last = 2**37 // cols - 3
    x = _randn(1, 3, cols, F32)
    got = th.dropout(device, x, th.RngKey(11), 0.5, first_row=last)
    assert torch.equal(got, _want(x, 11, 0.5, None, last))
    with pytest.raises(th.ThrmlError, match="at most 2\\^37"):
        th.dropout(device, x, th.RngKey(11), 0.5, first_row=last + 1)


def test_more_units_than_32_bits(device):
    """rows whose units lie 2^32 elements into their buffer"""
    rows, cols, stride = 3, 200, (1 << 31) + 64
    wide = torch.empty(2 * stride + cols, dtype=F16, device="cuda")
    x = wide.as_strided((rows, cols), (stride, 1))
    x.copy_(_randn(1, rows, cols, F16))
    assert torch.equal(th.dropout(device, x, th.RngKey(1), 0.5), th.dropout(device, x.contiguous(), th.RngKey(1), 0.5))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 33), (3, 7), (5, 700), (2, 2049)])
def test_writes_nothing_else(device, rows, cols, dtype):
    """what lies in front of the result, behind it and between its rows stays as it was"""
    for pad in (0, 5):
        x = _randn(3, rows, cols, dtype)
        wide = torch.full((4096 + rows * (cols + pad) + 8192,), 3.0, dtype=dtype, device="cuda")
        out = wide[4096:4096 + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        th.dropout(device, x, th.RngKey(2), 0.5, out=out)
        assert torch.equal(out, _want(x, 2, 0.5, None, 0))
        out.fill_(3.0)
        assert (wide == 3.0).all()
