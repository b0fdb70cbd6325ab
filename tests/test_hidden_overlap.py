"""Outputs that share memory with what other workgroups still read are refused, and those that
lie beside it are not, on CPU tensors: no GPU is used (a call that goes on to the device says
that x is on the CPU)."""
import itertools

import pytest
import torch
from test_head_args import _Device

import thrml_hip as th
from thrml_hip import hidden

B = torch.bfloat16
TAKEN = "x is on cpu"


def _gated(x, wg, wu, out):
    with pytest.raises(th.ThrmlError) as e:
        th.gated_linear(_Device(), x, wg, wu, out=out)
    return str(e.value)


def _dropout(x, out, residual=None):
    with pytest.raises(th.ThrmlError) as e:
        th.dropout(_Device(), x, th.RngKey(1), 0.5, residual=residual, out=out)
    return str(e.value)


def test_gated_linear():
    buf = torch.zeros(4096, dtype=B)
    rows = lambda at, n, stride, q: buf[at:].as_strided((n, q), (stride, 1))  # noqa: E731
    x, w = rows(0, 9, 64, 64), torch.zeros(64, 64, dtype=B)
    assert "h must not be x or a weight" in _gated(x[:8], w, w, x[1:])      # begins inside x
    assert "h must not be x or a weight" in _gated(x[1:], w, w, x[:8])
    assert "h must not be x or a weight" in _gated(x, w, w, x)
    inside = torch.zeros(100, 64, dtype=B)
    assert "h must not be x or a weight" in _gated(x[:8], inside[:64], w, inside[60:68])
    assert "h must not be x or a weight" in _gated(x[:8], w, inside[20:84], inside[14:22])
    assert TAKEN in _gated(x[:8], inside[:64], w, inside[64:72])            # behind the weight
    # columns of one buffer, side by side
    wide = torch.zeros(8, 128, dtype=B)
    assert TAKEN in _gated(wide[:, :64], w, w, wide[:, 64:])
    assert TAKEN in _gated(wide[:, 64:], w, w, wide[:, :64])
    assert "h must not be x or a weight" in _gated(wide[:, :64], w, w, wide[:, 63:127])
    # x's rows are every second one of out's buffer
    two = torch.zeros(16, 64, dtype=B)
    assert TAKEN in _gated(two[::2], w, w, two[1::2])
    assert "h must not be x or a weight" in _gated(two[::2], w, w, two[:8])
    # a copied operand is another memory
    assert TAKEN in _gated(two[:8].t().contiguous().t(), w, w, two[:8])


def test_dropout():
    buf = torch.zeros(600)
    x = buf.as_strided((5, 7), (20, 1))
    assert TAKEN in _dropout(x, x) and TAKEN in _dropout(buf[300:].as_strided((5, 7), (20, 1)), x, x)
    assert "out may be x or residual" in _dropout(x, buf.as_strided((5, 7), (7, 1)))      # x with another stride
    assert "out may be x or residual" in _dropout(x, buf[1:].as_strided((5, 7), (20, 1)))
    assert "out may be x or residual" in _dropout(buf[300:].as_strided((5, 7), (20, 1)), x, buf[40:].as_strided((5, 7), (7, 1)))
    assert TAKEN in _dropout(x, buf[7:].as_strided((5, 7), (20, 1)))
    assert "out may be x or residual" in _dropout(buf[:7].expand(5, 7), buf.as_strided((5, 7), (7, 1)))
    assert TAKEN in _dropout(buf[:7].expand(5, 7), buf[7:].as_strided((5, 7), (7, 1)))
    # one row: whatever its stride says
    assert TAKEN in _dropout(buf.as_strided((1, 7), (50, 1)), buf.as_strided((1, 7), (7, 1)))
    assert TAKEN in _dropout(x[:0], x[:0])
    # the key's seed
    words = torch.zeros(64, dtype=torch.int64)
    y = words.view(torch.float32).view(2, 64)
    with pytest.raises(th.ThrmlError, match="out must not hold the key"):
        th.dropout(_Device(), torch.zeros(2, 64), words[40:41], 0.5, out=y)


def test_every_small_layout():
    """against the sets of bytes"""
    buf = torch.zeros(64, dtype=torch.uint8)

    def cells(at, rows, q, stride):
        return {at + i * stride + j for i in range(rows) for j in range(q)}

    layouts = [(at, rows, q, stride) for at in (0, 1, 5, 11) for rows in (1, 2, 4) for q in (1, 3) for stride in (0, 3, 4, 7)]
    for a, b in itertools.product(layouts, layouts):
        ta, tb = (buf[at:].as_strided((rows, q), (stride, 1)) for at, rows, q, stride in (a, b))
        assert hidden._overlap(ta, tb) == bool(cells(*a) & cells(*b)), (a, b)
