"""Operators of a learned head's hidden block, on torch tensors of the device (no
counterpart in the reference):

  gated_linear       hidden units act(x @ w_gate.T) * (x @ w_up.T)
  gated_linear_grad  the gradients of a loss in x and both weights
  dropout            units kept or zeroed by the bits of a key
  linear_f8          a product in 8-bit floating point with a scale for each block

Streams, graphs and tensors that require a gradient are as in `head`: calls queue their
kernels on the device's stream, in order with torch's current one, and torch's gradients
do not go through them (gated_linear_grad gives the gradients).
"""
import struct

import numpy as np

from . import _lib, head
from ._lib import load
from .head import _matrix, _on_device, _out, _refuse, _run

_PACK = struct.Struct("@PiiQIIqPqPq").pack  # thrml_gated
ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU}
_NAMES = ("x", "w_gate", "w_up")


def _halves():
    """The 16-bit types."""
    if head.torch is None:
        head._setup()
    return head._FLOATS[1:]


def _layout(t):
    """(rows, bytes from one row to the next, bytes of a row) of a matrix with contiguous rows"""
    rows, cols = t.shape
    size = t.element_size()
    return (rows, t.stride(0) * size, cols * size) if rows > 1 and t.stride(0) else (min(rows, 1), cols * size, cols * size)


def _overlap(a, b):
    """Whether two matrices with contiguous rows share memory: rows of one may lie between
    those of the other."""
    (ra, sa, la), (rb, sb, lb) = _layout(a), _layout(b)
    d = b.data_ptr() - a.data_ptr()
    if not (ra and rb and la and lb) or d >= (ra - 1) * sa + la or -d >= (rb - 1) * sb + lb:
        return False
    if sa == sb or ra == 1 or rb == 1:  # rows i of a and j of b: d - la < (i - j) s < d + lb
        s = sb if ra == 1 else sa
        least = max((d - la) // s + 1, 1 - rb)
        return least < ra and least * s < d + lb
    if ra > rb:
        ra, sa, la, rb, sb, lb, d = rb, sb, lb, ra, sa, la, -d
    # row i of a and j of b share bytes where i sa - d - lb < j sb < i sa - d + la
    at = np.arange(ra, dtype=np.int64) * sa - d
    first = np.maximum((at - lb) // sb + 1, 0)
    return bool(((first < rb) & (first * sb < at + la)).any())


def _gated(x, w_gate, w_up, activation):
    """(the C descriptor, the tensors that it points into, rows, k, n)"""
    types = _halves()
    x, xs = _matrix("x", x, types)
    rows, k = x.shape
    same = (x.dtype,)
    w_gate, gs = _matrix("w_gate", w_gate, same, None, k)
    n = w_gate.shape[0]
    w_up, us = _matrix("w_up", w_up, same, n, k)
    if k == 0 or n == 0:
        _refuse("w_gate must have at least one row and column")
    act = ACTIVATIONS.get(activation)
    if act is None:
        _refuse(f"activation must be one of {', '.join(ACTIVATIONS)}")
    d = _PACK(x.data_ptr(), head._TYPES[x.dtype], act, rows, k, n, xs if rows > 1 else k, w_gate.data_ptr(),
              gs if n > 1 else k, w_up.data_ptr(), us if n > 1 else k)
    return d, (x, w_gate, w_up), rows, k, n


def gated_linear(device, x, w_gate, w_up, activation="silu", save=False, out=None):
    """Hidden units h [rows, n] = act(x @ w_gate.T) * (x @ w_up.T) of features x [rows, k]
    and weights [n, k], all bfloat16 or all float16; sums, activation and product in
    float32, rounded once.  activation: "silu", "gelu" (of the error function) or "relu".
    With save, (h, gate, up): also both products in float32, for gated_linear_grad.  out: a
    tensor for h, which shares no memory with x and the weights.

    Operands whose rows are not whole 16-byte pieces (k not a multiple of 8, a view that starts
    or steps elsewhere, weights of different strides) are copied first where x has more than 32
    rows, and else read as they lie, more slowly; gated_linear_grad always copies them.  The
    weights of a model are better kept aligned."""
    d, keep, rows, k, n = _gated(x, w_gate, w_up, activation)
    dtype = keep[0].dtype
    stride = n
    if out is None:
        _on_device(device, _NAMES, keep)
        out = head.torch.empty((rows, n), dtype=dtype, device=keep[0].device)
    else:
        _out("out", out, rows, n, dtype)
        if any(_overlap(out, t) for t in keep):
            _refuse("h must not be x or a weight, nor lie in their memory")
        _on_device(device, _NAMES + ("out",), keep + (out,))
        if rows > 1:
            stride = out.stride(0)
    where = out.device
    gate = up = None
    if save:
        gate, up = (head.torch.empty((rows, n), dtype=head.torch.float32, device=where) for _ in range(2))
    lib = load()
    size = lib.thrml_gated_work(device.handle, d, 0)
    work = head.torch.empty(size, dtype=head.torch.uint8, device=where) if size else None
    _run(device, lib.thrml_gated_forward, d, out.data_ptr(), stride, gate.data_ptr() if save else 0,
         up.data_ptr() if save else 0, work.data_ptr() if size else 0, size)
    return (out, gate, up) if save else out


def gated_linear_grad(device, grad, x, w_gate, w_up, gate, up, activation="silu", input_grad=True):
    """(dx, dw_gate, dw_up): the gradients of a loss in x [rows, k] and the weights [n, k],
    in their type, from grad [rows, n], its gradient in gated_linear's result in that type,
    and the products gate and up [rows, n] float32 that this kept.  With z = gate, u = up:
      dz = grad u act'(z),  du = grad act(z)   (rounded to the type)
      dx = dz @ w_gate + du @ w_up,  dw_gate = dz.T @ x,  dw_up = du.T @ x
    float16: where dz or du of a row (for dx) or of a unit (for dw_gate, dw_up) would pass 65504,
    they are divided by a power of two of that row or unit; results at the border of the type's
    range are summed again without the rounding of dz and du, so that they are infinite where
    the gradient is.  relu'(0) is 0.  Without rows the weights' gradients are 0.  input_grad
    False: dx is not computed, and None."""
    d, keep, rows, k, n = _gated(x, w_gate, w_up, activation)
    same = (keep[0].dtype,)
    grad, grad_stride = _matrix("grad", grad, same, rows, n)
    gate, _ = _matrix("gate", gate, head._FLOAT32, rows, n)
    up, _ = _matrix("up", up, head._FLOAT32, rows, n)
    gate, up = gate.contiguous(), up.contiguous()
    _on_device(device, _NAMES + ("grad", "gate", "up"), keep + (grad, gate, up), False)
    torch, where = head.torch, keep[0].device
    dx = torch.empty((rows, k), dtype=same[0], device=where) if input_grad else None
    dw_gate, dw_up = (torch.empty((n, k), dtype=same[0], device=where) for _ in range(2))
    lib = load()
    size = lib.thrml_gated_work(device.handle, d, 1)
    work = torch.empty(size, dtype=torch.uint8, device=where) if size else None
    _run(device, lib.thrml_gated_backward, d, grad.data_ptr(), grad_stride if rows > 1 else n, gate.data_ptr(),
         up.data_ptr(), dx.data_ptr() if input_grad else 0, k, dw_gate.data_ptr(), dw_up.data_ptr(),
         work.data_ptr() if size else 0, size)
    return dx, dw_gate, dw_up


def dropout(device, x, key, p, residual=None, first_row=0, out=None):
    """y [rows, cols] = (residual +) x with each unit kept and scaled, or replaced by 0, by
    the bits of a key: with the half words b of the key's ChaCha8 stream, i = (first_row +
    row) * cols + col and border = round(65536 p), kept where b[i] >= border and times
    65536 / (65536 - border), in float32, rounded once (p counts as border / 65536).  No
    mask is kept: the gradient in x is dropout(device, grad, key, p, first_row=first_row).

    key: an RngKey, used for nothing else, or its seed in an int64 tensor of one element
    on the device, which is read when the kernel runs: a captured call draws other bits
    when it changes.  first_row: where x is a part of a larger batch, its first row
    there.  out: a tensor for the result; it may be x or residual (the same rows), and share
    no other memory with them."""
    if head.torch is None:
        head._setup()
    torch = head.torch
    x, xs = _matrix("x", x, head._FLOATS)
    rows, cols = x.shape
    rs = rp = 0
    if residual is not None:
        residual, rs = _matrix("residual", residual, (x.dtype,), rows, cols)
        rp = residual.data_ptr()
    seed = at = 0
    seed_at = None
    if isinstance(key, torch.Tensor):
        if key.dtype != torch.int64 or key.numel() != 1:
            _refuse("key must be an RngKey or an int64 tensor of one element")
        seed_at, at = key, key.data_ptr()
    else:
        seed = getattr(key, "seed", None)
        if seed is None:
            _refuse("key must be an RngKey or an int64 tensor of one element")
    first_row = int(first_row)
    if not 0 <= first_row <= 1 << 37:
        _refuse("first_row must lie in 0 .. 2^37")
    if out is not None:
        _out("out", out, rows, cols, x.dtype)
        for t in (x, residual):
            same = t is not None and t.data_ptr() == out.data_ptr() and _layout(t) == _layout(out)
            if t is not None and not same and _overlap(out, t):
                _refuse("out may be x or residual, or other memory, not a part of theirs")
        if seed_at is not None and _overlap(out, seed_at.reshape(1, 1)):
            _refuse("out must not hold the key")
    _on_device(device, ("x", "residual", "key", "out"), (x, residual, seed_at, out))
    if out is None:
        out = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    _run(device, load().thrml_dropout, x.data_ptr(), head._TYPES[x.dtype], rows, cols, xs if rows > 1 else cols, rp,
         rs if rows > 1 else cols, seed, at, first_row, float(p), out.data_ptr(), out.stride(0) if rows > 1 else cols)
    return out


def linear_f8(device, x, w, w_scale, bias=None, out_dtype=None):
    """y [rows, q] = x @ w.T + bias in out_dtype (default: x's) with both sides in 8-bit
    floating point: w [q, k] float8_e4m3fn weights with a scale w_scale [ceil(q / 128),
    ceil(k / 128)] float32 for each block of 128 x 128, x [rows, k] activations that the
    call quantises in blocks of 128 of a row, s = max(2^-126, max |x| * (1 / 448)), a = x / s
    rounded to e4m3 (ties to even; in float32).  A block's sum times s w_scale is added in
    float32.  For results in 16 bits the sum within a block keeps 2^-16 of its largest
    product, for float32 all.  A row of x with an infinity or a NaN gives NaN.

    k is at most 2^20.  Weights whose rows are not whole 16-byte pieces are copied first where
    x has more than 64 rows, and else read as they lie, more slowly."""
    if head.torch is None:
        head._setup()
    torch = head.torch
    x, xs = _matrix("x", x, head._FLOATS)
    rows, k = x.shape
    w, ws = _matrix("w", w, (torch.float8_e4m3fn,), None, k)
    q = w.shape[0]
    if k == 0 or q == 0:
        _refuse("w must have at least one row and column")
    w_scale, scale_stride = _matrix("w_scale", w_scale, head._FLOAT32, (q + 127) // 128, (k + 127) // 128)
    if scale_stride != w_scale.shape[1]:
        w_scale = w_scale.contiguous()
    if bias is not None:
        bias = head._vector("bias", bias, q, head._FLOAT32)
    dtype = out_dtype or x.dtype
    code, in_code = head._type("out_dtype", dtype), head._TYPES[x.dtype]
    _on_device(device, ("x", "w", "w_scale", "bias"), (x, w, w_scale, bias))
    where = x.device
    y = torch.empty((rows, q), dtype=dtype, device=where)
    lib = load()
    wp, ws = w.data_ptr(), ws if q > 1 else k
    n = lib.thrml_linear_f8_work(device.handle, rows, k, wp, q, ws, code)
    work = torch.empty(n, dtype=torch.uint8, device=where) if n else None
    _run(device, lib.thrml_linear_f8, x.data_ptr(), in_code, rows, k, xs if rows > 1 else k, wp, q, ws,
         w_scale.data_ptr(), bias.data_ptr() if bias is not None else 0, y.data_ptr(), code, q,
         work.data_ptr() if n else 0, n)
    return y
