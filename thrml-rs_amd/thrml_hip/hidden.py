"""Operators of a learned head's hidden block, on torch tensors of the device (no
counterpart in the reference):

  gated_linear       hidden units act(x @ w_gate.T) * (x @ w_up.T)
  gated_linear_grad  the gradients of a loss in x and both weights

Streams, graphs and tensors that require a gradient are as in `head`: calls queue their
kernels on the device's stream, in order with torch's current one, and torch's gradients
do not go through them (gated_linear_grad gives the gradients).
"""
import struct

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
    With save, (h, gate, up): also both products, rounded to the type, for
    gated_linear_grad.  out: a tensor for h, other than x and the weights.

    Rows that are not whole 16-byte pieces (k not a multiple of 8, a view that starts or
    steps elsewhere) are copied first; the weights of a model are better kept aligned."""
    d, keep, rows, k, n = _gated(x, w_gate, w_up, activation)
    dtype = keep[0].dtype
    stride = n
    if out is None:
        _on_device(device, _NAMES, keep)
        out = head.torch.empty((rows, n), dtype=dtype, device=keep[0].device)
    else:
        _on_device(device, _NAMES + ("out",), keep + (_out("out", out, rows, n, dtype),))
        if rows > 1:
            stride = out.stride(0)
    where = out.device
    gate = up = None
    if save:
        gate, up = (head.torch.empty((rows, n), dtype=dtype, device=where) for _ in range(2))
    lib = load()
    size = lib.thrml_gated_work(device.handle, d, 0)
    work = head.torch.empty(size, dtype=head.torch.uint8, device=where) if size else None
    _run(device, lib.thrml_gated_forward, d, out.data_ptr(), stride, gate.data_ptr() if save else 0,
         up.data_ptr() if save else 0, work.data_ptr() if size else 0, size)
    return (out, gate, up) if save else out


def gated_linear_grad(device, grad, x, w_gate, w_up, gate, up, activation="silu", input_grad=True):
    """(dx, dw_gate, dw_up): the gradients of a loss in x [rows, k] and the weights [n, k],
    in their type, from grad [rows, n], its gradient in gated_linear's result, and the
    products gate and up that this kept.  With z = gate, u = up:
      dz = grad u act'(z),  du = grad act(z)   (rounded to the type)
      dx = dz @ w_gate + du @ w_up,  dw_gate = dz.T @ x,  dw_up = du.T @ x
    relu'(0) is 0.  Without rows the weights' gradients are 0.  input_grad False: dx is
    not computed, and None."""
    d, keep, rows, k, n = _gated(x, w_gate, w_up, activation)
    same = (keep[0].dtype,)
    grad, grad_stride = _matrix("grad", grad, same, rows, n)
    gate, _ = _matrix("gate", gate, same, rows, n)
    up, _ = _matrix("up", up, same, rows, n)
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
