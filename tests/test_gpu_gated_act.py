"""The activations and their derivatives, relative to their own size, where they are small:
against their definitions in 64 bits (hidden_reference.py)."""
import hidden_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LARGE = 2.0**14  # what activations are multiplied by: f16 holds 2^-14 of them with all its bits


def _bound(v, z, dtype):
    """Half a step of the type, and of f32: 16 u for the operations, and 4 z^2 u for the
    argument: exp(-z^2 / 2), which erfc behaves like, moves by z^2 times what its z or z^2 is
    rounded by (2 u each); exp(z) by |z| times that, which is less or, below 1, within the 16."""
    return ref.half_step(dtype) * v.abs() * (1 + 2.0**-10) + (16 + 4 * z * z) * ref.U32 * v.abs() + ref.tiny(dtype)


def _close(got, want, bound, what):
    """as ref.close; what the type cannot hold, from half a step above its largest on (f16:
    65504 + 16), is infinite"""
    beyond = want.abs() >= torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    assert torch.equal(got[beyond].double(), torch.inf * want[beyond].sign()), what
    ref.close(got[~beyond], want[~beyond], bound[~beyond], what)


def _arguments(dtype):
    """-12 .. 12 in steps that the type holds, and denser around the zeros of the derivatives"""
    z = torch.cat([torch.arange(-12 * 16, 12 * 16 + 1) / 16.0, -0.5 - torch.arange(65) / 64.0, -1.0 - torch.arange(65) / 128.0])
    return z.to(dtype).cuda()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 40), (1, 65, 40), (1, 8192, 40), (100, 64, 72), (700, 64, 600)])
def test_activation(device, rows, k, n, dtype, act):
    """z is one feature times 1, u one feature times LARGE: exact, whatever the kernel"""
    log_case(f"act {rows} {k} {n} {dtype} {act}")
    z = _arguments(dtype)
    wg = torch.zeros(n, k, device="cuda", dtype=dtype)
    wu = torch.zeros(n, k, device="cuda", dtype=dtype)
    wg[:, 0], wu[:, 1] = 1.0, LARGE
    for first in range(0, len(z), rows if rows > 1 else 37):
        x = torch.zeros(rows, k, device="cuda", dtype=dtype)
        x[:, 0] = z.roll(-first).repeat(-(-rows // len(z)))[:rows]
        x[:, 1] = 1.0
        v = x[:, :1].double()
        want = (ref.act(v, act)[0] * LARGE).expand(rows, n)
        _close(th.gated_linear(device, x, wg, wu, act), want, _bound(want, v, dtype), f"h from {first}")


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_derivative(device, dtype, act):
    """dz and du of one row are the gradients of weights whose features are 1"""
    log_case(f"act slope {dtype} {act}")
    z = _arguments(torch.float32)[None]
    n = z.shape[1]
    x, w = torch.ones(1, 8, device="cuda", dtype=dtype), torch.zeros(n, 8, device="cuda", dtype=dtype)
    dh, up = torch.full((1, n), 2.0**12, device="cuda", dtype=dtype), torch.full((1, n), 4.0, device="cuda")
    _, dwg, dwu = th.gated_linear_grad(device, dh, x, w, w, z, up, act)
    a, slope = ref.act(z[0].double(), act)
    # (a derivative is a sum of two terms, each as far off as its own size allows)
    t = z[0].double()
    cdf = {"silu": torch.sigmoid(t), "gelu": 0.5 * torch.erfc(-t * 0.5**0.5), "relu": slope}[act]
    size = ((cdf.abs() + (slope - cdf).abs()) * LARGE)[:, None].expand(n, 8)
    t = t[:, None].expand(n, 8)
    want = (slope * LARGE)[:, None].expand(n, 8)
    f32 = _bound(size, t, dtype) - ref.half_step(dtype) * size * (1 + 2.0**-10)
    _close(dwg, want, ref.half_step(dtype) * want.abs() * (1 + 2.0**-10) + f32, "dz")
    want = (a * 2.0**12)[:, None].expand(n, 8)
    _close(dwu, want, _bound(want, t, dtype), "du")
