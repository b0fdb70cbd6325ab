"""The operators of a learned head's hidden block from their definitions in 64 bits, on
the CPU or the device, with bounds of the error that 32-bit sums and the documented
roundings allow.  Nothing here is the library's."""
import math

import torch

U32 = 2.0**-24  # half a step of f32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half the distance of the smallest values"""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def act(z, name):
    """(act(z), act'(z))"""
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    phi = 0.5 * torch.erfc(-z * math.sqrt(0.5))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


STEEPEST = 1.13  # of the activations (gelu at sqrt 2: 1.129)


def gated(x, wg, wu, name):
    """{h, gate, up} and the error allowed for each: a sum of k products in f32 is off by at
    most k u sum |terms|, the activation by 8 u of its value or, where that is small, of
    its argument's (its exponential or error function by a few steps)."""
    dtype, k = x.dtype, x.shape[1]
    x, wg, wu = x.double(), wg.double(), wu.double()
    z, u = torch.mm(x, wg.t().contiguous()), torch.mm(x, wu.t().contiguous())
    ez, eu = (k * U32 * torch.mm(x.abs(), w.abs().t().contiguous()) for w in (wg, wu))
    a, _ = act(z, name)
    h = a * u
    eh = STEEPEST * ez * (u.abs() + eu) + (a.abs() + STEEPEST * ez) * eu + 16 * U32 * z.abs() * u.abs()
    out = {}
    for n, v, e in (("h", h, eh), ("gate", z, ez), ("up", u, eu)):
        step, least = (half_step(dtype), tiny(dtype)) if n == "h" else (U32, tiny(torch.float32))
        out[n] = v, e + step * (v.abs() + e) + least
    return out


def gated_grad(dh, x, wg, wu, z, u, name):
    """{dx, dw_gate, dw_up} and the error allowed for each, from the kept z and u: dz and du
    are rounded to the type (and computed in f32: 16 u of the factors), the sums are in f32."""
    dtype = x.dtype
    dh, x, wg, wu, z, u = (t.double() for t in (dh, x, wg, wu, z, u))
    a, slope = act(z, name)
    dz, du = dh * u * slope, dh * a
    ez = 16 * U32 * (dh * u).abs() * (1 + z.abs())
    eu = 16 * U32 * (dh * z).abs()
    ez, eu = (e + half_step(dtype) * (v.abs() + e) + tiny(dtype) for e, v in ((ez, dz), (eu, du)))
    terms = 2 * wg.shape[0]
    dx = torch.mm(dz, wg) + torch.mm(du, wu)
    ex = torch.mm(ez, wg.abs()) + torch.mm(eu, wu.abs())
    ex = ex + terms * U32 * (torch.mm(dz.abs() + ez, wg.abs()) + torch.mm(du.abs() + eu, wu.abs()))
    out = {"dx": (dx, ex)}
    rows = x.shape[0]
    for n, d, e in (("dw_gate", dz, ez), ("dw_up", du, eu)):
        dt, et = d.t().contiguous(), e.t().contiguous()
        out[n] = torch.mm(dt, x), torch.mm(et, x.abs()) + rows * U32 * torch.mm(dt.abs() + et, x.abs())
    return {n: (v, e + half_step(dtype) * (v.abs() + e) + tiny(dtype)) for n, (v, e) in out.items()}


def close(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by "
                           f"{float((err / bound).nan_to_num(1e30).max()):.3g} times what is allowed, first at "
                           f"{bad.nonzero()[0].tolist()}")


F8 = torch.float8_e4m3fn


def quantised(x):
    """(8-bit floats [rows, blocks, 128] and scales [rows, blocks] in 64 bits) of rows of
    f32: s = max(2^-126, max |x| times 1 / 448), a = x / s, both in f32, on the CPU"""
    rows, k = x.shape
    wide = torch.zeros(rows, -(-k // 128) * 128)
    wide[:, :k] = x.cpu().float()
    blocks = wide.view(rows, -1, 128)
    s = (blocks.abs().amax(2) * torch.tensor(1.0 / 448.0)).clamp(min=2.0**-126)
    return (blocks / s[:, :, None]).to(F8).double(), s.double()


def linear_f8(x, w, w_scale, bias, out):
    """(y, error allowed) on the CPU in 64 bits.  f32: k + 4 roundings of sums, scales and bias.
    16 bits: besides, in each block of 128 each product is off by at most 2^-16 of the
    largest, and the result by half a step."""
    (a, s), q, k = quantised(x), w.shape[0], x.shape[1]
    rows, blocks = s.shape
    ww = torch.zeros(q, blocks * 128, dtype=torch.float64)
    ww[:, :k] = w.cpu().double()
    ww = ww.view(q, blocks, 128)
    ws = w_scale.cpu().double().repeat_interleave(128, 0)[:q]
    left, right = (a * s[:, :, None]).flatten(1), (ww * ws[:, :, None]).flatten(1)
    y, size = left @ right.T, left.abs() @ right.abs().T
    if bias is not None:
        y = y + bias.cpu().double()
        size = size + bias.cpu().double().abs()
    err = (k + 4) * U32 * size + tiny(torch.float32) * k
    if out != torch.float32:
        err = err + 128 * 2.0**-16 * (a.abs().amax(2) * s) @ (ww.abs().amax(2) * ws).T
        err = err + half_step(out) * (y.abs() + err) + tiny(out)
    return y, err
