"""Every kind of tile that the products of a hidden block take, with the reduction whole and
split, in each pass and type, against the definitions in 64 bits.  Which kernel each shape
reaches is asserted without a GPU (test_host_hidden_tiles.py)."""
import hidden_reference as ref
import pytest
import test_gpu_gated as gated
import test_gpu_linear_f8 as f8
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# (tile, whether the reduction is split): rows, k, n
FORWARD = {
    ("64x32", False): (43, 264, 42), ("64x32", True): (39, 2952, 41), ("64x64", False): (578, 136, 425),
    ("64x64", True): (33, 2288, 560), ("128x128", False): (841, 136, 1167), ("128x128", True): (2059, 3680, 41),
    ("256x256", False): (913, 136, 2190), ("256x256", True): (4558, 6056, 100),
}
INPUT = {
    ("64x32", False): (33, 72, 134), ("64x32", True): (33, 80, 1429), ("64x64", False): (898, 520, 41),
    ("64x64", True): (519, 72, 1040), ("128x128", False): (2059, 1016, 40), ("128x128", True): (2066, 72, 1694),
    ("256x256", False): (2330, 1792, 40), ("256x256", True): (136, 2752, 6233),
}
WEIGHT = {
    ("64x32", False): (260, 80, 46), ("64x32", True): (2945, 96, 41), ("64x64", False): (137, 344, 679),
    ("64x64", True): (2266, 72, 277), ("128x128", False): (132, 1232, 781), ("128x128", True): (3481, 80, 1026),
    ("256x256", False): (520, 1032, 2056), ("256x256", True): (3407, 136, 8393),
}
# rows, k, q
F8_16 = {
    ("64x32", False): (43, 272, 42), ("64x32", True): (35, 3808, 41), ("64x64", False): (1040, 272, 453),
    ("64x64", True): (33, 4080, 1033), ("128x128", False): (386, 272, 4809), ("128x128", True): (2057, 6768, 70),
    ("256x256", False): (3659, 272, 2226), ("256x256", True): (577, 4752, 8580),
}
F8_32 = {
    ("64x32", False): (43, 272, 42), ("64x32", True): (39, 2960, 41), ("64x64", False): (1365, 272, 706),
    ("64x64", True): (1027, 5744, 65), ("128x128", False): (1347, 272, 2238),
}
# inner sizes of more than 64 blocks of 128: the weights' scales are loaded more than once
F8_LONG_16 = {"64x32": (65, 8304, 4322), "64x64": (43, 8256, 8534), "128x128": (196, 8240, 8982), "256x256": (2050, 8336, 4104)}
F8_LONG_32 = {"64x32": (36, 8272, 8484), "64x64": (4215, 8736, 195), "128x128": (325, 8368, 8268)}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tile", FORWARD)
def test_forward(device, tile, dtype):
    x, wg, wu, _ = gated._inputs(*FORWARD[tile], dtype)
    for act in ("silu", "gelu", "relu"):
        log_case(f"forward {tile} {dtype} {act}")
        h, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
        want = ref.gated(x, wg, wu, act)
        for name, got in (("h", h), ("gate", gate), ("up", up)):
            ref.close(got, *want[name], name)
        assert torch.equal(th.gated_linear(device, x, wg, wu, act), h)


@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (F16, "gelu"), (F16, "relu")])
@pytest.mark.parametrize("which,tile", [*(("dx", t) for t in INPUT), *(("dw", t) for t in WEIGHT)])
def test_gradients(device, which, tile, dtype, act):
    log_case(f"{which} {tile} {dtype} {act}")
    x, wg, wu, dh = gated._inputs(*(INPUT if which == "dx" else WEIGHT)[tile], dtype)
    _, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    again = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    for (name, (want, bound)), got, same in zip(ref.gated_grad(dh, x, wg, wu, gate, up, act).items(), grads, again):
        ref.close(got, want, bound, name)
        assert torch.equal(got, same), name


def _linear_f8(x, w, ws, bias, out):
    """hidden_reference.linear_f8 with its products on the device"""
    (a, s), q, k = ref.quantised(x), w.shape[0], x.shape[1]
    a, s = a.cuda(), s.cuda()
    blocks = s.shape[1]
    ww = torch.zeros(q, blocks * 128, dtype=torch.float64, device="cuda")
    ww[:, :k] = w.double()
    ww = ww.view(q, blocks, 128)
    scale = ws.double().repeat_interleave(128, 0)[:q]
    left, right = (a * s[:, :, None]).flatten(1), (ww * scale[:, :, None]).flatten(1).t().contiguous()
    y, size = torch.mm(left, right) + bias.double(), torch.mm(left.abs(), right.abs()) + bias.double().abs()
    err = (k + 4) * ref.U32 * size + ref.tiny(F32) * k
    if out != F32:
        err = err + 128 * 2.0**-16 * torch.mm(a.abs().amax(2) * s, (ww.abs().amax(2) * scale).t().contiguous())
        err = err + ref.half_step(out) * (y.abs() + err) + ref.tiny(out)
    return y, err


def _check_f8(device, shape, dtype, out):
    x, w, ws, bias = f8._inputs(*shape, dtype)
    got = th.linear_f8(device, x, w, ws, bias=bias, out_dtype=out)
    ref.close(got, *_linear_f8(x, w, ws, bias, out), "linear_f8")
    assert torch.equal(th.linear_f8(device, x, w, ws, bias=bias, out_dtype=out), got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tile", F8_16)
def test_f8_to_16_bits(device, tile, dtype):
    log_case(f"f8 {tile} {dtype}")
    _check_f8(device, F8_16[tile], dtype, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tile", F8_32)
def test_f8_to_32_bits(device, tile, dtype):
    log_case(f"f8 to f32 {tile} {dtype}")
    _check_f8(device, F8_32[tile], dtype, F32)


@pytest.mark.parametrize("tile", F8_LONG_16)
def test_f8_long(device, tile):
    log_case(f"f8 long {tile}")
    _check_f8(device, F8_LONG_16[tile], BF16, BF16)


@pytest.mark.parametrize("tile", F8_LONG_32)
def test_f8_long_to_32_bits(device, tile):
    log_case(f"f8 long to f32 {tile}")
    _check_f8(device, F8_LONG_32[tile], BF16, F32)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_quantised_by_the_workgroups(device, dtype):
    """one row to as many as fit, to each type"""
    for rows, k, q in ((1, 8320, 300), (1, 16384, 70000), (3, 4096, 40000), (8, 2048, 33000), (31, 512, 40000)):
        for out in {dtype, F32}:
            log_case(f"f8 own {rows} {k} {q} {dtype} {out}")
            _check_f8(device, (rows, k, q), dtype, out)
