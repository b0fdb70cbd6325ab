"""Every kind of tile of the 8-bit product, at remainders of rows, channels and columns, with
few and many steps of k, and weight rows at and off multiples of 16 bytes.
test_host_head_kernels.py holds each shape to the kernel that it is meant for."""
import head_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

# kernel: (rows, channels)
SHAPES = {
    "few": [(17, 1003), (130, 70)],
    "TileShape<1,1,2,2>": [(1100, 700), (1029, 515)],
    "TileShape<1,2,2,2>": [(1500, 1100), (1413, 1157)],
    "TileShape<2,2,2,4>": [(2050, 2055), (300, 20003)],
    "TileShape<4,2,2,4>": [(2100, 4090), (1029, 12003)],
}
# k, weight rows' padding, the first weight's byte: 1, 2, 3, 5 and 16 steps of 64 columns;
# straight into LDS (or registers) and not
COLUMNS = [(64, 0, 0), (80, 16, 48), (192, 0, 0), (272, 0, 0), (1008, 0, 0),
           (16, 0, 0), (64, 0, 4), (65, 0, 0), (100, 28, 0), (192, 4, 0), (270, 0, 1), (1001, 0, 0)]


def _direct(k, pad, shift):
    return k % 16 == 0 and (k + pad) % 16 == 0 and shift % 16 == 0


# the second shape of a kind with a few of them
CASES = [(kind, rows, q, k, pad, shift) for kind, shapes in SHAPES.items() for i, (rows, q) in enumerate(shapes)
         for k, pad, shift in (COLUMNS[1::4] if i else COLUMNS)]
OUTS = (torch.bfloat16, torch.float16, torch.float32)


@pytest.mark.parametrize("i", range(len(CASES)))
def test_tiles(device, i):
    """127 x 128 x k stays below 2^24: a product in f32 gives the integers."""
    kind, rows, q, k, pad, shift = CASES[i]
    out = OUTS[i % 3]
    log_case(f"tiles {kind} {rows} {k} {q} {pad} {shift} {out}")
    g = torch.Generator().manual_seed(rows + k + q)
    x = torch.randn(rows, k, generator=g).to(torch.bfloat16)
    w = torch.randint(-128, 128, (q, k), generator=g).to(torch.int8)
    ws = (0.5 + torch.rand(q, generator=g)) * 1e-3
    b = torch.randn(q, generator=g) if i % 2 else None
    wide = torch.full((q * (k + pad) + shift,), 99, dtype=torch.int8).cuda()
    view = wide[shift:].view(q, k + pad)[:, :k]
    view.copy_(w)
    a, s = ref.integers(x)
    want = ((a @ w.float().t()).double() * s.double()) * ws.double()
    bound = 4 * ref.EPS * want.abs()  # as ref.product
    if b is not None:
        want = want + b.double()
        bound = bound + ref.EPS * want.abs()
    got = th.linear_i8(device, x.cuda(), view, ws.cuda(), b.cuda() if b is not None else None, out)
    ref.close(got, want, bound, CASES[i])
