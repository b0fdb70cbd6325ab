"""The 8-bit product of rows whose scale is subnormal: magnitudes below 127 x 2^-126."""
import head_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

UNIT = 2.0**-149  # the smallest float32
# largest magnitudes in units: what 1 / 127 of them rounds down to a whole unit or to none,
# up to a scale of 2^16 units
PEAKS = [1, 2, 63, 64, 65, 126, 127, 128, 190, 191, 254, 317, 1000, 8001, 16319, 1 << 16, (1 << 23) - 1, 1 << 23]


@pytest.mark.parametrize("rows", [1, 6, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_subnormal_rows(device, dtype, rows):
    """Every activation is held to within half of a step of its row's scale, which is at
    most the largest magnitude / 127 rounded up to a unit (from 2^15 units on a unit more,
    as 1 / 127 and the product are rounded); the quotient is rounded once more before it
    is rounded to an integer, 2^-24 of 127.  The output's own roundings: 4 of them."""
    k, q = 200, 90
    g = torch.Generator().manual_seed(rows)
    w = torch.randint(-128, 128, (q, k), generator=g).to(torch.int8)
    ws = (0.5 + torch.rand(q, generator=g)) * 2.0**100
    for peak in PEAKS:
        if dtype == torch.bfloat16:
            peak <<= 16  # its units
            if peak > 1 << 30:
                continue
        log_case(f"subnormal rows {dtype} {rows} {peak}")
        n = torch.randint(-peak, peak + 1, (rows, k), generator=g).double()
        n[:, 5], n[:, 77] = peak, -peak
        x = (n * UNIT).to(dtype)
        xd = x.double()
        got = th.linear_i8(device, x.cuda(), w.cuda(), ws.cuda(), out_dtype=torch.float32).cpu().double()
        want = (xd @ w.double().t()) * ws.double()
        m = (xd.abs().amax(1, keepdim=True) / UNIT).round()  # exact
        step = torch.where(m < 2**15, torch.ceil(m / 127), m / 127 * (1 + 2.0**-22) + 1)
        bound = step * UNIT * (0.5 + 127 * 2.0**-24) * (w.double().abs().sum(1) * ws.double())
        assert ((got - want).abs() <= bound + 4 * ref.EPS * (want.abs() + bound)).all(), peak
