"""Draws whose scores lie closer together than f32 tells apart, with uniforms of every
size: what the hardware's logarithms are off by must never decide a pick."""
import head_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu


def _uniforms(kind, shape, g):
    if kind == "all":  # every exponent alike
        bits = torch.randint(1, 127 << 23, shape, generator=g, dtype=torch.int32)
    elif kind == "near 1":
        bits = (127 << 23) - 1 - (2.0 ** (24 * torch.rand(shape, generator=g))).to(torch.int32)
    elif kind == "near 0":
        bits = (1 << 23) + torch.randint(0, 1 << 24, shape, generator=g, dtype=torch.int32)
    else:  # where the score is near 0: u = 1 / e
        bits = 0x3ebc5ab2 + torch.randint(-1 << 16, 1 << 16, shape, generator=g, dtype=torch.int32)
    return bits.view(torch.float32)


@pytest.mark.parametrize("kind", ["all", "near 1", "near 0", "near 1 / e"])
@pytest.mark.parametrize("rows,q", [(512, 64), (64, 5000), (3, 70000), (150, 9001)])
def test_close_scores(device, rows, q, kind):
    """Logits that cancel the noise, but for their rounding to f32."""
    log_case(f"close scores {rows} {q} {kind}")
    g = torch.Generator().manual_seed(q)
    u = _uniforms(kind, (rows, q), g)
    z = torch.log(-torch.log(u.double())).float()
    want, _, _ = ref.sampled(z, u)
    index, _ = th.sample_logits(device, z.cuda(), u.cuda())
    assert index.cpu().tolist() == want.tolist()
    # the same by a temperature
    t = torch.full((rows,), 0.37)
    z = (z.double() * 0.37).float()
    want, _, _ = ref.sampled(z, u, temperature=t)
    index, _ = th.sample_logits(device, z.cuda(), u.cuda(), temperature=t.cuda())
    assert index.cpu().tolist() == want.tolist()
