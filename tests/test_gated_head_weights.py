"""GatedHead.quantised on the CPU: 8-bit weights and scales by the rule that linear_f8 has for
activations.  No GPU is used."""
import hidden_reference as ref
import pytest
import torch

from thrml_hip.conditional_head import GatedHead


def _quantised(w):
    head = object.__new__(GatedHead)
    head.w = w
    return head.quantised()


@pytest.mark.parametrize("size", [1.0, 1e30, 1e-30, 2.0**-118, 2.0**-126, 600 * 2.0**-149, 2.0**-149, 0.0])
def test_quantised(size):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(300, 200, generator=g)
    w[128:256, :128] *= size / w[128:256, :128].abs().max()
    q, scale = _quantised(w)
    assert q.dtype == torch.float8_e4m3fn and q.shape == w.shape and scale.shape == (3, 2)
    assert not q.float().isnan().any() and (scale >= 2.0**-126).all() and scale.isfinite().all()
    wide = scale.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :200]
    err = (q.double() * wide - w.double()).abs()
    # half a step of e4m3, or of its smallest values, and of the quotient in f32
    assert (err <= (2.0**-4 + 2 * ref.U32) * w.double().abs() + 2.0**-10 * wide).all()
    if size >= 2.0**-117:
        assert (q.float()[128:256, :128].abs().max() == 448.0).all()
