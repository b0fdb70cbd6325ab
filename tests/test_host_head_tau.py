"""Which temperatures of a distillation the C entry point takes: those whose reciprocal
f32 holds.  Against a stand-in of the HIP runtime (hostrun.py): no GPU is used."""
import hostrun
import pytest
from test_host_head import _c_calls, _distill


@pytest.mark.parametrize("weight", [None, 1 << 20])
def test_tau(weight):
    taus = [2.0**-149, 1e-40, 2.0**-128, 2.0**-127, 2.0**-126, 1e-30, 0.5, 1.0, 1e30, 3e38]
    got = hostrun.call(_c_calls, [_distill(tau=t, weight=weight) for t in taus])
    for t, (rc, text, launches) in zip(taus, got):
        if t < 2.0**-126:
            assert rc < 0 and "tau must be" in text and not launches, (t, text)
        else:
            assert rc == 0 and launches, (t, text)
