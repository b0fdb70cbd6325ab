"""Log-probabilities of drawn categories at low temperatures: their error follows the
distance to the row's largest logit, not the logits' size, and none is above 0."""
import head_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu


def _want(y, t, pick, q):
    """(log-probabilities, bounds) in 64 bits from logits y, which are exact, and t.

    With d = (largest - y) / t: the pick's d is a difference and a quotient.  In the sum
    of e^-d an exponent takes the difference, the reciprocal of t, its product with
    log2 e (itself rounded), and theirs: 5 roundings of d, which move log sum by at most
    their mean.  2^x is off by 2 roundings; 8 additions of a group, a rescaling (2^x, a
    product, an addition: 4) for each group of a lane and each of 28 merges (two each).
    Then the logarithm, 2, and the last difference."""
    yd, td = y.double(), t.double()[:, None]
    d = (yd.amax(1, keepdim=True) - yd) / td
    e = torch.exp(-d)
    total = e.sum(1)
    at = d.gather(1, pick.long()[:, None])[:, 0]
    want = -at - torch.log(total)
    mean = (torch.where(e > 0, e * d, 0.0)).sum(1) / total
    bound = ref.EPS * (2 * at + 5 * mean + 2 + 8 + 4 * (q / 4096 + 1) + 28 * 8 + 2 * torch.log(total) + want.abs())
    return want, bound


@pytest.mark.parametrize("lists", [False, True])
@pytest.mark.parametrize("t", [1.0, 0.05, 0.01, 0.001])
@pytest.mark.parametrize("rows,q", [(64, 40), (64, 5000), (4, 70000), (160, 9001)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logprob(device, dtype, rows, q, t, lists):
    log_case(f"logprob {dtype} {rows} {q} {t} {lists}")
    g = torch.Generator().manual_seed(q)
    z = 10.0 + 20.0 * torch.rand(rows, q, generator=g)
    z[::4, q // 3] = 37.0  # a dominant category
    z[1::4] = 5.0 + 0.01 * torch.rand(z[1::4].shape, generator=g)  # many of one size
    z = z.to(dtype)
    temperature = torch.full((rows,), t) * (1 + torch.arange(rows) / 1000)
    kw = {}
    if lists:
        kw = {"history": torch.randint(0, q, (rows, 30), generator=g, dtype=torch.int32),
              "repetition": torch.full((rows,), 1.1)}
        kw["history"][0] = q // 3
    y, _ = ref.processed(torch.float32, z, **kw)
    u = torch.rand(rows, q, generator=g)
    kw["temperature"] = temperature
    for uniforms in (u, None):
        index, _, _ = ref.sampled(z, uniforms, **kw)
        got, logprob = th.sample_logits(device, z.cuda(), None if uniforms is None else uniforms.cuda(),
                                        **{k: v.cuda() for k, v in kw.items()})
        assert got.cpu().tolist() == index.tolist()
        want, bound = _want(y, temperature, index, q)
        lp = logprob.cpu().double()
        assert (lp <= 0).all(), lp.max()
        off = (lp - want).abs() - bound
        assert (off <= 0).all(), (float((lp - want).abs().max()), off.argmax())
