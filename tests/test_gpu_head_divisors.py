"""Logits divided by every kind of positive number: temperatures and repetition penalties
from the smallest subnormal to infinity, by the definition in f32 (z / t)."""
import head_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = float("inf"), float("nan")
DIVISORS = [2.0**-149, 1e-45, 1e-40, 2.0**-129, 2.0**-128, 1.5 * 2.0**-128, 2.0**-127, 2.0**-126, 1e-37, 1e-30, 0.3,
            1.0, 7.0, 1e30, 1.3e38, 3e38, INF]
VALUES = [0.0, -0.0, 1e-45, -1e-45, 1e-42, -3e-41, 1e-39, -2e-39, 1.1e-38, 1e-30, -1e-20, 0.7, -1.0, 3.3, 1e4, -1e20,
          3e38, -3e38, INF, -INF, NAN, 1e-3]


def _held(got, want, what):
    """The quotient is a product with the reciprocal, corrected by its remainder: half a
    step, as much again where the remainder is too small for f32 and is lost, and a
    unit where the quotient is subnormal."""
    got, want = got.cpu().double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    near = ((got - want).abs() <= 3 * ref.EPS * want.abs() + 2.0**-149) & want.isfinite()
    bad = (~(same | near)).nonzero()
    assert not bad.numel(), (what, [(i.tolist(), float(got[tuple(i)]), float(want[tuple(i)])) for i in bad[:6]])


@pytest.mark.parametrize("times", [1, 64])  # few and many rows
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_temperatures(device, dtype, times):
    log_case(f"temperatures {dtype} {times}")
    t = torch.tensor(DIVISORS, dtype=F32).repeat(times)
    z = torch.tensor(VALUES, dtype=F32).to(dtype).expand(len(t), -1).contiguous()
    got = th.process_logits(device, z.cuda(), temperature=t.cuda(), out_dtype=F32)
    _held(got, z.float() / t[:, None], "z / t")
    # masked places hold -inf whatever the temperature
    mask = torch.full((1, 1), 0x2aaaaa, dtype=torch.int32)
    got = th.process_logits(device, z.cuda(), temperature=t.cuda(), mask=mask.cuda(), out_dtype=F32)
    assert (got[:, ::2] == -INF).all()
    _held(got[:, 1::2], (z.float() / t[:, None])[:, 1::2], "z / t, masked")


@pytest.mark.parametrize("times", [1, 64])
def test_repetition(device, times):
    log_case(f"repetition {times}")
    theta = torch.tensor(DIVISORS + [-d for d in DIVISORS] + [0.0], dtype=F32).repeat(times)
    z = torch.tensor(VALUES, dtype=F32).expand(len(theta), -1).contiguous()
    history = torch.arange(len(VALUES), dtype=torch.int32).expand(len(theta), -1).contiguous()
    got = th.process_logits(device, z.cuda(), history=history.cuda(), repetition=theta.cuda(),
                            prompt_lengths=torch.full((len(theta),), 99, dtype=torch.int32).cuda())
    want = torch.where(z > 0, z / theta[:, None], z * theta[:, None])
    _held(got, want, "repetition")


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("rows_times", [1, 16])
def test_both_in_place(device, rows_times, out):
    """Penalties and temperatures of every kind together, biases and a mask, into the logits
    themselves: one rounding for each of the steps, relative to the larger of its two
    sides, which the temperature divides too."""
    n = len(DIVISORS)
    t = torch.tensor(DIVISORS, dtype=F32).repeat_interleave(n).repeat(rows_times)
    theta = torch.tensor(DIVISORS, dtype=F32).repeat(n).repeat(rows_times)
    rows, q = len(t), 5000 // rows_times
    log_case(f"both {rows} {q} {out}")
    g = torch.Generator().manual_seed(rows)
    z = torch.tensor(VALUES, dtype=F32).repeat(q // len(VALUES) + 1)[:q].to(out).expand(rows, -1).contiguous()
    kw = {"history": torch.randint(0, q, (rows, 40), generator=g, dtype=torch.int32), "repetition": theta,
          "prompt_lengths": torch.full((rows,), 40, dtype=torch.int32), "temperature": t,
          "bias_ids": torch.randint(0, q, (rows, 5), generator=g, dtype=torch.int32),
          "bias_values": torch.randn(rows, 5, generator=g),
          "mask": torch.randint(-2**31, 2**31, (rows, (q + 31) // 32), generator=g).to(torch.int32)}
    want, _ = ref.processed(F32, z, **kw)
    zd = z.cuda()
    assert th.process_logits(device, zd, out=zd, **{k: v.cuda() for k, v in kw.items()}) is zd
    got, want = zd.cpu().double(), want.double()
    first, _ = ref.processed(F32, z, **{k: v for k, v in kw.items() if k not in ("temperature", "mask")})
    # each quotient as in _held: 3 roundings or a unit; the sum with a bias, below 8, is
    # relative to a penalised logit of at most 1.5 times itself or 8
    size = torch.where(first.isfinite(), torch.clamp(first.double().abs(), min=8.0), 0.0)
    off = (10 * ref.EPS * size + 2 * 2.0**-149) / t.double()[:, None]
    same = (got == want) | (got.isnan() & want.isnan())
    half = ref.HALF_STEP[out]
    near = ((got - want).abs() <= off + half * want.abs() + 2.0**-133) & want.isfinite()
    # beyond the type's range by its last rounding
    over = got.isinf() & (got.sign() == want.sign()) & (want.abs() > torch.finfo(out).max * (1 - 2 * half))
    bad = (~(same | near | over)).nonzero()
    assert not bad.numel(), [(i.tolist(), float(got[tuple(i)]), float(want[tuple(i)])) for i in bad[:6]]


def _logprob(z, index, kw):
    """In 64 bits from the steps before the temperature in f32, as they are defined: a
    penalty's rounding of a subnormal logit is no small part of it."""
    t = kw["temperature"].double()[:, None]
    y, _ = ref.processed(F32, z, **{k: v for k, v in kw.items() if k != "temperature"})
    x = torch.where(t < INF, y.double() / t, torch.where(y > -INF, 0.0, -INF).double())
    lp = x.gather(1, index.clamp(min=0).long()[:, None])[:, 0] - torch.logsumexp(x, 1)
    return torch.where(index < 0, NAN, lp)


@pytest.mark.parametrize("q", [40, 5000, 70000])
@pytest.mark.parametrize("lists", [False, True])
def test_samples(device, lists, q):
    """Logits of the temperature's own size, logits of zero, and logits whose quotients
    leave f32: a row that holds +inf, or nothing above -inf, has no distribution."""
    log_case(f"samples {lists} {q}")
    g = torch.Generator().manual_seed(q)
    temps = [2.0**-149, 1e-43, 1e-40, 2.0**-128, 2.0**-127, 2.0**-126, 1e-30, 1e30, 3e38, INF]
    rows = []
    for t in temps:
        scale = min(t, 1e37) if t < 3e38 else 1.0
        rows += [(t, 3.0 * torch.randn(q, generator=g).double() * scale), (t, torch.zeros(q).double()),
                 (t, torch.randn(q, generator=g).double())]
    # all of a row's quotients are -inf; all but those of zero
    rows += [(1e-40, torch.full((q,), -1.0).double()), (1e-40, -(torch.arange(q) % 3 > 0).double())]
    # a quotient that is no number counts, unless it is masked
    rows += [(INF, torch.where(torch.arange(q) == 6, -INF, 0.5).double()),
             (INF, torch.where(torch.arange(q) == 7, -INF, 0.5).double())]
    z = torch.stack([r for _, r in rows]).to(F32)
    kw = {"temperature": torch.tensor([t for t, _ in rows], dtype=F32),
          "mask": torch.randint(-2**31, 2**31, (1, (q + 31) // 32), generator=g).to(torch.int32) & ~128 | 64}
    if lists:
        kw["history"] = torch.randint(0, q, (len(rows), 50), generator=g, dtype=torch.int32)
        kw["repetition"] = torch.full((len(rows),), 1.25)
    u = torch.rand(len(rows), q, generator=g)
    for uniforms in (u, None):
        want, _, bound = ref.sampled(z, uniforms, **kw)
        index, logprob = th.sample_logits(device, z.cuda(), None if uniforms is None else uniforms.cuda(),
                                          **{k: v.cuda() for k, v in kw.items()})
        assert index.cpu().tolist() == want.tolist()
        ref.close(logprob, _logprob(z, want, kw), bound, "logprob")
