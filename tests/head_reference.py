"""The operators around a learned head by their definitions, on the CPU in 64 bits
(the processed logits also step by step in 32 bits: a pick is exact for those),
with bounds of what a computation in f32 may be off by.

A rounding is off by at most half a step, EPS = 2^-24 of the value in f32."""
import torch

EPS = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _counts(rows, q, history, lengths, prompt_lengths):
    seen = torch.zeros(rows, q, dtype=torch.bool)
    n = torch.zeros(rows, q, dtype=torch.int64)
    for r in range(rows):
        h = history[r]
        end = h.numel() if lengths is None else max(0, min(int(lengths[r]), h.numel()))
        begin = 0 if prompt_lengths is None else max(0, int(prompt_lengths[r]))
        ok = (h[:end] >= 0) & (h[:end] < q)
        seen[r, h[:end][ok].long()] = True
        late = h[begin:end]
        late = late[(late >= 0) & (late < q)].long()
        n[r] += torch.bincount(late, minlength=q)
    return seen, n


def _column(t, rows, default, dtype):
    return torch.full((rows, 1), default, dtype=dtype) if t is None else t.to(dtype)[:, None]


def processed(dtype, logits, history=None, lengths=None, prompt_lengths=None, repetition=None, presence=None,
              frequency=None, bias_ids=None, bias_values=None, temperature=None, mask=None):
    """(x, size): the processed logits with each step in dtype, and the sum of the
    magnitudes that the steps' roundings are relative to."""
    x = logits.to(dtype)
    rows, q = x.shape
    size = x.abs()
    if history is not None:
        seen, n = _counts(rows, q, history, lengths, prompt_lengths)
        theta = _column(repetition, rows, 1.0, dtype)
        x = torch.where(seen, torch.where(x > 0, x / theta, x * theta), x)
        size = torch.maximum(size, x.abs())
        less = _column(frequency, rows, 0.0, dtype) * n.to(dtype)
        pres = _column(presence, rows, 0.0, dtype)
        x = torch.where(n > 0, x - less, x)
        x = torch.where(n > 0, x - pres, x)
        size = size + torch.where(n > 0, less.abs() + pres.abs(), torch.zeros((), dtype=dtype))
    if bias_ids is not None:
        b = torch.zeros(rows, q, dtype=dtype)
        any_ = torch.zeros(rows, q, dtype=torch.bool)
        for r in range(rows):
            for i, v in zip(bias_ids[r].tolist(), bias_values[r].to(dtype)):
                if 0 <= i < q:
                    b[r, i] = b[r, i] + v
                    any_[r, i] = True
        x = torch.where(any_, x + b, x)
        size = size + b.abs()
    if temperature is not None:
        t = temperature.to(dtype)[:, None]
        one = torch.ones((), dtype=dtype)
        x = torch.where(t > 0, x / torch.where(t > 0, t, one), x)
        size = torch.where(t > 0, size / torch.where(t > 0, t, one), size)
    if mask is not None:
        j = torch.arange(q)
        words = mask.to(torch.int64)[:, j // 32]
        x = torch.where((words >> (j % 32)) & 1 != 0, x, torch.tensor(-float("inf"), dtype=dtype))
    return x, size.nan_to_num(posinf=0.0)


def sampled(logits, u=None, **kw):
    """(index, logprob in 64 bits, bound of logprob's error in f32)"""
    x, size = processed(torch.float32, logits, **kw)
    t = kw.get("temperature")
    rows, q = x.shape
    noisy = torch.full((rows, 1), u is not None)
    if t is not None and u is not None:
        noisy = (t > 0)[:, None]
    xd = x.double()
    score = xd
    if u is not None:
        noise = -torch.log(-torch.log(u.double()))
        score = torch.where(noisy, xd + noise, xd)
        low = torch.finfo(torch.float64).min
        score = torch.where((xd > -torch.inf) & (score == -torch.inf), low, score)
    index = torch.full((rows,), -1, dtype=torch.int32)
    logprob = torch.full((rows,), float("nan"), dtype=torch.float64)
    bound = torch.zeros(rows, dtype=torch.float64)
    x64, size64 = processed(torch.float64, logits, **kw)
    for r in range(rows):
        row = xd[r]
        if bool(row.isnan().any()) or bool((row == torch.inf).any()) or not bool((row > -torch.inf).any()):
            continue
        s = score[r]
        index[r] = int((s == s.max()).nonzero()[0])
        logprob[r] = x64[r, index[r]] - torch.logsumexp(x64[r], 0)
        finite = x64[r][x64[r] > -torch.inf]
        # x: at most 6 steps and the product with the reciprocal; the
        # exponentials: the product with log2 e and the hardware's 2^x, of at
        # most 64 below the maximum; a lane's additions, then the merges of 64
        # lanes, 16 waves and 64 segments; the logarithm and two differences
        spread = min(64.0, float(finite.max() - finite.min()))
        bound[r] = EPS * (10 * float(size64[r][x64[r] > -torch.inf].max()) + 3 * spread + 2 * q / 4096 + 64 +
                          4 * abs(float(logprob[r])))
    return index, logprob, bound


def distilled(logits, ids, teacher, weight=None, tau=1.0):
    """(loss, bound, grad, bound) in 64 bits"""
    z = logits.double() / tau
    rows, q = z.shape
    k = ids.shape[1]
    lse = torch.logsumexp(z, 1)
    loss, lb = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad = torch.zeros_like(z) if weight is not None else None
    gb = torch.zeros_like(z) if weight is not None else None
    for r in range(rows):
        ok = (ids[r] >= 0) & (ids[r] < q) & (teacher[r] > -torch.inf)
        at = ids[r][ok].long()
        if not at.numel():
            continue
        t = teacher[r][ok].double() / tau
        logp = torch.log_softmax(t, 0)
        p = logp.exp()
        terms = p * (logp - z[r, at] + lse[r])
        loss[r] = tau * tau * terms.sum()
        zmax = float(z[r][z[r] > -torch.inf].abs().max())
        spread = min(64.0, float(z[r].max() - z[r][z[r] > -torch.inf].min()))
        # lse: the scaled logits, exponentials and additions as in sampled();
        # p: the scaled teacher, e^x, the sum, the quotient; then the terms
        e_lse = EPS * (3 * zmax + 3 * spread + 2 * q / 2048 + 64)
        tspread = float(t.max() - t.min())
        e_p = EPS * (4 * float(t.abs().max()) + 2 * tspread + k / 256 + 32)
        size = (p * (logp.abs() + z[r, at].abs() + lse[r].abs())).sum()
        lb[r] = tau * tau * (e_lse + 2 * e_p * (1 + size) + EPS * (k / 256 + 32) * size)
        if weight is not None:
            f = abs(float(weight[r])) * tau
            sm = torch.exp(z[r] - lse[r])
            pk = torch.zeros(q, dtype=torch.float64).index_add_(0, at, p)
            grad[r] = float(weight[r]) * tau * (sm - pk)
            # softmax: lse's error, z's, the difference's, e^x; three products
            gb[r] = f * (sm * (e_lse + EPS * (4 * zmax + 16)) + pk * (e_p + EPS * (k + 8)))
    return loss, lb, grad, gb


def integers(x):
    """Rows as integers with a scale each, 1 / 127 and the quotients in f32."""
    xf = x.float()
    s = xf.abs().amax(1, keepdim=True) * torch.tensor(1 / 127)
    a = torch.round(xf / torch.where(s > 0, s, torch.ones(())))
    return a, s


def product(x, w, w_scale, bias=None):
    """(y, bound before the last rounding) in 64 bits"""
    a, s = integers(x)
    y = (a.double() @ w.double().t()) * s.double() * w_scale.double()
    bound = 4 * EPS * y.abs()  # the scale, the sum as f32, two products
    if bias is not None:
        y = y + bias.double()
        bound = bound + EPS * y.abs()
    return y, bound


def close(got, want, bound, what):
    """got within bound of want, plus the rounding to its own type."""
    assert got.shape == want.shape, what
    g = got.cpu().double()
    h = HALF_STEP[got.dtype]
    tiny = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}[got.dtype]
    same = (g == want) | (g.isnan() & want.isnan())
    # a value that the type's range does not hold
    over = want.abs() > torch.finfo(got.dtype).max * (1 - h)
    ok = same | ((g - want).abs() <= bound * (1 + h) + want.abs() * h + tiny) | (over & (g.sign() == want.sign()) & g.isinf())
    bad = (~ok).nonzero()
    assert not bad.numel(), (what, bad[:4].tolist(), [(float(g[tuple(i)]), float(want[tuple(i)])) for i in bad[:4]])
