"""The operators around a learned head over q categories, as they are measured:
the cases, what a program holds before a call, one call, and what that call
cannot do without.

  process   logits -> penalties for the categories of a row's history, biases,
            temperature, mask of the allowed categories -> logits
  sample    the same, and the row's next category (Gumbel-argmax over given
            uniforms; greedy where the temperature is 0) with its log-probability
  distill   loss of a student's logits against a teacher's top K logits
            ("loss"), or loss and gradient ("grad")
  linear    the head's product: rows of activations, quantised to 8-bit
            integers with a scale each, times 8-bit weights with a scale for
            each output channel

`own` chooses between the operators' plain form in elementary torch operations
and this repository's kernels.  Both take what `prepare` gives.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one dialogue at its next token: latency
        dict(name="process_r1_q32768_bf16", op="process", rows=1, q=32768, dtype="bf16", out="bf16",
             history=512, bias=0, mask="shared", pad=0),
        # a batch under a grammar with a mask of its own for each row, an odd
        # number of categories, rows of a wider buffer, biases by category
        dict(name="process_r48_q131071_f16", op="process", rows=48, q=131071, dtype="f16", out="f32",
             history=2047, bias=300, mask="rows", pad=9),
        # many rows of f32 logits with long histories, no mask
        dict(name="process_r512_q65536_f32", op="process", rows=512, q=65536, dtype="f32", out="f32",
             history=8192, bias=16, mask="none", pad=0),
        # a few dialogues answered one token at a time
        dict(name="sample_r4_q32768_bf16", op="sample", rows=4, q=32768, dtype="bf16", history=256,
             bias=0, mask="none", pad=0),
        # ragged sizes, masks of rows, some rows greedy
        dict(name="sample_r37_q50001_f16", op="sample", rows=37, q=50001, dtype="f16", history=1000,
             bias=64, mask="rows", pad=3),
        # a full serving batch over a large set of categories
        dict(name="sample_r256_q131072_bf16", op="sample", rows=256, q=131072, dtype="bf16",
             history=4096, bias=0, mask="shared", pad=0),
        # evaluation of a student on a held-out batch
        dict(name="distill_loss_r256_q65536_f32_k64", op="distill", grad=False, rows=256, q=65536,
             dtype="f32", k=64, tau=1.0, pad=0),
        # a training step with odd sizes and a softened teacher
        dict(name="distill_grad_r1021_q50001_f16_k33", op="distill", grad=True, rows=1021, q=50001,
             dtype="f16", k=33, tau=2.0, pad=0),
        # the training step of a large head
        dict(name="distill_grad_r2048_q131072_bf16_k128", op="distill", grad=True, rows=2048, q=131072,
             dtype="bf16", k=128, tau=1.0, pad=0),
        # the head for one token: the weights are read once
        dict(name="linear_r1_k4096_q32768_bf16", op="linear", rows=1, k=4096, q=32768, dtype="bf16",
             out="bf16", bias=False),
        # a ragged batch, odd inner size and number of categories
        dict(name="linear_r33_k1000_q50001_f16", op="linear", rows=33, k=1000, q=50001, dtype="f16",
             out="f32", bias=True),
        # scoring of a long prompt: a large product
        dict(name="linear_r4096_k4096_q16384_bf16", op="linear", rows=4096, k=4096, q=16384,
             dtype="bf16", out="bf16", bias=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["process", "sample", "distill", "linear"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "linear":
        rows, k = _spread(rng, 1, 4096), _spread(rng, 64, 8192)
        most = min(65536, (1 << 28) // k, 250_000_000_000 // (rows * k))
        return dict(op=op, rows=rows, k=k, q=_spread(rng, 64, most), dtype=dtype,
                    out=rng.choice(["f32", dtype]), bias=rng.random() < 0.5)
    q = _spread(rng, 1000, 131072)
    if op == "distill":
        return dict(op=op, grad=rng.random() < 0.7, rows=_spread(rng, 1, min(2048, (1 << 28) // q)), q=q,
                    dtype=dtype, k=_spread(rng, 1, 256), tau=rng.choice([1.0, 1.0, 2.0, 0.5]),
                    pad=rng.choice([0, 0, 1, 8]))
    c = dict(op=op, rows=_spread(rng, 1, min(512, (1 << 25) // q)), q=q, dtype=dtype,
             history=rng.choice([0, _spread(rng, 1, 8192)]), bias=rng.choice([0, _spread(rng, 1, 300)]),
             mask=rng.choice(["none", "shared", "rows"]), pad=rng.choice([0, 0, 1, 8]))
    if op == "process":
        c["out"] = rng.choice(["f32", dtype])
    return c


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(g, rows, q, dtype, pad):
    """Logits of a head: a few units wide, in rows of q + pad elements."""
    wide = torch.empty(rows, q + pad, dtype=DTYPES[dtype], device="cuda").normal_(0.0, 2.5, generator=g)
    return wide[:, :q]


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = _generator(seed)
    rows, q = case["rows"], case["q"]
    s = dict(case)
    if case["op"] == "linear":
        k = case["k"]
        x = torch.randn(rows, k, device="cuda", generator=g)
        # some channels of real activations are many times the others
        s["x"] = (x * (1.0 + 20.0 * (_rand(g, k) < 0.01))).to(DTYPES[case["dtype"]])
        w = torch.empty(q, k, dtype=torch.bfloat16, device="cuda").normal_(0.0, 36.0, generator=g)
        s["w"] = w.clamp_(-127, 127).round_().to(torch.int8)
        s["w_scale"] = (0.5 + _rand(g, q)) * (0.03 / math.sqrt(k))
        s["b"] = torch.randn(q, device="cuda", generator=g) * 0.1 if case["bias"] else None
        return s
    s["logits"] = _logits(g, rows, q, case["dtype"], case["pad"])
    if case["op"] == "distill":
        k = case["k"]
        # distinct categories: a progression from a random start
        step = max(1, (q - 1) // k)
        start = (_rand(g, rows, 1) * q).long()
        ids = (start + step * torch.arange(k, device="cuda")) % q
        # rows of fewer candidates are filled up with -1, some rows have none
        n = (k * (0.5 + 0.6 * _rand(g, rows, 1))).ceil().clamp(max=k)
        n = torch.where(_rand(g, rows, 1) < 0.02, torch.zeros_like(n), n)
        s["ids"] = torch.where(torch.arange(k, device="cuda") < n, ids, -1).to(torch.int32)
        s["teacher"] = torch.randn(rows, k, device="cuda", generator=g) * 3.0
        # a mean over the rows; f16 gradients carry a loss scale
        s["weight"] = (_rand(g, rows) + 0.5) * ((65536.0 if case["dtype"] == "f16" else 1.0) / rows)
        return s
    h, b = case["history"], case["bias"]
    # a history repeats its frequent categories
    s["history"] = (_rand(g, rows, h) ** 3 * q).to(torch.int32) if h else None
    s["lengths"] = ((0.5 + 0.5 * _rand(g, rows)) * h).to(torch.int32) if h else None
    s["prompt_lengths"] = (0.4 * _rand(g, rows) * h).to(torch.int32) if h else None
    s["repetition"] = 1.0 + 0.3 * _rand(g, rows) if h else None
    s["presence"] = 0.5 * _rand(g, rows) if h else None
    s["frequency"] = 0.2 * _rand(g, rows) if h else None
    if b:
        step = max(1, (q - 1) // b)
        ids = ((_rand(g, rows, 1) * q).long() + step * torch.arange(b, device="cuda")) % q
        s["bias_ids"] = torch.where(_rand(g, rows, b) < 0.1, -1, ids).to(torch.int32)
        s["bias_values"] = torch.randn(rows, b, device="cuda", generator=g) * 2.0
    else:
        s["bias_ids"] = s["bias_values"] = None
    t = 0.5 + _rand(g, rows)
    s["temperature"] = torch.where(_rand(g, rows) < 0.2, torch.zeros_like(t), t)
    if case["mask"] == "none":
        s["mask"] = None
    else:
        n, words = (1 if case["mask"] == "shared" else rows), (q + 31) // 32
        low, high = (torch.randint(0, 1 << 16, (n, words), device="cuda", generator=g) for _ in range(2))
        bits = low | high << 16
        s["mask"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    if case["op"] == "sample":
        s["u"] = _rand(g, rows, q)
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _processed(s):
    x = s["logits"].float()
    rows, q = x.shape
    if s["history"] is not None:
        at = torch.arange(s["history"].shape[1], device="cuda")
        live = at < s["lengths"][:, None]
        drawn = live & (at >= s["prompt_lengths"][:, None])
        ids = s["history"].long()
        # column q takes what does not count
        seen = torch.zeros(rows, q + 1, dtype=torch.bool, device="cuda")
        seen.scatter_(1, torch.where(live, ids, q), True)
        n = torch.zeros(rows, q + 1, device="cuda")
        n.scatter_add_(1, torch.where(drawn, ids, q), torch.ones_like(ids, dtype=torch.float32))
        seen, n = seen[:, :q], n[:, :q]
        theta = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / theta, x * theta), x)
        x = x - s["frequency"][:, None] * n
        x = torch.where(n > 0, x - s["presence"][:, None], x)
    if s["bias_ids"] is not None:
        b = torch.zeros(rows, q + 1, device="cuda")
        ids = s["bias_ids"].long()
        b.scatter_(1, torch.where(ids >= 0, ids, q), s["bias_values"])
        x = x + b[:, :q]
    t = s["temperature"][:, None]
    x = torch.where(t > 0, x / t, x)
    if s["mask"] is not None:
        bits = s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1
        x = torch.where(bits.flatten(1)[:, :q] != 0, x, -math.inf)
    return x


def _sampled(s):
    x = _processed(s)
    q = x.shape[1]
    # scores in 64 bits: which of two near ones is larger must not depend on rounding
    noise = -torch.log(-torch.log(s["u"].double()))
    score = torch.where(s["temperature"][:, None] > 0, x + noise, x.double())
    best = score.amax(1, keepdim=True)
    index = torch.where(score == best, torch.arange(q, device="cuda"), q).amin(1)
    m = x.amax(1)
    lse = m + torch.log(torch.exp(x - m[:, None]).sum(1))
    return {"index": index.to(torch.int32), "logprob": x.gather(1, index[:, None])[:, 0] - lse}


def _distilled(s):
    tau = s["tau"]
    z = s["logits"].float() / tau
    m = z.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    valid = s["ids"] >= 0
    ids = torch.where(valid, s["ids"], 0).long()
    t = torch.where(valid, s["teacher"] / tau, -math.inf)
    top = torch.where(valid.any(1, keepdim=True), t.amax(1, keepdim=True), 0.0)
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    p = torch.where(valid, e / total, 0.0)
    logp = torch.where(valid, t - top - torch.log(total), 0.0)
    loss = tau * tau * (p * (logp - (z.gather(1, ids) - lse))).sum(1)
    if not s["grad"]:
        return {"loss": loss}
    grad = torch.exp(z - lse) * (total > 0)
    grad.scatter_add_(1, ids, -p)
    grad *= tau * s["weight"][:, None]
    return {"loss": loss, "grad": grad.to(s["logits"].dtype)}


def _product(s):
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127.0
    a = torch.round(x / torch.where(scale > 0, scale, 1.0))
    y = a @ s["w"].float().T * scale * s["w_scale"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["out"]])


# ---------------------------------------------------------------------------
# The framework's calls

_device = []


def _framework():
    """The package and a program's device, on the stream that torch works on."""
    if not _device:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "thrml-rs_amd"))
        import thrml_hip

        dev = thrml_hip.Device(torch.cuda.current_device())
        dev.set_stream(torch.cuda.current_stream().cuda_stream)
        _device.extend([thrml_hip, dev])
    return _device


_ROW_ARGS = ("history", "lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias_ids",
             "bias_values", "temperature", "mask")


def _own(s):
    th, dev = _framework()
    op = s["op"]
    if op == "process":
        return th.process_logits(dev, s["logits"], out_dtype=DTYPES[s["out"]], **{n: s[n] for n in _ROW_ARGS})
    if op == "sample":
        index, logprob = th.sample_logits(dev, s["logits"], s["u"], **{n: s[n] for n in _ROW_ARGS})
        return {"index": index, "logprob": logprob}
    if op == "distill":
        if not s["grad"]:
            return {"loss": th.distill_loss(dev, s["logits"], s["ids"], s["teacher"], s["tau"])}
        loss, grad = th.distill_grad(dev, s["logits"], s["ids"], s["teacher"], s["weight"], s["tau"])
        return {"loss": loss, "grad": grad}
    return th.linear_i8(dev, s["x"], s["w"], s["w_scale"], bias=s["b"], out_dtype=DTYPES[s["out"]])


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "process":
        return _processed(state).to(DTYPES[state["out"]])
    if op == "sample":
        return _sampled(state)
    if op == "distill":
        return _distilled(state)
    return _product(state)


def work(case):
    """Bytes: every input once and every output once.  Operations: the product's
    multiplications and additions, or a few for each logit."""
    rows, q = case["rows"], case["q"]
    size = SIZES[case["dtype"]]
    if case["op"] == "linear":
        k = case["k"]
        bytes_ = rows * k * size + q * k + 4 * q * (2 if case["bias"] else 1) + rows * q * SIZES[case["out"]]
        return {"bytes": bytes_, "flops": 2.0 * rows * k * q}
    if case["op"] == "distill":
        n = rows * q
        return {"bytes": n * size * (2 if case["grad"] else 1) + 8 * rows * case["k"] + 8 * rows,
                "flops": (8.0 if case["grad"] else 5.0) * n}
    masks = {"none": 0, "shared": 1, "rows": rows}[case["mask"]]
    lists = 4 * rows * case["history"] + 8 * rows * case["bias"] + 4 * masks * ((q + 31) // 32)
    if case["op"] == "process":
        return {"bytes": rows * q * (size + SIZES[case["out"]]) + lists + 24 * rows, "flops": 4.0 * rows * q}
    return {"bytes": rows * q * (size + 4) + lists + 32 * rows, "flops": 12.0 * rows * q}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_row_values(s):
    """Every logit's own value, by what its category's entries say of it."""
    z = s["logits"].double()
    rows, q = z.shape
    row = torch.arange(rows, device=z.device)[:, None]
    if s["history"] is not None:
        h = s["history"].shape[1]
        key = (row * q + s["history"]).flatten()
        place = torch.arange(h, device=z.device).expand(rows, h).flatten()
        ends = s["lengths"].long().repeat_interleave(h)
        begins = s["prompt_lengths"].long().repeat_interleave(h)
        occurs = torch.bincount(key[place < ends], minlength=rows * q).view(rows, q)
        drawn = torch.bincount(key[(place < ends) & (place >= begins)], minlength=rows * q).view(rows, q)
        theta = s["repetition"].double()[:, None]
        factor = torch.where(z > 0, 1.0 / theta, theta)
        z = z * torch.where(occurs > 0, factor, torch.ones_like(factor))
        z = z - drawn * s["frequency"].double()[:, None] - (drawn > 0) * s["presence"].double()[:, None]
    if s["bias_ids"] is not None:
        ok = s["bias_ids"] >= 0
        at = (row * q + s["bias_ids"])[ok]
        z = z.clone()
        z.view(-1)[at] += s["bias_values"].double()[ok]
    t = s["temperature"].double()[:, None]
    z = z / torch.where(t > 0, t, torch.ones_like(t))
    if s["mask"] is not None:
        j = torch.arange(q, device=z.device)
        allowed = s["mask"][:, j // 32] & (torch.ones_like(j) << (j % 32))
        z = z.masked_fill(allowed.expand(rows, q) == 0, -math.inf)
    return z


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "process":
        return _exact_row_values(s)
    if case["op"] == "sample":
        z = _exact_row_values(s)
        # the smallest of independent exponential waiting times with rates e^z
        wait = -torch.log(s["u"].double())
        clock = torch.where(s["temperature"][:, None] > 0, torch.log(wait) - z, -z)
        pick = clock.argmin(1)
        chosen = torch.take_along_dim(z, pick[:, None], 1)[:, 0]
        return {"index": None, "logprob": chosen - torch.logsumexp(z, 1)}
    if case["op"] == "distill":
        tau, rows, q = case["tau"], case["rows"], case["q"]
        z = s["logits"].double() / tau
        lse = torch.logsumexp(z, 1)
        ok = s["ids"] >= 0
        row = torch.arange(rows, device=z.device)[:, None].expand_as(s["ids"])
        t = (s["teacher"].double() / tau).masked_fill(~ok, -math.inf)
        logp = torch.log_softmax(t, 1)[ok]  # rows without an entry have none here either
        at, owner = s["ids"][ok].long(), row[ok]
        terms = torch.exp(logp) * (logp - z[owner, at] + lse[owner])
        loss = torch.zeros(rows, dtype=torch.float64, device=z.device).index_add_(0, owner, terms) * tau**2
        if not case["grad"]:
            return {"loss": loss}
        z.sub_(lse[:, None]).exp_()
        z[~ok.any(1)] = 0.0
        z[owner, at] -= torch.exp(logp)
        return {"loss": loss, "grad": z.mul_((s["weight"].double() * tau)[:, None])}
    x = s["x"].double()
    peak = x.abs().max(1).values
    # the integers are those of the 32-bit quotients; the sum and the scales are in 64 bits
    step = (peak.float() / 127.0)[:, None]
    a = (s["x"].float() / step).round().double()
    y = torch.matmul(a, s["w"].double().t()) * torch.outer(peak / 127.0, s["w_scale"].double())
    return y if s["b"] is None else y + s["b"].double()
