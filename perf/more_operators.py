"""The operators of a learned head's hidden block, as they are measured: the
cases, what a program holds before a call, one call, and what that call cannot
do without.

  gated    hidden units act(x @ w_gate.T) * (x @ w_up.T) from rows of features
           ("forward"), or these and the gradients of a loss in the features and
           both weights ("train")
  dropout  units kept or zeroed by bits of a key's ChaCha8 stream, the kept ones
           scaled, plus a residual; without one it is the gradient's way back
  f8       the head's product in 8-bit floating point: activations quantised with
           a scale for each 128 of a row, weights with one for each 128 x 128

`own` chooses between the operators' plain form in elementary torch operations
and this repository's kernels.  Both take what `prepare` gives.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # the hidden units of one variable at its turn: the weights are read once
        dict(name="gated_r1_k4096_n16384_bf16", op="gated", train=False, rows=1, k=4096, n=16384,
             dtype="bf16", act="silu"),
        # a ragged batch answered at once, sizes that no tile divides
        dict(name="gated_r77_k1000_n2777_f16", op="gated", train=False, rows=77, k=1000, n=2777,
             dtype="f16", act="gelu"),
        # scoring of many states: a large product
        dict(name="gated_r4096_k4096_n8192_bf16", op="gated", train=False, rows=4096, k=4096, n=8192,
             dtype="bf16", act="silu"),
        # a step on the states of 4 chains of a 32 x 32 torus with 24 categories
        dict(name="gated_train_r4096_k96_n384_bf16", op="gated", train=True, rows=4096, k=96, n=384,
             dtype="bf16", act="silu"),
        # a step with odd sizes; f16 gradients carry a loss scale
        dict(name="gated_train_r1021_k2001_n5003_f16", op="gated", train=True, rows=1021, k=2001, n=5003,
             dtype="f16", act="gelu"),
        # the step of a large block
        dict(name="gated_train_r4096_k4096_n8192_bf16", op="gated", train=True, rows=4096, k=4096, n=8192,
             dtype="bf16", act="silu"),
        # a few variables: latency
        dict(name="dropout_r16_c4096_bf16", op="dropout", rows=16, cols=4096, dtype="bf16", p=0.1,
             residual=True, pad=0, first=0),
        # odd sizes in rows of a wider buffer, a part of a larger batch
        dict(name="dropout_r1021_c5003_f32", op="dropout", rows=1021, cols=5003, dtype="f32", p=0.5,
             residual=False, pad=9, first=2042),
        # the units of a large block
        dict(name="dropout_r4096_c16384_bf16", op="dropout", rows=4096, cols=16384, dtype="bf16", p=0.1,
             residual=True, pad=0, first=0),
        # the head for one variable: the weights are read once
        dict(name="f8_r1_k4096_q32768_bf16", op="f8", rows=1, k=4096, q=32768, dtype="bf16", out="bf16",
             bias=False),
        # a ragged batch, an inner size that ends inside a block, an odd number of categories
        dict(name="f8_r33_k1000_q50001_f16", op="f8", rows=33, k=1000, q=50001, dtype="f16", out="f32",
             bias=True),
        # scoring of many states: a large product
        dict(name="f8_r4096_k4096_q16384_bf16", op="f8", rows=4096, k=4096, q=16384, dtype="bf16",
             out="bf16", bias=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["gated", "gated", "dropout", "f8"])
    if op == "dropout":
        cols = _spread(rng, 24, 16384)
        return dict(op=op, rows=_spread(rng, 1, min(16384, (1 << 26) // cols)), cols=cols,
                    dtype=rng.choice(["bf16", "f16", "f32"]), p=rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)]),
                    residual=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 8]),
                    first=rng.choice([0, rng.randrange(1, 100000)]))
    rows, k = _spread(rng, 1, 4096), _spread(rng, 64, 8192)
    if rng.random() < 0.5:
        k = (k + 15) // 16 * 16
    if op == "f8":
        most = min(65536, (1 << 28) // k, 250_000_000_000 // (rows * k))
        dtype = rng.choice(["bf16", "f16", "f32"])
        return dict(op=op, rows=rows, k=k, q=_spread(rng, 64, most), dtype=dtype, out=rng.choice(["f32", dtype]),
                    bias=rng.random() < 0.5)
    most = min(16384, (1 << 26) // k, 130_000_000_000 // (rows * k))
    n = _spread(rng, 64, most)
    if rng.random() < 0.5:
        n = max(64, n // 16 * 16)
    return dict(op=op, train=rng.random() < 0.6, rows=rows, k=k, n=n, dtype=rng.choice(["bf16", "f16"]),
                act=rng.choice(["silu", "gelu", "relu"]))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    rows, dtype = case["rows"], DTYPES[case["dtype"]]
    if case["op"] == "dropout":
        cols, pad = case["cols"], case["pad"]
        for name in ("x", "residual") if case["residual"] else ("x",):
            s[name] = _randn(g, rows, cols + pad).to(dtype)[:, :cols]
        s["key"] = int(torch.randint(0, 1 << 62, (1,), device="cuda", generator=g))
        return s
    k = case["k"]
    if case["op"] == "gated":
        n = case["n"]
        s["x"] = _randn(g, rows, k).to(dtype)
        s["w_gate"], s["w_up"] = ((_randn(g, n, k) / math.sqrt(k)).to(dtype) for _ in range(2))
        if case["train"]:
            # a mean over the rows; f16 gradients carry a loss scale
            s["grad"] = (_randn(g, rows, n) * ((65536.0 if case["dtype"] == "f16" else 1.0) / rows)).to(dtype)
        return s
    q = case["q"]
    # some channels of real activations are many times the others
    large = 1.0 + 20.0 * (torch.rand(k, device="cuda", generator=g) < 0.01)
    s["x"] = (_randn(g, rows, k) * large).to(dtype)
    s["w"] = (_randn(g, q, k) * 100.0).clamp_(-448.0, 448.0).to(F8)
    blocks = (-(-q // 128), -(-k // 128))
    s["w_scale"] = (0.5 + torch.rand(*blocks, device="cuda", generator=g)) * (0.01 / math.sqrt(k))
    s["b"] = _randn(g, q) * 0.1 if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _act(z, name):
    """(act(z), act'(z))"""
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if name == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _gated(s):
    dtype = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    z, u = x @ wg.T, x @ wu.T
    a, slope = _act(z, s["act"])
    h = (a * u).to(dtype)
    if not s["train"]:
        return h
    grad = s["grad"].float()
    dz, du = grad * u * slope, grad * a
    dx = dz @ wg + du @ wu
    return {"h": h, "dx": dx.to(dtype), "dw_gate": (dz.T @ x).to(dtype), "dw_up": (du.T @ x).to(dtype)}


def _key_words(seed):
    """The 8 key words of a 64-bit seed: PCG32 with XSH-RR output."""
    words = []
    for _ in range(8):
        seed = (seed * 6364136223846793005 + 11634580027462260723) % (1 << 64)
        x, r = ((seed >> 18 ^ seed) >> 27) % (1 << 32), seed >> 59
        words.append((x >> r | x << (32 - r)) % (1 << 32))
    return words


def _signed(w):
    return w - (1 << 32) if w >= 1 << 31 else w


def _halves(seed, first, count):
    """Half words first .. first + count - 1 of the key's ChaCha8 stream (32 in a
    block of 64 bytes, the lower half of a word first), as int32."""
    b0, b1 = first // 32, (first + count + 31) // 32
    block = torch.arange(b0, b1, device="cuda")
    start = [0x61707865, 0x3320646E, 0x79622D32, 0x6B206574] + _key_words(seed)
    zero = torch.zeros(b1 - b0, dtype=torch.int32, device="cuda")
    start = [zero + _signed(w) for w in start]
    low = block & 0xFFFFFFFF
    start += [torch.where(low >= 1 << 31, low - (1 << 32), low).int(), (block >> 32).int(), zero, zero]
    v = list(start)

    def turn(d, a, n):
        d = d ^ a
        return d << n | (d >> (32 - n)) & ((1 << n) - 1)

    def quarter(a, b, c, d):
        for n, m in ((16, 12), (8, 7)):
            v[a] = v[a] + v[b]
            v[d] = turn(v[d], v[a], n)
            v[c] = v[c] + v[d]
            v[b] = turn(v[b], v[c], m)

    for _ in range(4):
        for i in range(4):
            quarter(i, 4 + i, 8 + i, 12 + i)
        for i in range(4):
            quarter(i, 4 + (i + 1) % 4, 8 + (i + 2) % 4, 12 + (i + 3) % 4)
    words = torch.stack([a + b for a, b in zip(v, start)], 1)
    halves = torch.stack([words & 0xFFFF, words >> 16 & 0xFFFF], 2).flatten()
    return halves[first - 32 * b0:first - 32 * b0 + count]


def _dropped(s):
    rows, cols = s["rows"], s["cols"]
    border = round(s["p"] * 65536)
    kept = (_halves(s["key"], s["first"] * cols, rows * cols) >= border).view(rows, cols)
    y = torch.where(kept, s["x"].float() * (65536.0 / (65536 - border)), 0.0)
    if torch.is_tensor(s["residual"]):
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _quantised(x):
    """(8-bit floats as f32, scale of each 128 of a row) of rows of f32"""
    rows, k = x.shape
    wide = torch.zeros(rows, (k + 127) // 128 * 128, device=x.device)
    wide[:, :k] = x
    blocks = wide.view(rows, -1, 128)
    scale = (blocks.abs().amax(2) * (1.0 / 448.0)).clamp(min=2.0**-126)
    return (blocks / scale[:, :, None]).to(F8).float(), scale


def _product(s):
    rows, k = s["x"].shape
    a, scale = _quantised(s["x"].float())
    x = (a * scale[:, :, None]).view(rows, -1)[:, :k]
    q = s["w"].shape[0]
    at = torch.arange(max(q, k), device="cuda") // 128
    w = s["w"].float() * s["w_scale"][at[:q, None], at[None, :k]]
    y = x @ w.T
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


def _own(s):
    th, dev = _framework()
    if s["op"] == "dropout":
        return th.dropout(dev, s["x"], th.RngKey(s["key"]), s["p"], first_row=s["first"],
                          residual=s["residual"] if torch.is_tensor(s["residual"]) else None)
    if s["op"] == "f8":
        return th.linear_f8(dev, s["x"], s["w"], s["w_scale"], bias=s["b"], out_dtype=DTYPES[s["out"]])
    if not s["train"]:
        return th.gated_linear(dev, s["x"], s["w_gate"], s["w_up"], s["act"])
    h, gate, up = th.gated_linear(dev, s["x"], s["w_gate"], s["w_up"], s["act"], save=True)
    dx, dw_gate, dw_up = th.gated_linear_grad(dev, s["grad"], s["x"], s["w_gate"], s["w_up"], gate, up, s["act"])
    return {"h": h, "dx": dx, "dw_gate": dw_gate, "dw_up": dw_up}


def run(state):
    if own:
        return _own(state)
    return {"gated": _gated, "dropout": _dropped, "f8": _product}[state["op"]](state)


def work(case):
    """Bytes: every input once and every output once.  Operations: the products'
    multiplications and additions; for dropout a few for each unit, and the
    generator's 400 for 32 of them."""
    rows, size = case["rows"], SIZES[case["dtype"]]
    if case["op"] == "dropout":
        n = rows * case["cols"]
        return {"bytes": n * size * (3 if case["residual"] else 2), "flops": 16.0 * n}
    k = case["k"]
    if case["op"] == "f8":
        q = case["q"]
        scales = 4 * -(-q // 128) * -(-k // 128)
        return {"bytes": rows * k * size + q * k + scales + (4 * q if case["bias"] else 0) + rows * q * SIZES[case["out"]],
                "flops": 2.0 * rows * k * q}
    n = case["n"]
    ends = rows * k + 2 * n * k + rows * n
    return {"bytes": size * ends * (2 if case["train"] else 1), "flops": 4.0 * rows * k * n * (3 if case["train"] else 1)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _keep_bits(seed, first, count):
    """numpy: the stream's half words as they lie in memory on a little-endian host."""
    b0, b1 = first // 32, (first + count + 31) // 32
    counter = np.arange(b0, b1, dtype=np.uint64)
    m = np.zeros((4, 4, b1 - b0), np.uint32)
    m[0] = np.frombuffer(b"expand 32-byte k", np.uint32)[:, None]
    s = np.uint64(seed)
    with np.errstate(over="ignore"):
        for i in range(8):
            s = s * np.uint64(6364136223846793005) + np.uint64(11634580027462260723)
            x = np.uint32((s ^ s >> np.uint64(18)) >> np.uint64(27) & np.uint64(0xFFFFFFFF))
            r = np.uint32(s >> np.uint64(59))
            m[1 + i // 4, i % 4] = x >> r | x << (np.uint32(32) - r & np.uint32(31))
        m[3, 0], m[3, 1] = counter & np.uint64(0xFFFFFFFF), counter >> np.uint64(32)
        a, b, c, d = (m[i].copy() for i in range(4))

        def rot(v, n):
            return v << np.uint32(n) | v >> np.uint32(32 - n)

        for half in range(8):  # a column round, then a diagonal one
            a += b
            d = rot(d ^ a, 16)
            c += d
            b = rot(b ^ c, 12)
            a += b
            d = rot(d ^ a, 8)
            c += d
            b = rot(b ^ c, 7)
            way = 1 if half % 2 == 0 else -1
            b, c, d = np.roll(b, -way, 0), np.roll(c, -2 * way, 0), np.roll(d, -3 * way, 0)
        out = np.stack([a, b, c, d]) + m
    bits = np.ascontiguousarray(out.reshape(16, -1).T).view(np.uint16).reshape(-1)
    return bits[first - 32 * b0:][:count]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        border = round(case["p"] * 65536)
        bits = _keep_bits(s["key"], case["first"] * cols, rows * cols)
        drop = torch.from_numpy(bits < border).cuda().view(rows, cols)
        y = (s["x"].double() / (1.0 - border / 65536)).masked_fill(drop, 0.0)
        return y.add_(s["residual"].double()) if case["residual"] else y
    if case["op"] == "f8":
        x, (rows, k), q = s["x"].float(), s["x"].shape, case["q"]
        y = torch.zeros(rows, q, dtype=torch.float64, device="cuda")
        for i in range(0, k, 128):
            part = x[:, i:i + 128]
            # the 8-bit values are those of the 32-bit quotients; products and sums are in 64 bits
            step = torch.clamp(part.abs().max(1, keepdim=True).values * torch.tensor(1.0 / 448.0, device="cuda"), min=2.0**-126)
            a = torch.div(part, step).to(F8).double() * step.double()
            w = s["w"][:, i:i + 128].double() * s["w_scale"][:, i // 128].double().repeat_interleave(128)[:q, None]
            y.addmm_(a, w.t().contiguous())
        return y if s["b"] is None else y + s["b"].double()
    leaves = [s[n].double().requires_grad_(case["train"]) for n in ("x", "w_gate", "w_up")]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[case["act"]]
    x, wg, wu = leaves
    h = act(torch.mm(x, wg.t())) * torch.mm(x, wu.t())
    if not case["train"]:
        return h
    dx, dwg, dwu = torch.autograd.grad(h, leaves, s["grad"].double())
    return {"h": h.detach(), "dx": dx, "dw_gate": dwg, "dw_up": dwu}
