"""The gated block and its gradient against their definitions in 64 bits
(hidden_reference.py): types, activations, sizes from one on, odd ones, strides,
padding that holds NaN, every kind of tile and splits of the reduction, other streams,
graphs."""
import math

import hidden_reference as ref
import pytest
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _rows(t, pad=0, shift=0):
    """t on the device as rows of a wider buffer of NaN, from element `shift` on"""
    rows, q = t.shape
    wide = torch.full((rows * (q + pad) + shift + 1,), math.nan, dtype=t.dtype, device="cuda")
    view = wide[shift:shift + rows * (q + pad)].view(rows, q + pad)[:, :q]
    view.copy_(t)
    return view


def _inputs(rows, k, n, dtype, seed=0, pad=0, shift=0):
    g = torch.Generator("cuda").manual_seed(seed + 7 * rows + k * 31 + n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = _rows(rand(rows, k).to(dtype), pad, shift)
    wg, wu = (_rows((rand(n, k) / math.sqrt(k)).to(dtype), pad, shift) for _ in range(2))
    return x, wg, wu, _rows(rand(rows, n).to(dtype), pad, shift)


def _check(device, x, wg, wu, dh, act):
    h, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
    want = ref.gated(x, wg, wu, act)
    for name, got in (("h", h), ("gate", gate), ("up", up)):
        assert got.dtype == (x.dtype if name == "h" else torch.float32) and got.is_contiguous()
        ref.close(got, *want[name], name)
    assert torch.equal(th.gated_linear(device, x, wg, wu, act), h)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    want = ref.gated_grad(dh, x, wg, wu, gate, up, act)
    for name, got in zip(("dx", "dw_gate", "dw_up"), grads):
        assert got.dtype == x.dtype
        ref.close(got, *want[name], name)
    none, dwg, dwu = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act, input_grad=False)
    assert none is None and torch.equal(dwg, grads[1]) and torch.equal(dwu, grads[2])


SIZES = [
    # rows, k, n
    (1, 1, 1), (1, 8, 1), (2, 3, 5), (1, 64, 32), (31, 65, 33), (33, 72, 95), (64, 128, 64), (7, 1000, 130),
    (65, 24, 1000), (257, 136, 260), (1000, 96, 384), (1, 4096, 700), (300, 64, 2048), (129, 4104, 24), (5, 2048, 2048),
]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_sizes(device, rows, k, n, dtype, act):
    log_case(f"gated {rows} {k} {n} {dtype} {act}")
    _check(device, *_inputs(rows, k, n, dtype), act)


@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (3, 5), (40, 8)])
@pytest.mark.parametrize("rows,k,n", [(3, 40, 48), (70, 200, 130), (513, 512, 264)])
def test_rows_of_wider_buffers(device, rows, k, n, pad, shift):
    """(NaN between the rows and behind the last)"""
    log_case(f"gated {rows} {k} {n} pad {pad} shift {shift}")
    _check(device, *_inputs(rows, k, n, BF16, pad=pad, shift=shift), "silu")


@pytest.mark.parametrize("rows,k,n", [(513, 320, 1100), (1100, 1024, 768), (2050, 520, 1032)])
def test_large_tiles(device, rows, k, n):
    log_case(f"gated {rows} {k} {n}")
    _check(device, *_inputs(rows, k, n, BF16), "silu")
    _check(device, *_inputs(rows, k, n, F16), "gelu")


def test_weights_of_other_strides(device):
    """one weight's rows lie otherwise than the other's, and a transposed one"""
    x, wg, wu, dh = _inputs(40, 64, 56, BF16)
    want = th.gated_linear(device, x, wg, wu)
    assert torch.equal(th.gated_linear(device, x, _rows(wg, 16), wu), want)
    assert torch.equal(th.gated_linear(device, x, wg, wu.t().contiguous().t()), want)
    assert torch.equal(th.gated_linear(device, x[:1].expand(40, 64), wg, wu), want[:1].expand(40, 56))


def test_out_and_no_rows(device):
    x, wg, wu, dh = _inputs(9, 64, 56, BF16)
    wide = torch.full((9, 60), 3.0, dtype=BF16, device="cuda")
    got = th.gated_linear(device, x, wg, wu, out=wide[:, :56])
    assert torch.equal(got, th.gated_linear(device, x, wg, wu)) and (wide[:, 56:] == 3.0).all()
    h, gate, up = th.gated_linear(device, x[:0], wg, wu, save=True)
    assert h.shape == gate.shape == (0, 56)
    dx, dwg, dwu = th.gated_linear_grad(device, dh[:0], x[:0], wg, wu, gate, up)
    assert dx.shape == (0, 64) and not dwg.any() and not dwu.any() and dwg.shape == dwu.shape == (56, 64)


@pytest.mark.parametrize("rows,k,n", [(70, 200, 130), (600, 264, 600)])
def test_infinities_stay_in_their_rows(device, rows, k, n):
    x, wg, wu, dh = _inputs(rows, k, n, BF16)
    want, gate, up = th.gated_linear(device, x, wg, wu, save=True)
    bad = x.clone()
    bad[1, 3], bad[rows - 1, k - 1] = math.inf, math.nan
    got = th.gated_linear(device, bad, wg, wu)
    ok = torch.ones(rows, dtype=torch.bool, device="cuda")
    ok[1] = ok[rows - 1] = False
    assert torch.equal(got[ok], want[ok]) and got[rows - 1].isnan().all() and not got[1].isfinite().any()
    # a gradient's row that is not finite reaches its own row of dx, and the weights
    dh2 = dh.clone()
    dh2[2, 5] = math.nan
    dx, dwg, dwu = th.gated_linear_grad(device, dh2, x, wg, wu, gate, up)
    clean = th.gated_linear_grad(device, dh, x, wg, wu, gate, up)
    ok[:] = True
    ok[2] = False
    units = torch.arange(n, device="cuda") != 5
    assert torch.equal(dx[ok], clean[0][ok]) and dx[2].isnan().all()
    assert torch.equal(dwg[units], clean[1][units]) and dwg[5].isnan().all()
    assert torch.equal(dwu[units], clean[2][units]) and dwu[5].isnan().all()


def test_gradient_by_differences(device):
    """the loss sum(dh h) along a direction: (f(t) - f(-t)) / 2t in 64 bits of the formula"""
    x, wg, wu, dh = _inputs(50, 48, 40, F16)
    _, gate, up = th.gated_linear(device, x, wg, wu, "gelu", save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, "gelu")
    g = torch.Generator("cuda").manual_seed(5)
    leaves = [t.double() for t in (x, wg, wu)]
    for i in range(3):
        way = torch.randn(leaves[i].shape, device="cuda", generator=g, dtype=torch.float64)

        def f(t):
            a, b, c = (v + t * way if j == i else v for j, v in enumerate(leaves))
            return float((ref.act(torch.mm(a, b.t().contiguous()), "gelu")[0] * torch.mm(a, c.t().contiguous()) * dh.double()).sum())

        want, got = (f(1e-5) - f(-1e-5)) / 2e-5, float((grads[i].double() * way).sum())
        # dz, du and the result: each half a step of f16; 8 of them of the norm
        norm = float((grads[i].double().norm() * way.norm()))
        assert abs(got - want) < 8 * 2.0**-11 * norm


def test_another_stream(device):
    x, wg, wu, dh = _inputs(300, 264, 200, BF16)
    want, gate, up = th.gated_linear(device, x, wg, wu, save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 1.0
        h, a, b = th.gated_linear(device, y, wg, wu, save=True)
        again = th.gated_linear_grad(device, dh * 1.0, y, wg, wu, a, b)
        copies = [t * 1.0 for t in (h, *again)]
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(copies, (want, *grads)))


def test_captured(device):
    """two captured calls that share nothing, replayed between eager ones on new inputs"""
    dev = th.Device(0)
    side = torch.cuda.Stream()
    dev.set_stream(side.cuda_stream)
    cases = [(37, 200, 130), (260, 264, 512)]
    ins = [_inputs(*c, BF16) for c in cases]
    step = lambda x, wg, wu, dh: (lambda h, a, b: (h, *th.gated_linear_grad(dev, dh, x, wg, wu, a, b)))(  # noqa: E731
        *th.gated_linear(dev, x, wg, wu, save=True))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in ins:
            step(*i)
    side.synchronize()
    graphs, outs = [], []
    for i in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(*i))
        graphs.append(graph)
    for turn in range(3):
        for i in ins:
            for t, new in zip(i, _inputs(i[0].shape[0], i[0].shape[1], i[1].shape[0], BF16, seed=turn + 1)):
                t.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for graph in graphs:
                graph.replay()
            eager = [step(*i) for i in ins]
            for graph in reversed(graphs):
                graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    del graphs
    torch.cuda.synchronize()
    dev.close()


@pytest.mark.parametrize("stride", [(1 << 22) - 8, 1 << 22])
def test_rows_far_apart(device, stride):
    """offsets that pass 32 bits, at the largest stride that tiles read as it lies and at
    the first that is copied"""
    rows, k, n = 600, 64, 72
    x, wg, wu, dh = _inputs(rows, k, n, BF16)
    wide = torch.empty((rows - 1) * stride + k, dtype=BF16, device="cuda")
    far = wide.as_strided((rows, k), (stride, 1))
    far.copy_(x)
    h, gate, up = th.gated_linear(device, x, wg, wu, save=True)
    assert torch.equal(th.gated_linear(device, far, wg, wu), h)
    for got, want in zip(th.gated_linear_grad(device, dh, far, wg, wu, gate, up), th.gated_linear_grad(device, dh, x, wg, wu, gate, up)):
        assert torch.equal(got, want)


def test_two_threads(device):
    """two devices' calls at once, each on its own stream, give what each gives alone"""
    import threading

    cases = [(70, 200, 130), (300, 264, 512)]
    ins = [_inputs(*c, BF16, seed=3) for c in cases]
    want = [th.gated_linear(device, x, wg, wu) for x, wg, wu, _ in ins]
    torch.cuda.synchronize()
    wrong, errors = [0, 0], []

    def work(i):
        try:
            dev, side = th.Device(0), torch.cuda.Stream()
            dev.set_stream(side.cuda_stream)
            with torch.cuda.stream(side):
                for _ in range(20):
                    x, wg, wu, _ = ins[i]
                    wrong[i] += int(not torch.equal(th.gated_linear(dev, x, wg, wu), want[i]))
            side.synchronize()
            dev.close()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and wrong == [0, 0]


def test_refuses_what_would_be_overwritten(device):
    x, wg, wu, _ = _inputs(64, 64, 64, BF16)
    for out in (x, wg, wu):
        with pytest.raises(th.ThrmlError, match="h must not be x or a weight"):
            th.gated_linear(device, x, wg, wu, out=out)


def test_tensors_that_require_a_gradient(device):
    x, wg, wu, dh = _inputs(9, 64, 64, BF16)
    x.requires_grad_(True)
    with pytest.raises(th.ThrmlError, match="x requires a gradient"):
        th.gated_linear(device, x, wg, wu)
    with torch.no_grad():
        _, gate, up = th.gated_linear(device, x, wg, wu, save=True)
    assert not any(t.requires_grad for t in th.gated_linear_grad(device, dh, x, wg, wu, gate, up))


@pytest.mark.parametrize("rows,k,n", [(5, 72, 90), (5, 70, 1000), (300, 264, 520)])
def test_large_f16_gradients(device, rows, k, n):
    """a loss scale that takes dz and du past 65504: results that are within it come out as
    exactly as ever, the others infinite, none NaN"""
    x, wg, wu, dh = _inputs(rows, k, n, F16)
    dh = (dh.float() * 13000).clamp(-60000, 60000).to(F16)
    x = x * 0.02  # (dw within the range)
    wg, wu = wg * 50, wu * 50
    _, gate, up = th.gated_linear(device, x, wg, wu, save=True)
    a, slope = ref.act(gate.double(), "silu")
    largest = max(float((dh.double() * up.double() * slope).abs().max()), float((dh.double() * a).abs().max()))
    assert largest > 65504
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up)
    # what is divided by 2^down is rounded in steps of at least 2^-24 times that
    step = ref.tiny(F16) * 2.0**(math.floor(math.log2(largest)) - 14)
    more = {"dx": step * (wg.double().abs() + wu.double().abs()).sum(0), "dw_gate": step * x.double().abs().sum(0)}
    more["dw_up"] = more["dw_gate"]
    for (name, (want, bound)), got in zip(ref.gated_grad(dh, x, wg, wu, gate, up, "silu").items(), grads):
        bound = bound + more[name] * 1.01
        assert not got.isnan().any()
        inside, outside = want.abs() + bound < 65504, want.abs() - bound > 65520
        assert inside.any()
        ref.close(got[inside], want[inside], bound[inside], name)
        assert got[outside].isinf().all()
