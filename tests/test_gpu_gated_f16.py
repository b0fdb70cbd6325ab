"""Gradients of the gated block in f16 at the edge of the type's range: which results are
infinite, next to 65520 too, and rows and units of very different size, against the
definition in 64 bits (hidden_reference.py) from the z and u that the forward call kept."""
import math

import hidden_reference as ref
import pytest
import test_gpu_hidden_tiles as tiles
import torch
from conftest import log_case

import thrml_hip as th

pytestmark = pytest.mark.gpu

F16 = torch.float16
BORDER = 65520.0  # what is rounded to f16 from here on is infinite


def _inputs(rows, k, n, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + 7 * rows + k * 31 + n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = rand(rows, k).to(F16)
    wg, wu = ((rand(n, k) / math.sqrt(k)).to(F16) for _ in range(2))
    return x, wg, wu, rand(rows, n)


def _exact(dh, x, wg, wu, z, u, act):
    """{name: (value, error of f32)}: what an f32 computation of dz and du (16 roundings of
    its factors, as in hidden_reference.gated_grad) leaves of each result, sums in 64 bits"""
    dh, x, wg, wu, z, u = (t.double() for t in (dh, x, wg, wu, z, u))
    a, slope = ref.act(z, act)
    dz, du = dh * u * slope, dh * a
    ez, eu = 16 * ref.U32 * (dh * u).abs() * (1 + z.abs()), 16 * ref.U32 * (dh * z).abs()
    dzt, dut, ezt, eut = (t.t().contiguous() for t in (dz, du, ez, eu))
    return {"dx": (torch.mm(dz, wg) + torch.mm(du, wu), torch.mm(ez, wg.abs()) + torch.mm(eu, wu.abs())),
            "dw_gate": (torch.mm(dzt, x), torch.mm(ezt, x.abs())), "dw_up": (torch.mm(dut, x), torch.mm(eut, x.abs()))}


# rows, k, n, what the gradients are multiplied by: in each some per cent of the results of dx,
# of the weights' gradients or of both pass the range; every kind of tile, with a split
# reduction and without, operands that are copied, and few rows
STEPS = [
    (5, 7040, 2000, 13107.0), (1, 264, 4104, 40000.0), (13, 2000, 1003, 20000.0), (40, 264, 392, 9000.0),
    (300, 264, 520, 5000.0), (600, 1032, 600, 2000.0), (65, 136, 6000, 8000.0), (520, 1032, 2056, 2500.0), (2050, 136, 136, 4000.0),
]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,n,size", STEPS)
def test_what_passes_the_range(device, rows, k, n, size, act):
    """infinite exactly where the definition is, but for what f32 cannot tell from 65520"""
    log_case(f"f16 range {rows} {k} {n} {size} {act}")
    x, wg, wu, dh = _inputs(rows, k, n)
    dh = (dh * size).clamp(-65504, 65504).to(F16)
    _, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    near = passed = 0
    for (name, (want, err)), got in zip(_exact(dh, x, wg, wu, gate, up, act).items(), grads):
        assert not got.isnan().any(), name
        told = (want.abs() - BORDER).abs() > err
        wrong = told & (got.isinf() != (want.abs() >= BORDER))
        assert not wrong.any(), (name, int(wrong.sum()), want[wrong][:5].tolist(), got[wrong][:5].tolist())
        assert ((got > 0) == (want > 0))[got.isinf()].all(), name
        near += int(((want.abs() - BORDER).abs() < 32.0).sum())
        passed += int((want.abs() >= BORDER).sum())
    assert near > 0 and passed > 0, "the case does not come near the border"


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,n", [(24, 72, 392), (300, 264, 520), (600, 1032, 600), (129, 4104, 24), (65, 136, 6000)])
def test_what_is_within_the_range_among_results_far_beyond_it(device, rows, k, n, act):
    """most results are some hundred times the range: the rounding of dz and du moves those
    within it by more than the range"""
    log_case(f"f16 far beyond {rows} {k} {n} {act}")
    x, wg, wu, dh = _inputs(rows, k, n)
    x, wg, wu, dh = x * 8, wg * 4, wu * 16, (dh * 16384).clamp(-65504, 65504).to(F16)
    _, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    within = 0
    for (name, (want, err)), got in zip(_exact(dh, x, wg, wu, gate, up, act).items(), grads):
        told = (want.abs() - BORDER).abs() > err
        wrong = told & (got.isinf() != (want.abs() >= BORDER))
        assert not got.isnan().any() and not wrong.any(), (name, int(wrong.sum()), want[wrong][:5].tolist(), got[wrong][:5].tolist())
        within += int((told & (want.abs() < BORDER)).sum())
    assert within > 0


def _down(largest):
    """by what power of two dz and du are divided whose largest magnitude is this"""
    return torch.where(largest > 65504, torch.floor(torch.log2(largest.clamp(min=1))) - 14, torch.zeros_like(largest))


def _compare(device, dh, x, wg, wu, act):
    """every result within what its own row's and unit's rounding of dz and du allows"""
    _, gate, up = th.gated_linear(device, x, wg, wu, act, save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, act)
    a, slope = ref.act(gate.double(), act)
    dz, du = (dh.double() * t for t in (up.double() * slope, a))
    # (a value next to a power of two may be rounded to it)
    scales = {"dx": torch.maximum(dz.abs().amax(1), du.abs().amax(1)), "dw_gate": dz.abs().amax(0), "dw_up": du.abs().amax(0)}
    least = {n: (ref.tiny(F16) * 2.0**_down(s * (1 + 2.0**-20)))[:, None] for n, s in scales.items()}
    assert max(float(s.max()) for s in scales.values()) > 65504 * 64
    other = {"dx": wg.double().abs().sum(0) + wu.double().abs().sum(0), "dw_gate": x.double().abs().sum(0)}
    other["dw_up"] = other["dw_gate"]
    exact = _exact(dh, x, wg, wu, gate, up, act)
    finite = 0
    for (name, (want, bound)), got in zip(ref.gated_grad(dh, x, wg, wu, gate, up, act).items(), grads):
        bound = bound + least[name] * other[name]
        assert not got.isnan().any(), name
        told = (want.abs() - BORDER).abs() > exact[name][1]
        assert not (told & (got.isinf() != (want.abs() >= BORDER))).any(), name
        fine = got.isfinite()
        finite += int(fine.sum())
        if fine.any():
            ref.close(got[fine], want[fine], bound[fine], name)
    assert finite


SHAPES = [(5, 72, 90), (24, 72, 392), (40, 264, 392), (300, 264, 520), (600, 1032, 600), (65, 136, 6000), (129, 4104, 24), (1, 264, 4104)]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_rows_of_different_size(device, rows, k, n, act):
    """a row whose dz and du pass the range does not take the bits of the others, whose
    gradients are 2^20 and 2^30 times smaller"""
    log_case(f"f16 rows {rows} {k} {n} {act}")
    x, wg, wu, dh = _inputs(rows, k, n)
    size = torch.full((rows,), 2.0**-6, device="cuda")
    size[1::3] = 2.0**-15
    size[::7] = 2.0**14
    dh = (dh * size[:, None]).clamp(-65504, 65504)
    _compare(device, dh.to(F16), x * 16, wg * 8, wu * 64, act)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_units_of_different_size(device, rows, k, n, act):
    """a unit whose dz and du pass the range does not take the bits of the others"""
    log_case(f"f16 units {rows} {k} {n} {act}")
    x, wg, wu, dh = _inputs(rows, k, n)
    dh = dh * 2.0**-10
    dh[:, ::5] *= 2.0**20
    dh[:, 1::5] *= 2.0**-4
    large = torch.ones(n, 1, device="cuda", dtype=F16)
    large[::5] = 512
    _compare(device, dh.to(F16), x * 16, wg * 8, wu * large * 8, act)


def test_an_infinite_unit_beside_one_that_passes_the_range(device):
    """dz = inf of one unit (x and the weights at the type's end) does not hide from the
    choice of the power of two that du of the same unit passes the range"""
    x = torch.full((3, 64), 60000.0, device="cuda", dtype=F16)
    wg = torch.full((8, 64), 1e-3, device="cuda", dtype=F16)
    wu = torch.full((8, 64), 1e-3, device="cuda", dtype=F16)
    dh = torch.full((3, 8), 64.0, device="cuda", dtype=F16)
    h, gate, up = th.gated_linear(device, x, wg, wu, "relu", save=True)
    gate[:, [0, 1, 3, 4, 5, 6, 7]] = 1.0
    up[:, 2] = math.inf  # (only there du passes the range, and dz beside it is infinite)
    dx, dwg, dwu = th.gated_linear_grad(device, dh, x * 2.0**-24, wg, wu, gate, up, "relu")
    du = dh.double() * gate.double()
    want = torch.mm(du.t().contiguous(), (x * 2.0**-24).double())
    assert float(du.abs().max()) > 65504 and float(want.abs().max()) < 65504
    assert dwg[2].isinf().all() and not dwg[2].isnan().any()
    err = (dwu.double() - want).abs()
    assert (err <= 8 * 2.0**-11 * want.abs()).all()


def test_captured(device):
    """a captured step, replayed on gradients that pass the range and that do not, in turn"""
    dev = th.Device(0)
    side = torch.cuda.Stream()
    dev.set_stream(side.cuda_stream)
    cases = [(300, 264, 520), (13, 1000, 1003)]
    ins = [[*_inputs(*c)] for c in cases]
    for i in ins:
        i[3] = i[3].to(F16)
    step = lambda x, wg, wu, dh: (lambda h, a, b: th.gated_linear_grad(dev, dh, x, wg, wu, a, b))(  # noqa: E731
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
    infinite = []
    for turn in range(4):
        for c, i in zip(cases, ins):
            for t, new in zip(i, _inputs(*c, seed=turn + 1)):
                t.copy_((new * 9000).clamp(-65504, 65504) if t is i[3] and turn % 2 else new)
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
        infinite.append(any(bool(t.isinf().any()) for want in eager for t in want))
    assert infinite == [False, True, False, True]
    del graphs
    torch.cuda.synchronize()
    dev.close()


@pytest.mark.parametrize("which,tile", [*(("dx", t) for t in tiles.INPUT), *(("dw", t) for t in tiles.WEIGHT)])
def test_every_kind_of_tile_at_the_border(device, which, tile):
    """the border lies at about two typical results of the product that reaches the tile"""
    rows, k, n = (tiles.INPUT if which == "dx" else tiles.WEIGHT)[tile]
    log_case(f"f16 border {which} {tile}")
    x, wg, wu, dh = _inputs(rows, k, n)
    wg, wu = wg * 16, wu * 16
    # dz and du are about 8 times dh
    typical = 8 * (16 * math.sqrt(2 * n / k) if which == "dx" else math.sqrt(rows))
    dh = (dh * (BORDER / 2 / typical)).clamp(-65504, 65504).to(F16)
    _, gate, up = th.gated_linear(device, x, wg, wu, "silu", save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, "silu")
    exact = _exact(dh, x, wg, wu, gate, up, "silu")
    for (name, (want, err)), got in zip(exact.items(), grads):
        told = (want.abs() - BORDER).abs() > err
        wrong = told & (got.isinf() != (want.abs() >= BORDER))
        assert not got.isnan().any() and not wrong.any(), (name, int(wrong.sum()), want[wrong][:5].tolist(), got[wrong][:5].tolist())
    for name in ("dx",) if which == "dx" else ("dw_gate", "dw_up"):
        want = exact[name][0]
        # (0.9 % of them are within 2 % of the border, of 1353 and more)
        assert (want.abs() >= BORDER).any() and ((want.abs() - BORDER).abs() < 0.02 * BORDER).any(), name


@pytest.mark.parametrize("rows,k,n,size", [(4, 4096, 1000, 9000.0), (40, 264, 392, 9000.0), (600, 1032, 600, 2000.0)])
def test_infinite_gradients_stay_in_their_rows_and_units(device, rows, k, n, size):
    """and do not make the finite results beside them near the border, nor far from it"""
    log_case(f"f16 infinite dh {rows} {k} {n}")
    x, wg, wu, dh = _inputs(rows, k, n)
    dh = (dh * size).clamp(-65504, 65504).to(F16)
    dh[1, 5] = math.inf
    _, gate, up = th.gated_linear(device, x, wg, wu, "silu", save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, "silu")
    dh[1, 5] = 0.0
    clean = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, "silu")
    for (name, (want, err)), got, without in zip(_exact(dh, x, wg, wu, gate, up, "silu").items(), grads, clean):
        bad = 1 if name == "dx" else 5
        assert not got[bad].isfinite().any(), name
        rest = torch.arange(len(got), device="cuda") != bad
        told = ((want.abs() - BORDER).abs() > err) & rest[:, None]
        assert not (told & (got.isinf() != (want.abs() >= BORDER))).any(), name
        assert torch.equal(got[rest], without[rest]), name


@pytest.mark.parametrize("rows,k,n,size", [(2, 3, 4000, 25000.0), (3, 1, 3000, 20000.0), (40, 7, 2500, 8000.0), (300, 9, 1003, 3000.0), (4000, 5, 70, 900.0)])
def test_few_features_at_the_border(device, rows, k, n, size):
    """rows of fewer columns than a wave takes together, in wider buffers of NaN"""
    log_case(f"f16 few features {rows} {k} {n}")
    x, wg, wu, dh = _inputs(rows, k, n)
    dh = (dh * size).clamp(-65504, 65504).to(F16)

    def wide(t):
        t, keep = torch.full((t.shape[0], t.shape[1] + 3), math.nan, device="cuda", dtype=F16), t
        t[:, 2:-1] = keep
        return t[:, 2:-1]

    x, wg, wu, dh = (wide(t) for t in (x, wg, wu, dh))
    _, gate, up = th.gated_linear(device, x, wg, wu, "gelu", save=True)
    grads = th.gated_linear_grad(device, dh, x, wg, wu, gate, up, "gelu")
    passed = 0
    for (name, (want, err)), got in zip(_exact(dh, x, wg, wu, gate, up, "gelu").items(), grads):
        told = (want.abs() - BORDER).abs() > err
        wrong = told & (got.isinf() != (want.abs() >= BORDER))
        assert not got.isnan().any() and not wrong.any(), (name, int(wrong.sum()), want[wrong][:5].tolist(), got[wrong][:5].tolist())
        passed += int((want.abs() >= BORDER).sum())
    assert passed > 0
