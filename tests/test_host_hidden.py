"""What the C entry points of a learned head's hidden block refuse, and the launches of
calls that they take, against a stand-in of the HIP runtime (hostrun.py): no GPU is used
and no kernel runs."""
import re

import hostrun
import thrml_hip as th
from thrml_hip import _lib, hidden

Q = 1 << 21
P = 1 << 20  # an address that nothing reads: kernels do not run there
WORK = 1 << 50


def _desc(x=P, dtype=2, act=0, rows=3, k=70, n=40, xs=70, wg=P, gs=70, wu=P, us=70):
    return hidden._PACK(x or 0, dtype, act, rows, k, n, xs, wg or 0, gs, wu or 0, us)


def _calls(calls):
    lib = _lib.load()
    dev = th.Device(0)
    out = []
    for name, args in calls:
        hostrun.clear_launches()
        rc = getattr(lib, name)(*[dev.handle if a == "ctx" else a for a in args])
        out.append((rc, lib.thrml_last_error().decode() if rc else "", sorted(hostrun.launches().items())))
    return out


def _forward(h=Q, hs=40, gate=P, up=P, work=P, have=WORK, ctx="ctx", **kw):
    return "thrml_gated_forward", [ctx, _desc(**kw), h, hs, gate, up, work, have]


def _backward(grad=P, gs=40, gate=P, up=P, dx=Q, dxs=70, dwg=Q, dwu=Q, work=P, have=WORK, **kw):
    wgs = kw.pop("wgs", 70)
    return "thrml_gated_backward", ["ctx", _desc(gs=wgs, **kw), grad, gs, gate, up, dx, dxs, dwg, dwu, work, have]


def _dropout(x=P, dtype=2, rows=3, cols=40, xs=40, res=None, rs=0, seed=1, at=None, first=0, p=0.5, y=P, ys=40, ctx="ctx"):
    return "thrml_dropout", [ctx, x, dtype, rows, cols, xs, res, rs, seed, at, first, p, y, ys]


def _f8(x=P, dtype=2, rows=3, k=70, xs=70, w=P, q=40, ws=70, sc=P, b=None, y=P, od=2, ys=40, work=P, have=WORK, ctx="ctx"):
    return "thrml_linear_f8", [ctx, x, dtype, rows, k, xs, w, q, ws, sc, b, y, od, ys, work, have]


REFUSED = [
    (_forward(ctx=None), "NULL argument"), (("thrml_gated_forward", ["ctx", None, P, 40, P, P, P, WORK]), "NULL argument"),
    (_forward(dtype=1), "must be bf16 or f16"), (_forward(dtype=0), "must be bf16 or f16"), (_forward(act=3), "unknown activation"),
    (_forward(act=-1), "unknown activation"), (_forward(k=0), "must be positive"), (_forward(n=0), "must be positive"),
    (_forward(k=(1 << 20) + 1, xs=1 << 21, gs=1 << 21, us=1 << 21), "at most 2\\^20"), (_forward(n=(1 << 20) + 1), "at most 2\\^20"),
    (_forward(rows=(1 << 30) + 1), "2\\^30 rows"), (_forward(x=None), "x is NULL"), (_forward(x=P + 1), "x is not aligned"),
    (_forward(xs=-70), "x: stride -70 is negative"), (_forward(wg=None), "w_gate is NULL"), (_forward(wu=P + 1), "w_up is not aligned"),
    (_forward(us=-1), "w_up: stride -1"), (_forward(h=None), "h is NULL"), (_forward(hs=39), "h: stride 39 makes rows overlap"),
    (_forward(gate=None), "gate and up go together"), (_forward(up=None), "gate and up go together"),
    (_forward(gate=P + 1), "gate is not aligned"), (_forward(rows=99, work=None), "work holds 0 bytes"), (_forward(rows=99, have=100), "work holds 100 bytes"),
    (_forward(rows=99, work=P + 8), "work is not aligned"),
    (_backward(grad=None), "grad is NULL"), (_backward(gs=-1), "grad: stride -1"), (_backward(gate=None), "gate is NULL"),
    (_backward(up=None), "up is NULL"), (_backward(dx=Q + 1), "dx is not aligned"), (_backward(dxs=69), "dx: stride 69"),
    (_backward(dwg=None), "dw_gate is NULL"), (_backward(dwu=Q + 1), "dw_up is not aligned"), (_backward(have=5), "work holds 5 bytes"),
    (_forward(h=P), "h must not be x or a weight"), (_backward(dx=P), "dx must not be"), (_backward(dwg=P), "dw_gate must not be"),
    (_backward(dwu=P), "dw_up must not be"),
    (_dropout(ctx=None), "NULL argument"), (_dropout(dtype=0), "x must be"), (_dropout(p=-0.1), "p must lie in"),
    (_dropout(p=1.1), "p must lie in"), (_dropout(p=float("nan")), "p must lie in"), (_dropout(x=None), "x is NULL"),
    (_dropout(x=P + 1), "x is not aligned"), (_dropout(xs=-1), "x: stride -1"), (_dropout(res=P + 1), "residual is not aligned"),
    (_dropout(res=P, rs=-4), "residual: stride -4"), (_dropout(y=None), "y is NULL"), (_dropout(ys=39), "y: stride 39"),
    (_dropout(at=P + 4), "seed_at is not aligned"), (_dropout(first=1 << 37), "at most 2\\^37"),
    (_dropout(rows=1 << 20, cols=1 << 18), "at most 2\\^37"), (_dropout(first=(1 << 64) - 1), "at most 2\\^37"),
    (_dropout(rows=(1 << 64) - 1, first=5), "at most 2\\^37"),
    (_f8(ctx=None), "NULL argument"), (_f8(k=0), "k must be positive"), (_f8(k=(1 << 20) + 1), "at most 2\\^20"),
    (_f8(q=0), "q must be positive"), (_f8(rows=(1 << 30) + 1), "2\\^30 rows"), (_f8(dtype=0), "x must be"), (_f8(od=7), "output must be"),
    (_f8(x=None), "x is NULL"), (_f8(w=None), "w is NULL"), (_f8(ws=-70), "w: stride -70"), (_f8(sc=None), "w_scale is NULL"),
    (_f8(sc=P + 2), "w_scale is not aligned"), (_f8(b=P + 2), "bias is not aligned"), (_f8(y=None), "y is NULL"),
    (_f8(ys=39), "rows overlap"), (_f8(rows=99, work=None), "work holds 0 bytes"), (_f8(rows=99, have=100), "bytes"), (_f8(rows=99, work=P + 4), "not aligned to 16"),
]


def test_c_refusals():
    for (call, msg), (rc, text, launches) in zip(REFUSED, hostrun.call(_calls, [c for c, _ in REFUSED])):
        assert rc < 0 and re.search(msg, text) and not launches, (call, msg, rc, text, launches)


def test_c_calls_that_do_nothing():
    calls = [_forward(rows=0, x=None, h=None, gate=None, up=None, work=None, have=0), _dropout(rows=0, x=None, y=None),
             _dropout(cols=0, x=None, y=None), _f8(rows=0, x=None, y=None, sc=None, work=None, have=0)]
    assert [(rc, k) for rc, _, k in hostrun.call(_calls, calls)] == [(0, [])] * 4


def test_c_calls_that_run():
    calls = [_forward(), _forward(gate=None, up=None), _forward(rows=1 << 22, xs=0), _backward(), _backward(dx=None),
             _backward(rows=0, x=None, grad=None, gate=None, up=None, dx=None, work=None, have=0), _dropout(), _dropout(res=P, rs=40),
             _dropout(rows=1 << 27, xs=0), _dropout(p=0.0), _dropout(p=1.0), _f8(), _f8(rows=1 << 20, xs=0), _f8(q=1 << 20, ys=1 << 20),
             _forward(k=1 << 20, n=1 << 20, xs=1 << 20, gs=1 << 20, us=1 << 20, hs=1 << 20),
             _backward(k=1 << 20, n=1 << 16, xs=1 << 20, wgs=1 << 20, us=1 << 20, gs=1 << 16, dxs=1 << 20)]
    for call, (rc, text, launches) in zip(calls, hostrun.call(_calls, calls)):
        assert rc == 0 and launches, (call, text)


def _names(calls):
    got = hostrun.call(_calls, calls)
    assert all(rc == 0 for rc, _, _ in got), got
    return [" ".join(k for k, _ in names).replace(" ", "") for _, _, names in got]


def test_aligned_operands_are_not_copied():
    for k, pad, shift, copied in ((64, 0, 0, False), (64, 8, 0, False), (64, 8, 16, False), (65, 0, 0, True), (64, 1, 0, True),
                                  (64, 0, 2, True), (63, 1, 0, True)):
        names, = _names([_forward(rows=99, k=k, xs=k + pad, gs=k + pad, us=k + pad, x=P + shift, wg=P + shift, wu=P + shift)])
        assert ("gated_pack_kernel" in names) == copied, (k, pad, shift, names)
    for k, pad, shift, copied in ((64, 0, 0, False), (80, 16, 0, False), (64, 0, 16, False), (64, 8, 0, True), (72, 0, 0, True), (64, 0, 8, True)):
        names, = _names([_f8(rows=99, k=k, xs=k, ws=k + pad, w=P + shift)])
        assert ("f8_pack_kernel" in names) == copied, (k, pad, shift, names)


def test_work_is_what_calls_take():
    """a call with exactly the bytes that the work function gives runs, with 1 less it does not"""
    for rc, enough in hostrun.call(_work_calls):
        assert (rc == 0) == enough


def _work_calls():
    lib, dev = _lib.load(), th.Device(0)
    out = []
    for rows, k, n in ((1, 4096, 512), (70, 200, 130), (1100, 520, 768), (64, 8192, 64)):
        d = _desc(rows=rows, k=k, n=n, xs=k, gs=k, us=k)
        for back in (0, 1):
            w = lib.thrml_gated_work(dev.handle, d, back)
            f = lib.thrml_gated_backward if back else lib.thrml_gated_forward
            a = (P, n, P, P, Q, k, Q, Q) if back else (Q, n, P, P)
            for have in (w, w - 1) if w else ():
                out.append((f(dev.handle, d, *a, P, have), have == w))
        w = lib.thrml_linear_f8_work(dev.handle, rows, k, P, n, k, 1)
        for have in (w, w - 1) if w else ():
            out.append((lib.thrml_linear_f8(dev.handle, P, 2, rows, k, k, P, n, k, P, None, P, 1, n, P, have), have == w))
    return out


def test_few_unaligned_rows_are_read_as_they_lie():
    for call, kernel in ((_forward(rows=16, k=71), "gated_few_kernel"), (_forward(rows=32, k=71, work=None, have=0), "gated_few_kernel"),
                         (_f8(rows=64, k=71, xs=71), "f8_few_kernel")):
        names, = _names([call])
        assert kernel in names and "pack" not in names and "tile" not in names, (call, names)


def test_each_kind_of_tile():
    """the shapes that the GPU tests name reach the tiles that they are meant for"""
    names = _names([_forward(rows=r, k=k, n=n, xs=k, gs=k, us=k, hs=n) for r, k, n in ((1, 4096, 704), (64, 4096, 8192), (512, 1024, 4096), (2056, 1024, 2048))])
    for shape, got in zip(("64,32,1,1,4", "64,32,1,2,2", "64,64,2,2,1", "128,64,2,4,1"), names):
        mangled = "".join(f"Li{n}E" for n in shape.split(","))
        assert shape in got or mangled in got, (shape, got)
    assert "join" in names[0]
