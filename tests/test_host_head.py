"""What the C entry points around a learned head refuse, and the launches of calls
that they take, against a stand-in of the HIP runtime (hostrun.py): no GPU is used and
no kernel runs."""
import ctypes
import re

import hostrun
import thrml_hip as th
from thrml_hip import _lib

P = 1 << 20  # an address that nothing reads: kernels do not run there


def _logits(**kw):
    d = dict(logits=P, dtype=1, q=70, rows=3, logits_stride=70)
    d.update(kw)
    return _lib.Logits(**d)


def _c_calls(calls):
    lib = _lib.load()
    dev = th.Device(0)
    out = []
    for name, args, kw in calls:
        args = [dev.handle if a == "ctx" else ctypes.byref(_logits(**kw)) if a == "d" else a for a in args]
        hostrun.clear_launches()
        rc = getattr(lib, name)(*args)
        out.append((rc, lib.thrml_last_error().decode() if rc else "", sorted(hostrun.launches())))
    return out


def _process(kw=None, out=P, dtype=1, stride=70, ctx="ctx", d="d"):
    return "thrml_process_logits", [ctx, d, out, dtype, stride], kw or {}


def _sample(kw=None, u=P, us=70, index=P, lp=P, work=P, n=1 << 30):
    return "thrml_sample_logits", ["ctx", "d", u, us, index, lp, work, n], kw or {}


def _distill(z=P, dtype=1, rows=3, q=70, zs=70, ids=P, ts=5, k=5, tau=1.0, weight=P, loss=P, grad=2 * P, gs=70, work=P,
             n=1 << 30):
    return "thrml_distill", ["ctx", z, dtype, rows, q, zs, ids, 5, P, ts, k, tau, weight, loss, grad, gs, work, n], {}


def _linear(x=P, dtype=1, rows=3, k=70, xs=70, w=P, q=40, ws=70, sc=P, b=None, y=P, od=1, ys=40, work=P, n=1 << 30):
    return "thrml_linear_i8", ["ctx", x, dtype, rows, k, xs, w, q, ws, sc, b, y, od, ys, work, n], {}


REFUSED = [
    (_process(ctx=None), "NULL argument"), (_process(d=None), "NULL argument"), (_process(out=None), "out is NULL"),
    (_process(dtype=0), "output must be"), (_process(dtype=4), "output must be"), (_process(out=P + 2), "out is not aligned"),
    (_process(stride=69), "rows overlap"), (_process(dict(logits=None)), "logits is NULL"),
    (_process(dict(dtype=0)), "logits must be"), (_process(dict(q=0)), "q must be positive"),
    (_process(dict(q=(1 << 30) + 1)), "2\\^30 categories"), (_process(dict(rows=(1 << 30) + 1)), "2\\^30 rows"),
    (_process(dict(logits=P + 1, dtype=2)), "logits is not aligned"), (_process(dict(logits_stride=-70)), "is negative"),
    (_process(dict(history_len=5)), "history is NULL"), (_process(dict(history=P, history_len=1 << 29)), "2\\^29 - 1"),
    (_process(dict(history=P + 1, history_len=5)), "history is not aligned"),
    (_process(dict(n_bias=2, bias_ids=P)), "bias_values is NULL"), (_process(dict(mask=P, mask_stride=2)), "mask: stride 2"),
    (_process(dict(mask=P + 2)), "mask is not aligned"), (_process(dict(temperature=P + 2)), "temperature is not aligned"),
    (_sample(index=None), "index is NULL"), (_sample(lp=None), "logprob is NULL"), (_sample(u=P + 1), "u is not aligned"),
    (_sample(us=-1), "u: stride -1 is negative"), (_sample(dict(q=1 << 20, logits_stride=1 << 20), us=1 << 20, n=3), "bytes"),
    (_sample(dict(q=1 << 20, logits_stride=1 << 20), us=1 << 20, work=None), "work holds 0 bytes"),
    (_sample(dict(q=1 << 20, logits_stride=1 << 20), us=1 << 20, work=P + 8), "aligned to 16"),
    (_distill(tau=0.0), "tau must be"), (_distill(tau=float("nan")), "tau must be"), (_distill(tau=float("inf")), "tau must be"),
    (_distill(k=4097), "at most 4096 candidates"), (_distill(q=0), "q must be positive"), (_distill(dtype=0), "logits must be"),
    (_distill(z=None), "logits is NULL"), (_distill(ids=None), "ids is NULL"), (_distill(loss=None), "loss is NULL"),
    (_distill(grad=None), "grad is NULL"), (_distill(gs=69), "rows overlap"), (_distill(grad=P), "must not be the logits"),
    (_distill(weight=P + 1), "weight is not aligned"),
    (_distill(q=1 << 17, zs=1 << 17, gs=1 << 17, work=None), "work holds 0 bytes"),
    (_linear(k=0), "k must be positive"), (_linear(k=131073), "at most 131072"), (_linear(q=0), "q must be positive"),
    (_linear(dtype=0), "x must be"), (_linear(od=7), "output must be"), (_linear(x=None), "x is NULL"),
    (_linear(w=None), "w is NULL"), (_linear(sc=None), "w_scale is NULL"), (_linear(y=None), "y is NULL"),
    (_linear(ys=39), "rows overlap"), (_linear(ws=-70), "w: stride -70"), (_linear(rows=99, work=None), "work holds 0 bytes"),
    (_linear(rows=99, n=100), "bytes"), (_linear(b=P + 2), "bias is not aligned"),
]


def test_c_refusals():
    got = hostrun.call(_c_calls, [c for c, _ in REFUSED])
    for (call, msg), (rc, text, launches) in zip(REFUSED, got):
        assert rc < 0 and re.search(msg, text) and not launches, (call, msg, rc, text, launches)


def test_c_calls_that_do_nothing():
    calls = [_process(dict(rows=0, logits=None), out=None), _sample(dict(rows=0, logits=None), index=None, lp=None, work=None, n=0),
             _distill(rows=0, z=None, loss=None, grad=None), _linear(rows=0, x=None, y=None, work=None, n=0)]
    assert [(rc, k) for rc, _, k in hostrun.call(_c_calls, calls)] == [(0, [])] * 4


def test_c_calls_that_run():
    calls = [_process(), _process(dict(rows=1 << 30, logits_stride=0), stride=70), _sample(),
             _sample(dict(rows=1 << 30, logits_stride=0), us=0), _distill(), _distill(rows=1 << 30, zs=0, ts=0), _linear(),
             _linear(rows=1 << 24, xs=0, ys=40, n=1 << 40), _linear(q=1 << 30, ys=1 << 30, rows=1)]
    for call, (rc, text, launches) in zip(calls, hostrun.call(_c_calls, calls)):
        assert rc == 0 and launches, (call, text)
