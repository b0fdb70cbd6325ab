"""What the Python functions around a learned head refuse, on CPU tensors: no GPU is
used."""
import pytest
import torch

import thrml_hip as th


class _Device:
    """A device's attributes without a context: a call that got as far as the
    library would fail on it."""

    ordinal = 0
    handle = None
    stream = None


Z = torch.zeros(3, 70)
I = torch.zeros(3, 5, dtype=torch.int32)
F = torch.zeros(3, 5)
V = torch.zeros(3)
VI = torch.zeros(3, dtype=torch.int32)
W = torch.zeros(4, 70, dtype=torch.int8)
S = torch.zeros(4)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=Z.double()), "logits must be a float32"),
    (dict(logits=[[1.0]]), "logits must be a float32"),
    (dict(logits=Z[0]), r"logits must have shape"),
    (dict(logits=Z[:, :0]), "at least one category"),
    (dict(history=I.long()), "history must be a int32"),
    (dict(history=I[:2]), "history must have shape"),
    (dict(lengths=VI), "lengths needs a history"),
    (dict(repetition=V), "repetition needs a history"),
    (dict(history=I, lengths=V), "lengths must be a int32"),
    (dict(history=I, presence=V[:2]), r"presence must be a float32 tensor of shape \[3\]"),
    (dict(bias_ids=I), "go together"),
    (dict(bias_values=F), "go together"),
    (dict(bias_ids=I, bias_values=F[:, :4]), "bias_values must have shape"),
    (dict(temperature=V[None]), "temperature must be"),
    (dict(temperature=1.0), "temperature must be"),
    (dict(mask=I[:, :3].float()), "mask must be a int32"),
    (dict(mask=I[:, :4]), "mask must have shape"),
    (dict(mask=I[:2, :3]), "mask must have 1 or 3 rows"),
    (dict(), "logits is on cpu"),
])
def test_logit_rows(kw, msg):
    kw = {"logits": Z, **kw}
    z = kw.pop("logits")
    for f in (th.process_logits, th.sample_logits):
        with pytest.raises(th.ThrmlError, match=msg):
            f(_Device(), z, **kw)


def test_outputs_and_uniforms():
    for kw, msg in ((dict(out_dtype=torch.int32), "out_dtype must be"), (dict(out=Z[:2]), "out must be"),
                    (dict(out=Z.half()), "out must be"), (dict(out=torch.zeros(70, 3).t()), "out must be")):
        with pytest.raises(th.ThrmlError, match=msg):
            th.process_logits(_Device(), Z, **kw)
    t = torch.zeros(70, 3).t()
    with pytest.raises(th.ThrmlError, match="only where their rows are contiguous"):
        th.process_logits(_Device(), t, out=t)
    for u in (Z[:, :69], Z.double(), Z[0]):
        with pytest.raises(th.ThrmlError, match="u must"):
            th.sample_logits(_Device(), Z, u)


@pytest.mark.parametrize("args,msg", [
    ((Z.int(), I, F, V), "logits must be a float32"), ((Z, I.long(), F, V), "ids must be a int32"),
    ((Z, I, F[:, :3], V), "teacher must have shape"), ((Z, I[:1], F, V), "ids must have shape"),
    ((Z, I, F, None), "weight is needed"), ((Z, I, F, V[:1]), "weight must be"), ((Z, I, F.half(), V), "teacher must be"),
    ((Z, I, F, V), "logits is on cpu"),
])
def test_distill(args, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.distill_grad(_Device(), *args)


@pytest.mark.parametrize("args,kw,msg", [
    ((Z.long(), W, S), {}, "x must be a float32"), ((Z, W.short(), S), {}, "w must be a int8"),
    ((Z, W[:, :69], S), {}, "w must have shape"), ((Z, W, S[:3]), {}, "w_scale must be"),
    ((Z, W, None), {}, "w_scale is needed"), ((Z, W, S), dict(bias=S.half()), "bias must be"),
    ((Z[:, :0], W[:, :0], S), {}, "at least one row and column"), ((Z, W[:0], S[:0]), {}, "at least one row and column"),
    ((Z, W, S), dict(out_dtype=torch.int8), "out_dtype must be"), ((Z, W, S), {}, "x is on cpu"),
])
def test_linear(args, kw, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.linear_i8(_Device(), *args, **kw)
