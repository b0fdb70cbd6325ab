"""What the Python functions of a learned head's hidden block refuse, on CPU tensors: no GPU
is used."""
import pytest
import torch
from test_head_args import _Device

import thrml_hip as th

B = torch.bfloat16
X = torch.zeros(3, 70, dtype=B)
W = torch.zeros(40, 70, dtype=B)
H = torch.zeros(3, 40, dtype=B)
G = torch.zeros(3, 40)
KEY = th.RngKey(1)
W8 = torch.zeros(200, 70, dtype=torch.uint8).view(torch.float8_e4m3fn)
S8 = torch.zeros(2, 1)


@pytest.mark.parametrize("args,kw,msg", [
    ((X.float(), W, W), {}, "x must be a bfloat16 or float16"), ((X[0], W, W), {}, "x must have shape"),
    ((X, W.half(), W), {}, "w_gate must be a bfloat16 tensor"), ((X, W, W.float()), {}, "w_up must be a bfloat16 tensor"),
    ((X, W[:, :69], W), {}, "w_gate must have shape"), ((X, W, W[:39]), {}, "w_up must have shape"),
    ((X[:, :0], W[:, :0], W[:, :0]), {}, "at least one row and column"), ((X, W[:0], W[:0]), {}, "at least one row and column"),
    ((X, W, W, "tanh"), {}, "activation must be one of silu, gelu, relu"), ((X, W, W, None), {}, "activation must be"),
    ((X, W, W), dict(out=H[:2]), "out must be"), ((X, W, W), dict(out=H.half()), "out must be"),
    ((X, W, W), {}, "x is on cpu"), (([[1.0]], W, W), {}, "x must be a"),
])
def test_gated(args, kw, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.gated_linear(_Device(), *args, **kw)


@pytest.mark.parametrize("args,msg", [
    ((H.half(), X, W, W, G, G), "grad must be a bfloat16 tensor"), ((H[:2], X, W, W, G, G), "grad must have shape"),
    ((H, X, W, W, G[:, :39], G), "gate must have shape"), ((H, X, W, W, H, G), "gate must be a float32 tensor"), ((H, X, W, W, G, None), "up must be a"),
    ((H, X, W, W, G, G, "none"), "activation must be"), ((H, X, W, W, G, G), "x is on cpu"),
])
def test_gated_grad(args, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.gated_linear_grad(_Device(), *args)


@pytest.mark.parametrize("x,key,p,kw,msg", [
    (X.int(), KEY, 0.5, {}, "x must be a float32"), (X[0], KEY, 0.5, {}, "x must have shape"),
    (X, 5, 0.5, {}, "key must be an RngKey or"), (X, None, 0.5, {}, "key must be"),
    (X, torch.zeros(2, dtype=torch.int64), 0.5, {}, "key must be"), (X, torch.zeros(1), 0.5, {}, "key must be"),
    (X, KEY, 0.5, dict(residual=X.half()), "residual must be a bfloat16 tensor"),
    (X, KEY, 0.5, dict(residual=X[:2]), "residual must have shape"), (X, KEY, 0.5, dict(first_row=-1), "first_row must lie"), (X, KEY, 0.5, dict(first_row=1 << 64), "first_row must lie"),
    (X, KEY, 0.5, dict(out=X[:2]), "out must be"), (X, KEY, 0.5, {}, "x is on cpu"),
])
def test_dropout(x, key, p, kw, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.dropout(_Device(), x, key, p, **kw)


def test_dropout_in_place_needs_rows():
    t = torch.zeros(70, 3, dtype=B).t()
    with pytest.raises(th.ThrmlError, match="out must be|only where their rows are contiguous"):
        th.dropout(_Device(), t, KEY, 0.5, out=t)


@pytest.mark.parametrize("args,kw,msg", [
    ((X.long(), W8, S8), {}, "x must be a float32"), ((X, W, S8), {}, "w must be a float8_e4m3fn"),
    ((X, W8[:, :69], S8), {}, "w must have shape"), ((X, W8, S8[:1]), {}, "w_scale must have shape"),
    ((X, W8, S8.half()), {}, "w_scale must be a float32"), ((X, W8, None), {}, "w_scale must be a"),
    ((X, W8, torch.zeros(200, 1)), {}, "w_scale must have shape"), ((X, W8, S8), dict(bias=torch.zeros(199)), "bias must be"),
    ((X[:, :0], W8[:, :0], S8[:, :0]), {}, "at least one row and column"), ((X, W8[:0], S8[:0]), {}, "at least one row and column"),
    ((X, W8, S8), dict(out_dtype=torch.int8), "out_dtype must be"), ((X, W8, S8), {}, "x is on cpu"),
])
def test_linear_f8(args, kw, msg):
    with pytest.raises(th.ThrmlError, match=msg):
        th.linear_f8(_Device(), *args, **kw)
