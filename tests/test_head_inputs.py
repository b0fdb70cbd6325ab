"""Arguments that the functions around a learned head have to refuse or take, on CPU
tensors: no GPU is used."""
import threading

import pytest
import torch

import thrml_hip as th
from test_head_args import _Device, F, I, S, V, VI, W, Z

X = torch.zeros(2, 70)


def _grad(t):
    return t.clone().requires_grad_()


CALLS = {
    "logits of process_logits": lambda: th.process_logits(_Device(), _grad(Z)),
    "a computed logits": lambda: th.process_logits(_Device(), _grad(Z) * 2.0),
    "transposed logits": lambda: th.process_logits(_Device(), _grad(Z.t().contiguous()).t()),
    "temperature": lambda: th.process_logits(_Device(), Z, temperature=_grad(V)),
    "presence": lambda: th.process_logits(_Device(), Z, history=I, lengths=VI, presence=_grad(V)),
    "bias_values": lambda: th.process_logits(_Device(), Z, bias_ids=I, bias_values=_grad(F)),
    "out": lambda: th.process_logits(_Device(), Z, out=_grad(Z)),
    "logits of sample_logits": lambda: th.sample_logits(_Device(), _grad(Z)),
    "logits of distill_loss": lambda: th.distill_loss(_Device(), _grad(Z), I, F),
    "teacher of distill_loss": lambda: th.distill_loss(_Device(), Z, I, _grad(F)),
    "x": lambda: th.linear_i8(_Device(), _grad(X), W, S),
    "w_scale": lambda: th.linear_i8(_Device(), X, W, _grad(S)),
    "bias": lambda: th.linear_i8(_Device(), X, W, S, bias=_grad(S)),
}


@pytest.mark.parametrize("what", CALLS)
def test_gradients_do_not_end_unsaid(what):
    """A result that torch would not differentiate is refused where it asks for that, and
    computed where it does not (here: as far as the tensors' place)."""
    with pytest.raises(th.ThrmlError, match="requires a gradient"):
        CALLS[what]()
    with torch.no_grad(), pytest.raises(th.ThrmlError, match="is on cpu"):
        CALLS[what]()
    with torch.inference_mode(), pytest.raises(th.ThrmlError, match="is on cpu"):
        CALLS[what]()


def test_distill_grad_takes_leaves():
    """It gives the gradient itself."""
    for z, t, w in ((_grad(Z), F, V), (Z, _grad(F), V), (Z, F, _grad(V))):
        with pytest.raises(th.ThrmlError, match="is on cpu"):
            th.distill_grad(_Device(), z, I, t, w)


def test_second_thread_during_the_first_call(monkeypatch):
    """Nothing of the module is seen half set up: a call from another thread, made between
    any two steps of the first call's setup, is checked as any other."""
    from thrml_hip import head

    seen = []

    class Types(dict):
        def update(self, *args):
            if not seen:
                seen.append(None)
                t = threading.Thread(target=other)
                t.start()
                t.join()
            super().update(*args)

    def other():
        try:
            th.process_logits(_Device(), Z)
        except th.ThrmlError as e:
            seen.append(str(e))

    for name in ("_FLOATS", "_INT32", "_FLOAT32", "_INT8", "_WORDS"):
        monkeypatch.setattr(head, name, ())
    monkeypatch.setattr(head, "torch", None)
    monkeypatch.setattr(head, "_TYPES", Types())
    with pytest.raises(th.ThrmlError, match="is on cpu"):
        th.process_logits(_Device(), Z)
    assert len(seen) == 2 and "is on cpu" in seen[1]
