"""The states that a head is distilled from, without a GPU: what PottsTorus hands to the
sampler."""
import types

import numpy as np
import pytest

import thrml_hip as th
from thrml_hip import conditional_head


@pytest.mark.parametrize("q", [2, 24, 256, 257, 700, 65536])
def test_initial_states_are_uniform(monkeypatch, q):
    """Every category of a model may come first: a twentieth of 20000 uniform draws, give or
    take 6 standard deviations, in each twentieth of the range."""
    given = []
    state = types.SimpleNamespace(set_global=given.append, get_global=lambda: np.zeros((8, 2500), np.uint16))
    torus = types.SimpleNamespace(q=q, n=2500, order=np.arange(2500), program=types.SimpleNamespace(new_state=lambda n: state))
    monkeypatch.setattr(conditional_head, "run_blocks", lambda *a: None)
    out = conditional_head.PottsTorus.states(torus, th.RngKey(5), 8, 3)
    assert out.shape == (8, 2500)
    init = np.asarray(given[0]).astype(np.int64)
    assert init.shape == (8, 2500) and init.min() >= 0 and init.max() < q
    bins = min(q, 20)
    n = np.bincount(init.ravel() * bins // q, minlength=bins)
    share = np.bincount(np.arange(q) * bins // q, minlength=bins) / q
    assert (abs(n - 20000 * share) < 6 * np.sqrt(20000 * share * (1 - share))).all()
