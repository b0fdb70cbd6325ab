"""The operators around a learned head as the package uses them together: a head
distilled from a Potts model's conditionals, and categories drawn from it."""
import numpy as np
import pytest
import torch
from conftest import log_case

import thrml_hip as th
from thrml_hip.conditional_head import ConditionalHead, PottsTorus, distil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def trained():
    log_case("distil")
    dev = th.Device(0)
    dev.set_stream(torch.cuda.current_stream().cuda_stream)
    torus = PottsTorus(dev, 16, 12, 1.0, np.linspace(0.5, -0.5, 12))
    head = ConditionalHead(dev, 48, 12)
    losses = distil(torus, head, th.RngKey(3), 40, top=12)
    yield dev, torus, head, losses
    torch.cuda.synchronize()
    dev.close()


def test_first_step_is_the_formula(trained):
    """From zero weights the first loss is that of the uniform distribution, and the step
    is the mean of (softmax - p) x."""
    dev, torus, _, losses = trained
    k = th.RngKey(3).split(40)[0]
    x, logits = torus.conditionals(torus.states(k, 4, 20))
    p = torch.softmax(logits.double(), 1)
    want = (p * (torch.log(p) + np.log(12))).sum(1).mean()
    assert abs(losses[0] - float(want)) < 64 * 2.0**-24 * (1 + np.log(12)) * 12
    head = ConditionalHead(dev, 48, 12)
    head.train_step(x, torch.arange(12, device="cuda", dtype=torch.int32).expand(x.shape[0], -1), logits, 1.0)
    step = -((1 / 12 - p).t() @ x.double()) / x.shape[0]
    # a sum of 1024 rows in f32, terms of at most 1 / 1024
    assert (head.w.double() - step).abs().max() < 2.0**-24 * 1024


def test_loss_falls(trained):
    """Gradient descent on one batch: the loss is convex with a curvature of at most (4 +
    1) / 2 (features of squared length 4, the bias; softmax 1/2), so that steps of 0.4 never
    raise it, but for what the weights' rounding to 8 bits moves the logits: 4 features by
    half a step each, which moves a loss by at most twice that."""
    dev, torus, _, losses = trained
    x, logits = torus.conditionals(torus.states(th.RngKey(4), 2, 20))
    ids = torch.arange(12, device="cuda", dtype=torch.int32).expand(x.shape[0], -1)
    head = ConditionalHead(dev, 48, 12)
    steps = [float(head.train_step(x, ids, logits, 0.4)) for _ in range(60)]
    slack = 2 * 4 * 0.5 * float(head.w.abs().max()) / 127 + 1e-5
    assert all(b <= a + slack for a, b in zip(steps, steps[1:]))
    assert steps[-1] < 0.5 * steps[0] and losses[-1] < losses[0]


def test_draws(trained):
    dev, torus, head, _ = trained
    x, _ = torus.conditionals(torus.states(th.RngKey(9), 8, 20))
    rows = x.shape[0]
    u = torch.rand(rows, 12, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    logits = head.logits(x)
    w, scale = head.quantised()
    want = (x.double() @ w.double().t()) * scale.double() + head.b.double()
    # one-hot rows quantise exactly: 1 is 127 steps of 1 / 127
    assert (logits.double() - want).abs().max() < 8 * 2.0**-24 * float(want.abs().max() + head.b.abs().max() + 1)
    index, logprob = head.draw(x, u)
    score = logits.double() - torch.log(-torch.log(u.double()))
    assert torch.equal(index.long(), score.argmax(1))
    assert (logprob.double() - torch.log_softmax(logits.double(), 1).gather(1, index.long()[:, None])[:, 0]).abs().max() < 1e-5
    # ruled out categories and what a row has drawn before
    mask = torch.full((1, 1), -1 << 4, dtype=torch.int32, device="cuda")
    history = index[:, None].contiguous()
    again, _ = head.draw(x, u, mask=mask, history=history, presence=torch.full((rows,), 1e4, device="cuda"))
    assert (again >= 4).all() and not (again == index).any()
