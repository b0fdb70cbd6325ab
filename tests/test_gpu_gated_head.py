"""The operators of a hidden block as the package uses them together: a head with a gated
block, dropout and an 8-bit product, distilled from a Potts model's conditionals."""
import hidden_reference as ref
import numpy as np
import pytest
import torch
from conftest import log_case

import thrml_hip as th
from thrml_hip.conditional_head import GatedHead, PottsTorus, distil

pytestmark = pytest.mark.gpu

Q, FEATURES, HIDDEN = 12, 48, 200
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def torus():
    dev = th.Device(0)
    dev.set_stream(torch.cuda.current_stream().cuda_stream)
    yield PottsTorus(dev, 16, Q, 1.0, np.linspace(0.5, -0.5, Q))
    torch.cuda.synchronize()
    dev.close()


@pytest.mark.parametrize("key", [None, th.RngKey(77)])
def test_a_step_is_the_gradient(torus, key):
    """every weight's step against the formulas in 64 bits, from the units that the step
    saw (gated_linear and dropout again) and the quantised weights"""
    log_case(f"gated head {key}")
    dev = torus.device
    x, teacher = torus.conditionals(torus.states(th.RngKey(3), 2, 10))
    rows = x.shape[0]
    head = GatedHead(dev, FEATURES, HIDDEN, Q, seed=1, activation="gelu", p=0.3)
    before = [t.clone() for t in (head.w_gate, head.w_up, head.w, head.b)]
    w8, scale = head.quantised()
    ids = torch.arange(Q, device="cuda", dtype=torch.int32).expand(rows, -1)
    loss = head.train_step(x, ids, teacher, 1.0, key=key)
    steps = [a.double() - b.double() for a, b in zip(before, (head.w_gate, head.w_up, head.w, head.b))]

    xb, wg, wu = x.to(BF16), before[0].to(BF16), before[1].to(BF16)
    h, gate, up = th.gated_linear(dev, xb, wg, wu, "gelu", save=True)
    kept = torch.ones_like(h)
    if key is not None:
        kept = th.dropout(dev, kept, key, 0.3)
        h = th.dropout(dev, h, key, 0.3)
    y, ey = (t.cuda() for t in ref.linear_f8(h, w8, scale, before[3], torch.float32))
    p = torch.softmax(teacher.double(), 1)
    logq = torch.log_softmax(y, 1)
    want = (p * (torch.log(p) - logq)).sum(1)
    assert abs(float(loss) - float(want.mean())) < 2 * float(ey.max()) + 64 * ref.U32 * (1 + float(logq.abs().max()))
    # a softmax moves by at most half of what its arguments do
    grad = (torch.exp(logq) - p) / rows
    eg = (ey.amax(1, keepdim=True) + 64 * ref.U32) / rows
    back = scale.double().repeat_interleave(128, 0)[:Q].repeat_interleave(128, 1)[:, :HIDDEN] * w8.double()

    def near(got, want, err, weight):
        # the step itself: a difference of f32 weights
        ref.close(got, want, err + 2.0 * ref.U32 * (weight.double().abs() + want.abs()), "step")

    gt = grad.t().contiguous()
    near(steps[3], grad.sum(0), eg.sum() + rows * ref.U32 * grad.abs().sum(0), before[3])
    near(steps[2], gt @ h.double(), eg.sum() * h.double().abs().amax(0) + rows * ref.U32 * (gt.abs() @ h.double().abs()), before[2])
    dh, edh = grad @ back, eg * back.abs().sum(0) + Q * ref.U32 * (grad.abs() @ back.abs())
    scaled = kept.double()
    # rounded to bf16, and where there is dropout once more
    edh = scaled * (edh + 2 * 2.0**-8 * dh.abs() * 1.01) + 2.0**-133
    dh = dh * scaled
    sums = ref.gated_grad(dh, xb, wg, wu, gate, up, "gelu")
    a, slope = ref.act(gate.double(), "gelu")
    for i, (name, factor) in enumerate((("dw_gate", up.double() * slope), ("dw_up", a))):
        moved = torch.mm((edh * factor.abs()).t().contiguous(), xb.double().abs())
        value, err = sums[name]
        near(steps[i], value, err + 1.1 * moved, before[i])


def test_training_and_draws(torus):
    dev = torus.device
    head = GatedHead(dev, FEATURES, HIDDEN, Q, p=0.1)
    losses = distil(torus, head, th.RngKey(5), 10, top=Q, lr=0.2)
    again = GatedHead(dev, FEATURES, HIDDEN, Q, p=0.1)
    assert losses == distil(torus, again, th.RngKey(5), 10, top=Q, lr=0.2) and torch.equal(head.w_gate, again.w_gate)
    assert all(np.isfinite(losses))
    x, _ = torus.conditionals(torus.states(th.RngKey(9), 8, 20))
    logits = head.logits(x)
    w8, scale = head.quantised()
    h = th.gated_linear(dev, x.to(BF16), head.w_gate.to(BF16), head.w_up.to(BF16))
    ref.close(logits.cpu(), *ref.linear_f8(h, w8, scale, head.b, torch.float32), "logits")
    u = torch.rand(x.shape[0], Q, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    index, logprob = head.draw(x, u)
    score = logits.double() - torch.log(-torch.log(u.double()))
    assert torch.equal(index.long(), score.argmax(1))
    assert (logprob.double() - torch.log_softmax(logits.double(), 1).gather(1, index.long()[:, None])[:, 0]).abs().max() < 1e-5
    mask = torch.full((1, 1), -1 << 4, dtype=torch.int32, device="cuda")
    assert (head.draw(x, u, mask=mask)[0] >= 4).all()
