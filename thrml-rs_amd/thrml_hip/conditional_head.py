"""A learned head distilled from a categorical model's conditionals, and drawn from:
the operators of `head` together, on a Potts torus.

The model gives each node's conditional over q categories from its four neighbours.  A
linear head over the neighbours' one-hot features learns it from states that the
sampler visits: the head's product in 8-bit integers gives its logits, the gradient
against the conditional's top candidates trains it, and sample_logits draws categories
from it, with categories ruled out by a mask or made less likely by what a row has
drawn before.

    python -m thrml_hip.conditional_head        (thrml-rs_amd/ on the path)
"""
import numpy as np

from . import (CategoricalProgram, Device, RngKey, distill_grad, linear_i8, make_nearest_neighbor_lattice,
               run_blocks, sample_logits)


class PottsTorus:
    """Potts model on a torus with one coupling and one field for all nodes."""

    def __init__(self, device, side, q, coupling, field):
        self.device, self.q = device, int(q)
        self.n, edges, even, odd = make_nearest_neighbor_lattice(side)
        self.coupling = float(coupling)
        self.field = np.ascontiguousarray(field, dtype=np.float32)
        weights = np.broadcast_to(self.coupling * np.eye(q, dtype=np.float32), (len(edges), q, q))
        self.program = CategoricalProgram(self.n, q, edges, np.ascontiguousarray(weights),
                                          np.tile(self.field, (self.n, 1)), [even, odd], device)
        # global state order: the even block's nodes, then the odd block's
        self.order = np.concatenate([even.nodes, odd.nodes])
        neighbours = [[] for _ in range(self.n)]
        for u, v in edges:
            neighbours[u].append(v)
            neighbours[v].append(u)
        self.neighbours = np.array(neighbours)  # [n, 4]

    def states(self, key, chains, sweeps):
        """[chains, n] categories by node after a run from uniform states."""
        st = self.program.new_state(chains)
        st.set_global(np.random.default_rng(key.seed).integers(0, self.q, (chains, self.n)))
        run_blocks(key, self.program, st, (), sweeps)
        by_node = np.empty((chains, self.n), np.int64)
        by_node[:, self.order] = st.get_global()
        return by_node

    def conditionals(self, states):
        """(features [rows, 4 q], logits [rows, q]) of every node in every state, on the
        device: the neighbours' one-hot categories, and the model's conditional."""
        import torch

        near = torch.from_numpy(states[:, self.neighbours].reshape(-1, 4)).cuda(self.device.ordinal)
        one_hot = torch.nn.functional.one_hot(near, self.q).float()
        logits = self.coupling * one_hot.sum(1) + torch.from_numpy(self.field).to(one_hot.device)
        return one_hot.flatten(1), logits


class ConditionalHead:
    """Logits = x @ w.T + b with w in 8-bit integers, a scale for each category; training
    keeps w in float32."""

    def __init__(self, device, features, q):
        import torch

        self.device = device
        self.w = torch.zeros(q, features, device=f"cuda:{device.ordinal}")
        self.b = torch.zeros(q, device=self.w.device)

    def quantised(self):
        """(int8 weights, scales)"""
        scale = self.w.abs().amax(1) / 127.0
        scale = scale.masked_fill(scale == 0.0, 1.0)
        return (self.w / scale[:, None]).round_().char(), scale

    def logits(self, x):
        w, scale = self.quantised()
        return linear_i8(self.device, x, w, scale, bias=self.b)

    def train_step(self, x, ids, teacher, lr, tau=1.0):
        """One step of gradient descent on the mean loss, which it returns (of before
        the step).  The gradient passes the quantisation straight through."""
        import torch

        rows = x.shape[0]
        loss, grad = distill_grad(self.device, self.logits(x), ids, teacher,
                                  torch.full((rows,), 1.0 / rows, device=x.device), tau)
        self.w -= lr * torch.mm(grad.t(), x)
        self.b -= lr * grad.sum(0)
        return loss.mean()

    def draw(self, x, u=None, **rows):
        """(categories, log-probabilities) for rows of features; `rows` as sample_logits
        takes them (history, penalties, biases, temperature, mask)."""
        return sample_logits(self.device, self.logits(x), u, **rows)


def distil(torus, head, key, steps, chains=4, sweeps=20, top=8, lr=0.8):
    """Trains head on the conditionals of states that torus's sampler visits; the mean
    losses of the steps."""
    losses = []
    for k in key.split(steps):
        x, logits = torus.conditionals(torus.states(k, chains, sweeps))
        teacher, ids = logits.topk(min(top, torus.q), dim=1)
        losses.append(float(head.train_step(x, ids.int(), teacher, lr)))
    return losses


def main():
    import torch

    dev = Device(0)
    dev.set_stream(torch.cuda.current_stream().cuda_stream)
    q = 24
    torus = PottsTorus(dev, 32, q, 1.2, np.linspace(0.4, -0.4, q))
    head = ConditionalHead(dev, 4 * q, q)
    losses = distil(torus, head, RngKey(1), 300, top=q)
    print(f"mean loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    x, logits = torus.conditionals(torus.states(RngKey(2), 8, 20))
    u = torch.rand(x.shape[0], q, device=x.device)
    index, logprob = head.draw(x, u)
    exact = torch.log_softmax(logits, 1).gather(1, index.long()[:, None])[:, 0]
    print(f"{index.numel()} categories drawn, log-probabilities within "
          f"{float((logprob - exact).abs().mean()):.3f} of the model's on average")
    # the same rows without the first 8 categories, and less of what they drew before
    mask = torch.full((1, 1), -1 << 8, dtype=torch.int32, device=x.device)
    again, _ = head.draw(x, u, mask=mask, history=index[:, None].contiguous(),
                         presence=torch.full((x.shape[0],), 2.0, device=x.device))
    print(f"with a mask: categories {int(again.min())}..{int(again.max())}, {int((again == index).sum())} drawn twice")
    torch.cuda.synchronize()


if __name__ == "__main__":
    main()
