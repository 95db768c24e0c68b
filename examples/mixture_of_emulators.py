"""A mixture of emulators: trained for a few steps, then asked for single columns.

Columns of 12 features belong to one of several regimes, each with its own
response.  A gate (an ordinary ponni_b200 model) gives every column logits over
the experts; the two experts with the largest logits answer, each a dense
layer, weighted by the gate.  A training step runs

    gate -> route_columns -> gather_columns -> expert_product -> combine_rows
    and back: combine_rows_backward -> expert_product_backward
              -> gather_columns_backward, route_columns_backward

then one GradientSet clips the gradients of all parameters together and packs
them into the flat order that set_trainable_parameters_device takes.

    python examples/mixture_of_emulators.py [--steps 60] [--batch 4096]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ponni_b200 as pb  # noqa: E402


def regimes(features, outputs, count, generator):
    """The truth: a center and a linear response for each regime."""
    r = lambda *s: torch.randn(*s, generator=generator, device="cuda")  # noqa: E731
    return 2.0 * r(count, features), r(count, features, outputs) * features ** -0.5


def columns(center, response, batch, generator):
    """Feature-major inputs [features, batch] around the regimes' centers, and the answers [outputs, batch]."""
    which = torch.randint(len(center), (batch,), generator=generator, device="cuda")
    x = center[which] + 0.5 * torch.randn(batch, center.shape[1], generator=generator, device="cuda")
    y = torch.einsum("bf,bfo->bo", x, response[which])
    return x.t().contiguous(), y.t().contiguous()


class Mixture:
    """A gate and `experts` dense layers features -> outputs, in single precision."""

    def __init__(self, features, outputs, experts, top_k=2, seed=1):
        rng = np.random.default_rng(seed)
        self.top_k = top_k
        self.gate = pb.create_inference_model(pb.Matvec(rng.normal(0, features ** -0.5, (features, experts))),
                                              pb.Bias(np.zeros(experts)))
        self.weights = torch.from_numpy(rng.normal(0, features ** -0.5, (experts, features, outputs))).float().cuda()
        self.bias = torch.zeros(experts, outputs, device="cuda")
        # Gradient buffers that keep their place, and all parameters as one vector in the same order.
        self.d_gate = torch.zeros(features + 1, experts, device="cuda")
        self.d_weights, self.d_bias = torch.zeros_like(self.weights), torch.zeros_like(self.bias)
        self.gradients = pb.GradientSet([self.d_gate, self.d_weights, self.d_bias])
        self.flat = torch.empty(self.gradients.total, device="cuda")
        self.gate_values = self.gate.get_trainable_parameters_device()

    def forward(self, x):
        logits = self.gate.forward_batch_parallel(x)
        routing = pb.route_columns(logits, self.top_k)
        rows = pb.gather_columns(x, routing)
        answers = pb.expert_product(rows, self.weights, routing.offset, bias=self.bias)
        return pb.combine_rows(answers, routing), (logits, routing, rows, answers)

    def step(self, x, y, rate, max_norm):
        """One step of clipped gradient descent on the mean squared error; (loss, gradient norm)."""
        out, (logits, routing, rows, answers) = self.forward(x)
        error = out - y
        d_answers, d_weight = pb.combine_rows_backward(error * (2.0 / y.shape[1]), answers, routing)
        _, d_weights, d_bias = pb.expert_product_backward(d_answers, rows, self.weights, routing.offset,
                                                          need_rows=False)
        d_logits = pb.route_columns_backward(logits, routing, d_weight)
        self.d_gate[:-1] = x @ d_logits.t()
        self.d_gate[-1] = d_logits.sum(1)
        self.d_weights.copy_(d_weights)
        self.d_bias.copy_(d_bias)
        norm = self.gradients.clip(max_norm, out=self.flat)
        gate, weights, bias = self.flat.split([t.numel() for t in self.gradients.tensors])
        self.gate_values.sub_(gate, alpha=rate)
        self.gate.set_trainable_parameters_device(self.gate_values)
        self.weights.sub_(weights.view_as(self.weights), alpha=rate)
        self.bias.sub_(bias.view_as(self.bias), alpha=rate)
        return error.square().sum(0).mean(), norm


def main(steps=60, batch=4096, features=12, outputs=5, experts=6, seed=3):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    truth = regimes(features, outputs, 4, g)
    model = Mixture(features, outputs, experts)
    first = last = None
    for i in range(steps):
        loss, norm = model.step(*columns(*truth, batch, g), rate=0.1, max_norm=5.0)
        last = loss.item()
        first = last if first is None else first
        if i % 20 == 0 or i == steps - 1:
            print(f"step {i}: loss {last:.4f}, gradient norm {norm.item():.3f}")
    x, y = columns(*truth, 3, g)
    alone = torch.cat([model.forward(x[:, i:i + 1].contiguous())[0] for i in range(3)], 1)  # one column at a time
    together = model.forward(x)[0]
    pb.check_operators()
    print(f"single columns: {(alone - y).abs().mean():.4f} from the truth, {(alone - together).abs().max():.1e} from the batch")
    return first, last, (alone - together).abs().max().item()


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--batch", type=int, default=4096)
    a = p.parse_args()
    main(a.steps, a.batch)
