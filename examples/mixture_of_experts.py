"""A small mixture-of-experts classifier, trained with orthogonalised updates.

    python examples/mixture_of_experts.py [--device hip] [--steps 40]

Each layer's tokens go through a router (sigmoid scores, a balancing bias), the gated feed-forward units of their two best
experts, and back into the residual stream. Matrices are updated by muon_step, the output bias by sgd_step, and the
balancing bias by the experts' loads, without a gradient.
"""

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import vectorcore_amd as vc  # noqa: E402


def clusters(n, features, classes, rng):
    """Points around two centres per class: a class is no single direction."""
    centres = rng.standard_normal((classes, 2, features)).astype(np.float32)
    labels = rng.integers(0, classes, n)
    x = centres[labels, rng.integers(0, 2, n)] + 0.4 * rng.standard_normal((n, features)).astype(np.float32)
    return x.astype(np.float32), labels


class MixtureOfExperts:
    def __init__(self, features, classes, width=64, hidden=48, experts=8, top_k=2, layers=2, seed=0, device="cpu"):
        rng = np.random.default_rng(seed)
        self.experts, self.top_k, self.device = experts, top_k, device

        def matrix(*shape):
            bound = (3.0 / shape[-2]) ** 0.5
            return vc.Tensor(rng.uniform(-bound, bound, shape).astype(np.float32), requires_grad=True, device=device)

        self.first, self.last = matrix(features, width), matrix(width, classes)
        self.layers = [dict(router=matrix(width, experts), gate=matrix(experts, width, hidden),
                            up=matrix(experts, width, hidden), down=matrix(experts, hidden, width),
                            bias=np.zeros(experts, np.float32)) for _ in range(layers)]
        self.last_bias = vc.Tensor.zeros((classes,), requires_grad=True, device=device)
        self.matrices = [self.first, self.last]
        for layer in self.layers:
            self.matrices += [layer[n] for n in ("router", "gate", "up", "down")]
        self.momenta = [vc.Tensor.zeros(m.shape, device=device) for m in self.matrices]

    def __call__(self, x):
        h, self.chosen = x @ self.first, []
        for layer in self.layers:
            weights, chosen = vc.route(h @ layer["router"], self.top_k, bias=vc.Tensor(layer["bias"], device=self.device),
                                       score="sigmoid")
            plan = vc.ExpertPlan(chosen, self.experts)
            rows = vc.expert_linear(vc.expert_gated(h, layer["gate"], layer["up"], plan), layer["down"], plan, ordered=True)
            h = h + vc.expert_combine(rows, weights, plan)
            self.chosen.append(chosen)
        return h @ self.last + self.last_bias

    def step(self, x, labels, lr=0.02):
        logits = self(x)
        loss = vc.cross_entropy(logits, labels)
        loss.backward()
        vc.muon_step(self.matrices, self.momenta, lr, weight_decay=0.01)
        vc.sgd_step([self.last_bias], lr)
        vc.zero_grad(self.matrices + [self.last_bias])
        for layer, chosen in zip(self.layers, self.chosen):  # experts above the mean load become less liked
            load = np.bincount(chosen.numpy().astype(int).ravel(), minlength=self.experts)
            layer["bias"] -= np.float32(1e-3) * np.sign(load - load.mean()).astype(np.float32)
        return loss.item()


def train(device="cpu", steps=40, n=1024, features=16, classes=4, seed=0):
    rng = np.random.default_rng(seed)
    x, labels = clusters(n, features, classes, rng)
    model = MixtureOfExperts(features, classes, seed=seed, device=device)
    data = vc.Tensor(x, device=device)
    losses = [model.step(data, labels) for _ in range(steps)]
    right = (model(data).argmax(1).numpy() == labels).mean()
    return losses, right


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--device", default="hip" if vc.hip_available() else "cpu")
    parser.add_argument("--steps", type=int, default=40)
    args = parser.parse_args()
    losses, right = train(args.device, args.steps)
    print(f"{args.device}: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps, {100 * right:.1f}% right")
